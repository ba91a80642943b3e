// What the kernels over a paged cache share: a wave finds the sequence and the cache place of a row, and a page's bytes.
#pragma once
#include "kernels.h"

namespace oavsr {

constexpr int kBadPage = 1, kBadLength = 2;      // bits of *status (include/omni_avsr.h: OAVSR_PAGED_BAD_*)

constexpr int64_t kMaxThreads = (1ll << 32) - 1;      // of a launch, in one dimension

__device__ __forceinline__ void paged_report(int* status, int bit) {
  if (status) atomicOr(status, bit);             // (the same word whoever comes first)
}

// The last sequence whose first row is <= row, by all lanes of a wave together (64 entries of cu_q a step: one step up to 64 sequences, two up to 4096).
// Any content of cu_q ends it inside [0, n_seqs).
__device__ __forceinline__ int wave_find_seq(const int* __restrict__ cu_q, int n_seqs, int row, int lane) {
  int lo = 0, span = n_seqs;
  while (span > 1) {
    const int step = (span + 63) >> 6, i = lane * step;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(i < span && cu_q[lo + (i < span ? i : 0)] <= row);
    const int k = (m ? 63 - __builtin_clzll(m) : 0) * step;
    lo += k;
    span = span - k < step ? span - k : step;
  }
  return lo;
}

// A sequence of the batch, checked: nq new tokens from row q0 on; nq = 0 for one that must be skipped.
struct SeqInfo { int q0, nq, ctx; bool bad; };
__host__ __device__ __forceinline__ SeqInfo paged_seq(const PagedBatch& b, int s) {
  SeqInfo i;
  const int e = b.cu_q[s + 1];
  i.q0 = b.cu_q[s];
  i.ctx = b.ctx_len[s];
  const int64_t n = (int64_t)e - i.q0;
  const bool skip = n < 0 || i.q0 < 0 || e > b.rows || n > b.max_q;
  i.nq = skip ? 0 : (int)n;
  i.bad = skip || i.ctx < 0 || i.ctx > b.max_ctx;
  if (i.ctx < 0) i.ctx = 0;
  return i;
}

// Reports any bad sequence of the batch, those that bring no rows among them: one wave of a launch.
__device__ __forceinline__ void report_bad_lengths(const PagedKv& kv, const PagedBatch& b, int lane) {
  bool bad = false;
  for (int s = lane; s < b.n_seqs; s += 64) bad |= paged_seq(b, s).bad;
  if (bad) paged_report(kv.status, kBadLength);
}

// The page that holds place `pos` (0 <= pos < max_ctx) of sequence s; -1: its number is none of the pool's.
__host__ __device__ __forceinline__ int paged_page(const PagedKv& kv, const PagedBatch& b, int s, int pos, int page_shift) {
  const int page = b.table[(int64_t)s * b.ld_table + (pos >> page_shift)];
  return (unsigned)page < (unsigned)kv.n_pages ? page : -1;
}
__host__ __device__ __forceinline__ int page_shift_of(const PagedKv& kv) { return 31 - __builtin_clz(kv.page_size); }

// four e4m3 bytes -> f32
__device__ __forceinline__ void e4m3_to_f32(unsigned w, float* out) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  out[0] = a[0]; out[1] = a[1]; out[2] = b[0]; out[3] = b[1];
}

}  // namespace oavsr
