// Rows into and out of a paged key / value cache, and the norm + rotation of queries and keys in the same pass.
//
// qk_rope_kernel: a fused row is [q heads | k heads | v heads] x head_dim.  Per q and k head, in f32,
//     x <- x * rsqrt(mean x^2 + eps) * gain,     (a, b) <- m (a cos t - b sin t, b cos t + a sin t),  t = pos * f_i,
// one rounding at the end; then q to its buffer, k to its buffer or (CACHE) its page, v to its page, in 8 bits (F8) with one scale per head.
//   * HBM bound: a row is read once and written once.  head_dim / 16 lanes own a head, a lane two (bf16) or four (f32) 16-byte pieces of it: neighbouring
//     lanes' are neighbours (f32, 8192 rows of 32 + 8 heads x 128: 65 us with two of 32 bytes, 55 so), and those that turn with each other are one
//     lane's, so a rotation needs no exchange between lanes; the norm's and the scale's reductions are butterflies over those 4 or 8 lanes.
//   * The angle of a far position does not fit 32 bits (pos = 10^5, f = 1: spacing 0.008): it is formed in f64 as a number of quarter turns, whose
//     fraction is exact to 2^-25 of a turn after the integer part is dropped.  A wave computes the row's <= 64 angles once, one per lane, and every head
//     it handles reads them from LDS.
#include "paged.h"

namespace oavsr {
namespace {

constexpr int kThreads = 256, kWaves = 4;

// 16 bytes that the kernel reads once: non-temporal, which leaves the caches to what is written and read next (norm + rotation of 4096 rows of 32 + 8 heads x
// 128 and a pass over its q: 28.3 us, without the hint 30.0, with one on the stores too 30.4; of 13500: 86, 95, 85.  Where the rows themselves still lie in
// the Infinity Cache the hint costs: 28.5 against 25.7).  16384 rows alone 57 us, 5.9 TB/s.
__device__ __forceinline__ Chunk16 load_once(const void* p) {
  Chunk16 c;
  c.v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return c;
}
// 16 values of a head as the 16-byte pieces at elements at[0], at[1], ...
template <typename T> struct Pieces {
  static constexpr int E = 16 / (int)sizeof(T), N = 16 / E;
  int at[N];
  __device__ __forceinline__ void load(const T* p, float* x) const {
#pragma unroll
    for (int k = 0; k < N; ++k) chunk_to_f32<T>(load_once(p + at[k]), x + k * E);
  }
  __device__ __forceinline__ void store(T* p, const float* x) const {
#pragma unroll
    for (int k = 0; k < N; ++k) *reinterpret_cast<Chunk16*>(p + at[k]) = chunk_from_f32<T>(x + k * E);
  }
};

// cos and sin of pos * f
__device__ __forceinline__ float2 turn_of(int pos, float f) {
  const double quarters = (double)pos * (double)f * 0.63661977236758134308;      // 2 / pi
  const double whole = __builtin_rint(quarters);
  float s, c;
  sincospif(0.5f * (float)(quarters - whole), &s, &c);                           // within an eighth of a turn of 0
  const int k = (int)((long long)whole & 3);
  const float c1 = (k & 1) ? s : c, s1 = (k & 1) ? c : s;
  return make_float2((k == 1 || k == 2) ? -c1 : c1, (k & 2) ? -s1 : s1);
}

// x / scale as an f32 that rounds to e4m3 as the exact quotient does: cut off towards zero, the lowest bit set where anything was cut (round to odd).
// Plain f32 division lands on the middle between two e4m3 values too often (bf16 inputs: 8-bit numerators) and then picks the even one on no ground.
// x - y * scale has to be exact: its lowest bit is scale's times y's, 2^-56 of scale for the smallest y that does not become zero (2^-10), and f32 ends at
// 2^-149.  So scale must not lie below 2^-93: the caller multiplies smaller ones, and their x, by a power of two.
__device__ __forceinline__ float quotient_odd(float x, float scale, float inv) {
  const float y0 = x * inv, y = fmaf(fmaf(-y0, scale, x), inv, y0);
  const float r = fmaf(-y, scale, x);                                            // exact
  const bool unlike = (__builtin_bit_cast(int, r) ^ __builtin_bit_cast(int, y)) < 0;
  const int over = (r != 0.f && unlike) ? 1 : 0;                                 // |y| > |x / scale|
  const int bits = (__builtin_bit_cast(int, y) - over) | (r != 0.f ? 1 : 0);
  return __builtin_bit_cast(float, bits);
}

struct Pages { PagedKv kv; PagedBatch b; };
struct NoPages {};

template <typename T, int HD, bool CACHE, bool F8>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(const QkRopeArgs p, const std::conditional_t<CACHE, Pages, NoPages> pages, int parts) {
  constexpr int LPH = HD / 16, HPW = 64 / LPH;       // lanes per head, heads per wave
  __shared__ float2 turns[kWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * kWaves + wave;
  const int row = (int)(task / parts), part = (int)(task - (int64_t)row * parts);
  if (row >= p.rows) {
    if constexpr (CACHE)
      if (wave == 0) report_bad_lengths(pages.kv, pages.b, lane);      // the workgroup behind the rows
    return;
  }

  int pos = 0, page = -1, off = 0;
  if constexpr (CACHE) {
    const PagedKv& kv = pages.kv;
    const PagedBatch& b = pages.b;
    const int s = wave_find_seq(b.cu_q, b.n_seqs, row, lane);
    const SeqInfo q = paged_seq(b, s);
    if (row < q.q0 || row >= q.q0 + q.nq) return;    // behind the last sequence, or of a skipped one
    pos = q.ctx - (q.nq - (row - q.q0));
    if (pos < 0) return;
    if (pos < b.max_ctx) {
      page = paged_page(kv, b, s, pos, page_shift_of(kv));
      off = pos & (kv.page_size - 1);
      if (page < 0 && lane == 0 && part == 0) paged_report(kv.status, kBadPage);
    }
    if (p.pos) pos = p.pos[row];
  } else if (p.inv_freq) pos = p.pos[row];

  const int rl = p.inv_freq ? p.rot_dim / 16 : 0;    // lanes of a head that rotate
  const int c = lane % LPH;
  float cs[8], sn[8];
  if (p.inv_freq) {
    if (lane < p.rot_dim / 2) {
      const float2 t = turn_of(pos, p.inv_freq[lane]);
      turns[wave][lane] = make_float2(t.x * p.rot_scale, t.y * p.rot_scale);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // The lane's pieces of a head: neighbouring lanes' are neighbours, and what turns with each other is one lane's.
  using P = Pieces<T>;
  P pc;
#pragma unroll
  for (int k = 0; k < P::N; ++k)
    pc.at[k] = c >= rl ? 16 * rl + P::E * (c - rl + k * (LPH - rl)) : p.interleaved ? P::E * (c + k * rl) : P::E * (c + k % (P::N / 2) * rl) + (k < P::N / 2 ? 0 : 8 * rl);
  if (c < rl) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 t = turns[wave][p.interleaved ? (pc.at[2 * i / P::E] + 2 * i % P::E) / 2 : pc.at[i / P::E] + i % P::E];
      cs[i] = t.x;
      sn[i] = t.y;
    }
  }

  const int heads = p.n_heads + p.n_kv_heads + (CACHE ? p.n_kv_heads : 0);
  for (int h0 = part * HPW; h0 < heads; h0 += parts * HPW) {
    const int h = h0 + lane / LPH;
    if (h >= heads) continue;                        // (whole heads: the lanes of a butterfly stay or leave together)
    const bool is_q = h < p.n_heads, is_v = h >= p.n_heads + p.n_kv_heads;
    if (CACHE && !is_q && page < 0) continue;
    const T* src = reinterpret_cast<const T*>(p.qkv) + (int64_t)row * p.ld + (int64_t)h * HD;
    float x[16];
    pc.load(src, x);
    if (!is_v) {
      if (p.q_gain) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, 64);
        const float r = 1.f / sqrtf(ss * (1.f / HD) + p.eps);
        const float* gain = is_q ? p.q_gain : p.k_gain;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f32x4 g = *reinterpret_cast<const f32x4*>(gain + pc.at[i / P::E] + i % P::E);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i + j] = x[i + j] * r * g[j];
        }
      }
      if (c < rl) {
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = x[2 * i], bb = x[2 * i + 1];
            x[2 * i] = a * cs[i] - bb * sn[i];
            x[2 * i + 1] = bb * cs[i] + a * sn[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = x[i], bb = x[8 + i];
            x[i] = a * cs[i] - bb * sn[i];
            x[8 + i] = bb * cs[i] + a * sn[i];
          }
        }
      }
    }
    if (is_q || !CACHE) {
      T* dst = is_q ? reinterpret_cast<T*>(p.q_out) + (int64_t)row * p.ldq + (int64_t)h * HD
                    : reinterpret_cast<T*>(p.k_out) + (int64_t)row * p.ldk + (int64_t)(h - p.n_heads) * HD;
      pc.store(dst, x);
    } else if constexpr (CACHE) {
      const PagedKv& kv = pages.kv;
      const int kh = is_v ? h - p.n_heads - p.n_kv_heads : h - p.n_heads;
      const int64_t tok = (int64_t)kh * kv.page_size + off;
      void* base = is_v ? kv.V : kv.K;
      if constexpr (F8) {
        float m = 0.f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) { m = fmaxf(m, fabsf(x[i])); odd |= !(fabsf(x[i]) <= 3.402823466e38f); }
        if (odd) m = INFINITY;
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const float scale = m == INFINITY ? NAN : fmaxf(m / 448.f, 1.17549435e-38f);
        const float up = scale < 0x1p-64f ? 0x1p64f : 1.f, qscale = scale * up, inv = 1.f / qscale;      // (exact, and the quotient's own)
        char* dst = reinterpret_cast<char*>(base) + (int64_t)page * kv.page_stride + tok * HD;
#pragma unroll
        for (int k = 0; k < P::N; ++k) {
          int w[P::E / 4];
#pragma unroll
          for (int j = 0; j < P::E / 4; ++j) {
            const float* y = x + P::E * k + 4 * j;
            int pk = 0;
            pk = __builtin_amdgcn_cvt_pk_fp8_f32(quotient_odd(y[0] * up, qscale, inv), quotient_odd(y[1] * up, qscale, inv), pk, false);
            pk = __builtin_amdgcn_cvt_pk_fp8_f32(quotient_odd(y[2] * up, qscale, inv), quotient_odd(y[3] * up, qscale, inv), pk, true);
            w[j] = pk;
          }
          if constexpr (P::E == 8) *reinterpret_cast<int2*>(dst + pc.at[k]) = make_int2(w[0], w[1]);
          else *reinterpret_cast<int*>(dst + pc.at[k]) = w[0];
        }
        if (c == 0) (is_v ? kv.v_scale : kv.k_scale)[(int64_t)page * kv.scale_stride + tok] = scale;
      } else {
        T* dst = reinterpret_cast<T*>(base) + (int64_t)page * kv.page_stride + tok * HD;
        pc.store(dst, x);
      }
    }
  }
}

// Cached rows back as values: a wave per row, head_dim / 16 lanes per head, keys' heads then values' heads.  HBM bound.
template <typename T, int HD, bool F8>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(const PagedKv kv, const PagedBatch b, T* __restrict__ k_out, int64_t ldk, T* __restrict__ v_out, int64_t ldv) {
  constexpr int LPH = HD / 16, HPW = 64 / LPH;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * kWaves + wave;
  if (task >= b.rows) {
    if (wave == 0) report_bad_lengths(kv, b, lane);      // the workgroup behind the rows
    return;
  }
  const int row = (int)task;
  const int s = wave_find_seq(b.cu_q, b.n_seqs, row, lane);
  const SeqInfo q = paged_seq(b, s);
  if (row < q.q0 || row >= q.q0 + q.nq) return;
  const int pos = q.ctx - (q.nq - (row - q.q0));
  if (pos < 0) return;
  int page = -1;
  if (pos < b.max_ctx) {
    page = paged_page(kv, b, s, pos, page_shift_of(kv));
    if (page < 0 && lane == 0) paged_report(kv.status, kBadPage);
  }
  const int off = pos & (kv.page_size - 1), c = lane % LPH;
  using P = Pieces<T>;
  P pc;
#pragma unroll
  for (int k = 0; k < P::N; ++k) pc.at[k] = P::E * (c + k * LPH);
  for (int h0 = 0; h0 < 2 * kv.n_kv_heads; h0 += HPW) {
    const int h = h0 + lane / LPH;
    if (h >= 2 * kv.n_kv_heads) continue;
    const bool is_v = h >= kv.n_kv_heads;
    const int kh = is_v ? h - kv.n_kv_heads : h;
    T* dst = is_v ? v_out : k_out;
    if (!dst) continue;
    dst += (int64_t)row * (is_v ? ldv : ldk) + (int64_t)kh * HD;
    float x[16];
    if (page < 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.f;
    } else {
      const int64_t tok = (int64_t)kh * kv.page_size + off;
      const void* base = is_v ? kv.V : kv.K;
      if constexpr (F8) {
        const char* src = reinterpret_cast<const char*>(base) + (int64_t)page * kv.page_stride + tok * HD;
        const float scale = (is_v ? kv.v_scale : kv.k_scale)[(int64_t)page * kv.scale_stride + tok];
#pragma unroll
        for (int k = 0; k < P::N; ++k)
          if constexpr (P::E == 8) {
            const auto w = __builtin_nontemporal_load(reinterpret_cast<const unsigned __attribute__((ext_vector_type(2)))*>(src + pc.at[k]));
            e4m3_to_f32(w[0], x + 8 * k);
            e4m3_to_f32(w[1], x + 8 * k + 4);
          } else e4m3_to_f32(__builtin_nontemporal_load(reinterpret_cast<const unsigned*>(src + pc.at[k])), x + 4 * k);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= scale;
      } else pc.load(reinterpret_cast<const T*>(base) + (int64_t)page * kv.page_stride + tok * HD, x);
    }
    pc.store(dst, x);
  }
}

__global__ void take_status_kernel(int* status, int* taken) { *taken = atomicExch(status, 0); }

int check_rope(const QkRopeArgs& a, const char* who) {
  OAVSR_REQUIRE(a.dtype == DT_F32 || a.dtype == DT_BF16, "%s: unknown dtype %d", who, a.dtype);
  OAVSR_REQUIRE(a.rows >= 0 && a.n_heads > 0 && a.n_kv_heads > 0, "%s: bad sizes (rows %d, heads %d / %d)", who, a.rows, a.n_heads, a.n_kv_heads);
  OAVSR_REQUIRE(a.head_dim == 64 || a.head_dim == 128, "%s: head_dim %d unsupported", who, a.head_dim);
  const int vec = a.dtype == DT_F32 ? 4 : 8;
  OAVSR_REQUIRE(a.ld >= (int64_t)(a.n_heads + 2 * a.n_kv_heads) * a.head_dim && a.ldq >= (int64_t)a.n_heads * a.head_dim, "%s: row strides shorter than the rows", who);
  OAVSR_REQUIRE(a.ld % vec == 0 && a.ldq % vec == 0 && a.ldk % vec == 0, "%s: rows must be 16-byte aligned", who);
  OAVSR_REQUIRE(a.rows == 0 || (a.qkv && a.q_out), "%s: null rows", who);
  OAVSR_REQUIRE((((uintptr_t)a.qkv | (uintptr_t)a.q_out | (uintptr_t)a.k_out | (uintptr_t)a.q_gain | (uintptr_t)a.k_gain) & 15) == 0, "%s: pointers must be 16-byte aligned", who);
  OAVSR_REQUIRE(!a.q_gain == !a.k_gain, "%s: gains for both queries and keys, or for neither", who);
  OAVSR_REQUIRE(!a.q_gain || a.eps >= 0.f, "%s: eps %g", who, a.eps);
  OAVSR_REQUIRE(!a.inv_freq || (a.rot_dim > 0 && a.rot_dim <= a.head_dim && a.rot_dim % 16 == 0), "%s: %d rotated dimensions (a multiple of 16 up to head_dim)", who, a.rot_dim);
  return 0;
}

// Waves per row.  One wave per row and pass of heads gives every head its own wave (few rows: a decode step's latency); from kManyRows rows on a wave takes
// all heads of its row and forms the row's angles once (kernel alone, 28 / 4 heads x 128 with norms, a wave per head / per row: 64 rows 2.9 / 4.9 us, 1024
// 5.2 / 7.4, 2047 10.7 / 9.9, 3500 15.5 / 14.1; 32 / 8 x 64: 2.6 / 3.4, 3.7 / 4.2, 6.4 / 6.9, 10.9 / 11.2; f32 16 / 2 x 128: 2.8 / 3.6, 5.1 / 6.2, 10.7 /
// 9.6, 14.8 / 14.3).
constexpr int kManyRows = 2048;
template <typename T, bool CACHE, bool F8>
int launch_rope_t(const QkRopeArgs& a, const PagedKv& kv, const PagedBatch& b, hipStream_t st) {
  const int hpw = 64 / (a.head_dim / 16), heads = a.n_heads + (CACHE ? 2 : 1) * a.n_kv_heads;
  const int parts = a.rows >= kManyRows ? 1 : ceil_div(heads, hpw);
  const int64_t blocks = ceil_div64((int64_t)a.rows * parts, kWaves) + (CACHE ? 1 : 0);
  OAVSR_REQUIRE(blocks * kThreads <= kMaxThreads, "paged: %d rows are too many for one launch", a.rows);
  std::conditional_t<CACHE, Pages, NoPages> pages;
  if constexpr (CACHE) { pages.kv = kv; pages.b = b; }
  if (a.head_dim == 64) hipLaunchKernelGGL((qk_rope_kernel<T, 64, CACHE, F8>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a, pages, parts);
  else hipLaunchKernelGGL((qk_rope_kernel<T, 128, CACHE, F8>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a, pages, parts);
  OAVSR_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename T, bool F8>
int launch_read_t(const PagedKv& kv, const PagedBatch& b, void* k_out, int64_t ldk, void* v_out, int64_t ldv, hipStream_t st) {
  const int64_t blocks = ceil_div64(b.rows, kWaves) + 1;
  OAVSR_REQUIRE(blocks * kThreads <= kMaxThreads, "paged_read: %d rows are too many for one launch", b.rows);
  const dim3 grid((unsigned)blocks);
  if (kv.head_dim == 64) hipLaunchKernelGGL((paged_read_kernel<T, 64, F8>), grid, dim3(kThreads), 0, st, kv, b, (T*)k_out, ldk, (T*)v_out, ldv);
  else hipLaunchKernelGGL((paged_read_kernel<T, 128, F8>), grid, dim3(kThreads), 0, st, kv, b, (T*)k_out, ldk, (T*)v_out, ldv);
  OAVSR_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace

int check_paged(const PagedKv& kv, const PagedBatch& b, const char* who) {
  OAVSR_REQUIRE(kv.dtype == DT_F32 || kv.dtype == DT_BF16, "%s: unknown dtype %d", who, kv.dtype);
  OAVSR_REQUIRE(kv.format == KV_SAME || kv.format == KV_E4M3, "%s: unknown cache format %d", who, kv.format);
  OAVSR_REQUIRE(kv.head_dim == 64 || kv.head_dim == 128, "%s: head_dim %d unsupported", who, kv.head_dim);
  OAVSR_REQUIRE(kv.page_size >= 16 && kv.page_size <= 256 && (kv.page_size & (kv.page_size - 1)) == 0, "%s: page_size %d (a power of two, 16 .. 256)", who, kv.page_size);
  OAVSR_REQUIRE(kv.n_kv_heads > 0 && kv.n_kv_heads <= 65535 && kv.n_pages >= 0, "%s: bad cache sizes (kv heads %d, pages %d)", who, kv.n_kv_heads, kv.n_pages);
  const int vec = kv.format == KV_E4M3 ? 16 : kv.dtype == DT_F32 ? 4 : 8;
  OAVSR_REQUIRE(kv.page_stride >= (int64_t)kv.n_kv_heads * kv.page_size * kv.head_dim && kv.page_stride % vec == 0, "%s: page stride %lld", who, (long long)kv.page_stride);
  OAVSR_REQUIRE(kv.n_pages == 0 || (kv.K && kv.V), "%s: null cache", who);
  OAVSR_REQUIRE((((uintptr_t)kv.K | (uintptr_t)kv.V | (uintptr_t)kv.k_scale | (uintptr_t)kv.v_scale) & 15) == 0, "%s: pointers must be 16-byte aligned", who);
  if (kv.format == KV_E4M3) {
    OAVSR_REQUIRE(kv.n_pages == 0 || (kv.k_scale && kv.v_scale), "%s: an 8-bit cache needs its scales", who);
    OAVSR_REQUIRE(kv.scale_stride >= (int64_t)kv.n_kv_heads * kv.page_size && kv.scale_stride % 4 == 0, "%s: scale stride %lld", who, (long long)kv.scale_stride);
  }
  OAVSR_REQUIRE(b.n_seqs >= 0 && b.rows >= 0 && b.max_q >= 0 && b.max_ctx >= 0, "%s: bad batch sizes (sequences %d, rows %d, max_q %d, max_ctx %d)", who, b.n_seqs, b.rows, b.max_q, b.max_ctx);
  OAVSR_REQUIRE(b.max_ctx <= (1 << 30), "%s: max_ctx %d", who, b.max_ctx);
  OAVSR_REQUIRE(b.n_seqs == 0 || (b.cu_q && b.ctx_len && (b.table || b.max_ctx == 0)), "%s: null batch", who);
  OAVSR_REQUIRE(b.ld_table >= 0 && b.ld_table <= (1ll << 31) && b.max_ctx <= b.ld_table * kv.page_size, "%s: a table of %lld pages does not hold max_ctx %d", who, (long long)b.ld_table, b.max_ctx);
  return 0;
}

int check_paged_host(const PagedKv& kv, const PagedBatch& b) {
  OAVSR_TRY(check_paged(kv, b, "paged_check_host"));
  int bits = 0;
  for (int s = 0; s < b.n_seqs; ++s) {
    const SeqInfo q = paged_seq(b, s);
    if (q.bad) bits |= kBadLength;
    const int n = q.nq == 0 ? 0 : q.ctx < b.max_ctx ? q.ctx : b.max_ctx;      // no launch reads the pages of a sequence that brings no rows, or is skipped
    for (int pos = 0; pos < n; pos += kv.page_size)
      if (paged_page(kv, b, s, pos, page_shift_of(kv)) < 0) bits |= kBadPage;
  }
  return bits;
}

int launch_paged_take_status(const PagedKv& kv, int* taken, hipStream_t st) {
  OAVSR_REQUIRE(kv.status && taken, "paged_take_status: null status");
  hipLaunchKernelGGL(take_status_kernel, dim3(1), dim3(1), 0, st, kv.status, taken);
  OAVSR_CHECK_HIP(hipGetLastError());
  return 0;
}

int launch_qk_norm_rope(const QkRopeArgs& a, hipStream_t st) {
  OAVSR_TRY(check_rope(a, "qk_norm_rope"));
  OAVSR_REQUIRE(a.ldk >= (int64_t)a.n_kv_heads * a.head_dim, "qk_norm_rope: row strides shorter than the rows");
  OAVSR_REQUIRE(a.rows == 0 || (a.k_out && (a.pos || !a.inv_freq)), "qk_norm_rope: null rows or positions");
  if (a.rows == 0) return 0;
  const PagedKv kv; const PagedBatch b;
  return a.dtype == DT_F32 ? launch_rope_t<float, false, false>(a, kv, b, st) : launch_rope_t<bf16_t, false, false>(a, kv, b, st);
}

int launch_paged_append(const PagedKv& kv, const PagedBatch& b, const QkRopeArgs& a, hipStream_t st) {
  OAVSR_TRY(check_paged(kv, b, "paged_append"));
  OAVSR_TRY(check_rope(a, "paged_append"));
  OAVSR_REQUIRE(a.rows == b.rows && a.dtype == kv.dtype && a.n_kv_heads == kv.n_kv_heads && a.head_dim == kv.head_dim,
                "paged_append: rows (%d, dtype %d, %d kv heads of %d) are not the batch's and the cache's (%d, dtype %d, %d of %d)", a.rows, a.dtype, a.n_kv_heads,
                a.head_dim, b.rows, kv.dtype, kv.n_kv_heads, kv.head_dim);
  if (nothing_to_do(kv, b)) return 0;
  if (kv.format == KV_E4M3) return a.dtype == DT_F32 ? launch_rope_t<float, true, true>(a, kv, b, st) : launch_rope_t<bf16_t, true, true>(a, kv, b, st);
  return a.dtype == DT_F32 ? launch_rope_t<float, true, false>(a, kv, b, st) : launch_rope_t<bf16_t, true, false>(a, kv, b, st);
}

int launch_paged_read(const PagedKv& kv, const PagedBatch& b, void* k_out, int64_t ldk, void* v_out, int64_t ldv, hipStream_t st) {
  OAVSR_TRY(check_paged(kv, b, "paged_read"));
  const int vec = kv.dtype == DT_F32 ? 4 : 8;
  const int64_t width = (int64_t)kv.n_kv_heads * kv.head_dim;
  OAVSR_REQUIRE((!k_out || (ldk >= width && ldk % vec == 0)) && (!v_out || (ldv >= width && ldv % vec == 0)), "paged_read: row strides %lld / %lld", (long long)ldk, (long long)ldv);
  OAVSR_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "paged_read: pointers must be 16-byte aligned");
  if (nothing_to_do(kv, b) || (b.rows && !k_out && !v_out)) return 0;      // (empty outputs have no address)
  if (kv.format == KV_E4M3) return kv.dtype == DT_F32 ? launch_read_t<float, true>(kv, b, k_out, ldk, v_out, ldv, st) : launch_read_t<bf16_t, true>(kv, b, k_out, ldk, v_out, ldv, st);
  return kv.dtype == DT_F32 ? launch_read_t<float, false>(kv, b, k_out, ldk, v_out, ldv, st) : launch_read_t<bf16_t, false>(kv, b, k_out, ldk, v_out, ldv, st);
}

}  // namespace oavsr
