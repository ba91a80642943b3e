// Attention of a batch's new tokens over a paged cache (include/omni_avsr.h: oavsr_op_paged_attention).
//
// A kv head serves a group of G = n_heads / n_kv_heads query heads, so the (new token, head of the group) pairs of a sequence are the rows of one problem:
// packed row r = token * G + head, all against the same keys and values, which a workgroup fetches once for its rows.  Softmax in one pass over the keys:
// running maximum m (nearly), sum l and O, rescaled when m is raised, in base 2 (scale * log2 e folded into the scores).
//
// S^T = K Q^T and O^T = V^T P^T on 16x16 or 32x32 matrix instructions: a lane then owns one query column, its softmax is lane-local but for two exchanges, and the
// accumulator registers of S^T are the B operand of the second product.
//
// Keys behind a sequence's context are never fetched.  A tile that some of the workgroup's rows see only in part (an edge tile) is masked; P = 0 there
// does not suffice, since 0 * NaN and 0 * infinity are NaN: where such a tile's values hold one (rare), its second product runs without those values, and
// they are then added for the rows that see them.
#include <algorithm>
#include "paged.h"

namespace oavsr {
namespace {

constexpr int kThreads = 256;
constexpr int KT = 64;                               // keys per tile

struct PagedAttnKArgs {
  PagedKv kv;
  PagedBatch b;
  const void* Q; int64_t ldq;
  void* O; int64_t ldo;
  float* lse;
  float scale2;                                      // scale * log2 e
  int n_heads, group, split, tiles;                  // split: keys per workgroup (0: all); tiles: of all sequences (bound)
  float* part;                                       // split: [splits][rows][n_heads][head_dim] O / l, then [splits][rows][n_heads] (m, l)
  float2* part_ml;
};

template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  static __device__ __forceinline__ void run(const Chunk16& a, const Chunk16& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
  }
};
template <> struct Mma16<float> {
  static __device__ __forceinline__ void run(const Chunk16& a, const Chunk16& b, f32x4& c) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a.v), fb = __builtin_bit_cast(f32x4, b.v);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[s], fb[s], c, 0, 0, 0);
  }
};

// The sequence and the first packed row of tile `tile` of ROWS packed rows, sequences' tiles one after the other: all lanes of a wave, 64 sequences a step.
struct TileAt { int seq, r0; };
template <int ROWS>
__device__ __forceinline__ TileAt wave_find_tile(const PagedBatch& b, int group, int tile, int lane) {
  int before = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += 64) {
    const int s = s0 + lane;
    const int64_t packed = s < b.n_seqs ? (int64_t)paged_seq(b, s).nq * group : 0;
    const int n = (int)((packed + ROWS - 1) / ROWS);
    int up = n;                                      // inclusive scan over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(up, o, 64); if (lane >= o) up += t; }
    const unsigned long long m = __builtin_amdgcn_ballot_w64(before + up > tile);
    if (m) {
      const int k = __builtin_ctzll(m);
      TileAt t;
      t.seq = s0 + k;
      t.r0 = (tile - before - (__shfl(up, k, 64) - __shfl(n, k, 64))) * ROWS;
      return t;
    }
    before += __shfl(up, 63, 64);
  }
  return TileAt{-1, 0};
}

__device__ __forceinline__ bool chunk_finite(const Chunk16& c, bf16_t) {
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (c.v[i] & 0x7f807f80u) + 0x00800080u;       // an exponent of all ones carries into the sign
  return (bad & 0x80008000u) == 0;
}
__device__ __forceinline__ bool chunk_finite(const Chunk16& c, float) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) ok = ok && (c.v[i] & 0x7f800000u) != 0x7f800000u;
  return ok;
}

__device__ __forceinline__ bool e4m3_finite(const Chunk16& c) {
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (c.v[i] & 0x7f7f7f7fu) + 0x01010101u;
  return (bad & 0x80808080u) == 0;
}
__device__ __forceinline__ bool is_finite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u; }
// zeros in the place of infinities and NaN
__device__ __forceinline__ bf16x8 finite_part(bf16x8 x) {
  u32x4 v = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((v[i] & 0x7f80u) == 0x7f80u) v[i] &= 0xffff0000u;
    if ((v[i] & 0x7f800000u) == 0x7f800000u) v[i] &= 0x0000ffffu;
  }
  return __builtin_bit_cast(bf16x8, v);
}

// Splits that hold keys of a row that sees `see` of them.  A row of one split (or none) is finished by that split's workgroup; the others leave partial results.
__device__ __forceinline__ int splits_of(const PagedAttnKArgs& p, int see) { return p.split && see > p.split ? (see - 1) / p.split + 1 : 1; }
// 1 / l of a finished row.  l = 0: no key is seen (zeros), or every seen one scores -infinity, of which the softmax is NaN.  (A split of such keys
// beside others is a partial result like any: no weight.)
__device__ __forceinline__ float inverse_sum(float l, bool sees_keys) { return l == 0.f ? (sees_keys ? NAN : 0.f) : 1.f / l; }

// ---- pieces of the streaming kernels -----------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

// max over lanes l, l ^ 16, l ^ 32, l ^ 48 / l, l ^ 32 by exchanges of the register file (no LDS round trip).  The second operand is kept apart from the
// first: the instruction swaps two registers.
__device__ __forceinline__ float max_xor32(float x) {
  float y = x;
  asm volatile("" : "+v"(y));
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float max_xor16_32(float x) {
  float y = x;
  asm volatile("" : "+v"(y));
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  return max_xor32(fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
}

// The running maximum need not be the maximum: any number near it keeps the exponentials in range and cancels in O / l.  It is raised, and O and l rescaled,
// only when some row's scores pass it, and then by kSlack more than they do, so that this is rare (with the exact maximum some row of a wave finds a new one in
// nearly every of the first dozens of tiles, and each time all of O is multiplied).  Weights stay between 2^-8, at the largest score, and 1: none
// takes a sum out of range that the values themselves do not.
constexpr float kSlack = 8.f;
__device__ __forceinline__ float raise_max(float& m_run, float mt) {
  const bool up = mt > m_run;                          // of this row alone: a row's bits do not follow the wave's other rows
  const float m_new = up ? mt + kSlack : m_run, alpha = up ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
  m_run = m_new;
  return alpha;
}

// Where 16-byte piece c of row r lies in an image of rows of RB bytes: c ^ swizzle.  LDS has 64 banks of 4 bytes, and serves 16 lanes of a 16-byte read at
// a time (of 16 rows that differ mod 16) or 32 of an 8-byte transposing one (4 neighbouring rows, 64 bytes of each).  So 16 rows have to put one piece into 16
// different places of 256 bytes, and 4 neighbouring rows their groups of four pieces into different quarters.
template <int RB> __device__ __forceinline__ constexpr int swizzle(int row) {
  return RB >= 256 ? ((row & 3) << 2) | ((row >> 2) & 3) : RB == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
}

// A page's number by scalar load (the table is the kernel's to read only), checked.
__device__ __forceinline__ int uniform_page(const PagedAttnKArgs& p, int seq, int key, int shift) {
  const int* t = p.b.table + (int64_t)seq * p.b.ld_table + (key >> shift);
  const int page = *reinterpret_cast<const __attribute__((address_space(4))) int*>((uintptr_t)t);
  return (unsigned)page < (unsigned)p.kv.n_pages ? page : -1;
}

// what a key row that is no key (behind the context, or of a page that is none) is fetched from: 16 rows
__device__ const Chunk16 kZeroRows[16 * 512 / 16] = {};

// f32 values: a lane reads four neighbours of a row at a time, one for each of four products, so that product dt of the O^T tiles holds the dimensions
// f32_dim(dt, 0 .. 15) in its rows.
__device__ __forceinline__ constexpr int f32_dim(int dt, int m) { return (dt >> 2) * 64 + 4 * m + (dt & 3); }
template <bool F8, int RB>
__device__ __forceinline__ void read_values4(const char* sV, int krow, int d, float (&out)[4]) {
  const int byte = d * (F8 ? 1 : 4);
  const char* at = sV + krow * RB + (((byte >> 4) ^ swizzle<RB>(krow)) << 4) + (byte & 15);
  if constexpr (F8) e4m3_to_f32(*reinterpret_cast<const unsigned*>(at), out);
  else chunk_to_f32<float>(*reinterpret_cast<const Chunk16*>(at), out);
}

__device__ __forceinline__ bf16x4 e4m3_to_bf16(unsigned w) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
  return bf16x4{a[0], a[1], b[0], b[1]};                // exact
}
// Transposing reads of four (two) 16-column blocks, waited for where they are made (the builtin makes the compiler wait for every LDS-DMA on its way
// first): lane 4 q + p of 16 gives the address of columns 4 p .. of row q and gets rows 0 .. 3 of its own column.  b16: two blocks of rows, AT bytes behind
// `at` and BT behind `bt`; b8: eight rows, lane 2 q + h giving bytes 8 h .. of row q.
template <int AT, int BT>
__device__ __forceinline__ void read_tr16_x4(const unsigned (&at)[4], const unsigned (&bt)[4], u32x4 (&out)[4]) {
  i32x2 a[4], b[4];
  asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %12 offset:%17\n\tds_read_b64_tr_b16 %2, %9 offset:%16\n\tds_read_b64_tr_b16 %3, %13 offset:%17\n\t"
               "ds_read_b64_tr_b16 %4, %10 offset:%16\n\tds_read_b64_tr_b16 %5, %14 offset:%17\n\tds_read_b64_tr_b16 %6, %11 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%17\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0]), "=&v"(b[0]), "=&v"(a[1]), "=&v"(b[1]), "=&v"(a[2]), "=&v"(b[2]), "=&v"(a[3]), "=&v"(b[3])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(bt[0]), "v"(bt[1]), "v"(bt[2]), "v"(bt[3]), "n"(AT), "n"(BT)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = u32x4{(unsigned)a[i][0], (unsigned)a[i][1], (unsigned)b[i][0], (unsigned)b[i][1]};
}
template <int AT, int BT>
__device__ __forceinline__ void read_tr16_x2(const unsigned (&at)[2], const unsigned (&bt)[2], u32x4 (&out)[2]) {
  i32x2 a[2], b[2];
  asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %6 offset:%9\n\tds_read_b64_tr_b16 %2, %5 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%9\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0]), "=&v"(b[0]), "=&v"(a[1]), "=&v"(b[1])
               : "v"(at[0]), "v"(at[1]), "v"(bt[0]), "v"(bt[1]), "n"(AT), "n"(BT)
               : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) out[i] = u32x4{(unsigned)a[i][0], (unsigned)a[i][1], (unsigned)b[i][0], (unsigned)b[i][1]};
}
__device__ __forceinline__ void read_tr8_x4(const unsigned (&at)[4], i32x2 (&out)[4]) {
  asm volatile("ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\tds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(out[0]), "=&v"(out[1]), "=&v"(out[2]), "=&v"(out[3])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
               : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)(lds_ptr)(void*)p; }

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// ---- few rows per sequence: single tokens ------------------------------------------------------------------------------------------------------
//
// A workgroup per (sequence, kv head, split of its keys) whose packed rows are the <= 16 columns of the matrix instructions.  HBM bound: G flop per byte of
// a bf16 cache, 2 G of an 8-bit one.  (Not f32 rows over 8 bits: the instructions work on 16 columns whatever G, 32 flop per byte, which the f32 pipe does
// at 4 TB/s, and the bytes are widened beside it: 97 sequences of up to 6000, 28 / 4 heads x 128: 167 us, 2.1 TB/s; f32 bytes, up to 3000: 130 us, 5.0.)  Each wave streams its own tiles of KT keys (wave, wave + NW, ...) through a private ring of NS tiles in LDS, fetched by LDS-DMA and
// awaited by counted vmcnt, so there is no barrier in the loop.  The 8 waves of a CU share its LDS: two tiles each where they are small, one where they are
// 16 KB (f32 or bf16 at head_dim 128), other waves' tiles being on their way while one is computed.  16 keys lie in one page, so an instruction's page is
// uniform: scalar loads, one page base per 16 keys.  The waves' (m, l, O) meet in LDS in wave order.  The cache is read once and the loads say so
// (non-temporal): 691 MB of 97 sequences 121 us, 5.7 TB/s with the join; without the hint 15 % more.
constexpr int kOnce = 2;                              // nt of a load to LDS
template <typename T, bool F8, int HD> struct DecodeShape {
  static constexpr int KT = sizeof(T) == 4 ? 16 : 32;                        // keys per wave tile
  static constexpr int RB = HD * (F8 ? 1 : (int)sizeof(T));                  // bytes of a cached row
  static constexpr int IMG = KT * RB, STAGE = 2 * IMG + (F8 ? 256 : 0);      // K image, V image, scales
};

template <typename T, bool F8, int HD, int NW, int NS>
__global__ __launch_bounds__(NW * 64, 2) void paged_decode_kernel(const PagedAttnKArgs p) {
  using Sh = DecodeShape<T, F8, HD>;
  constexpr int KT = Sh::KT, RB = Sh::RB, IMG = Sh::IMG, STAGE = Sh::STAGE, NCH = RB / 16;
  constexpr int RPI = 1024 / RB, NI = IMG / 1024;      // rows per DMA instruction, instructions per image
  constexpr int NSUB = KT / 16, NDT = HD / 16, NOFF = 16 / RPI;
  constexpr int VM = 2 * NI + (F8 ? 1 : 0);
  constexpr int RS = 17, JOIN = HD * RS * 4 + 128;      // (m, l, O) of the wave, O's dimensions RS floats apart: lanes that read every fourth meet other banks
  constexpr int RING = STAGE * NS > JOIN ? STAGE * NS : JOIN;      // the ring, afterwards those
  static_assert(VM * (NS - 1) <= 63, "vmcnt");
  __shared__ __attribute__((aligned(1024))) char smem[NW * RING];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 15, g = lane >> 4;
  const int G = p.group, KV = p.kv.n_kv_heads, kvh = blockIdx.x % KV, unit = blockIdx.x / KV, split = unit / p.tiles, seq = unit - split * p.tiles;
  const SeqInfo sq = paged_seq(p.b, seq);
  if (sq.bad && tid == 0) paged_report(p.kv.status, kBadLength);
  const int packed = sq.nq * G;
  if (packed == 0) return;
  const int first_pos = sq.ctx - sq.nq, kmax = min(sq.ctx, p.b.max_ctx);
  const int kend_all = max(0, min(first_pos + sq.nq, kmax));
  const int kbeg = p.split ? split * p.split : 0;
  if (split > 0 && kbeg >= kend_all) return;
  const int kend = p.split ? min(kend_all, kbeg + p.split) : kend_all;
  char* ring = smem + wave * RING;

  // ---- the ring
  const int shift = page_shift_of(p.kv);
  int loff[NOFF];                                      // byte offset of this lane's piece inside the rows of an instruction
#pragma unroll
  for (int j = 0; j < NOFF; ++j) {
    const int r = j * RPI + lane / NCH;
    loff[j] = (lane / NCH) * RB + (((lane % NCH) ^ swizzle<RB>(r)) << 4);
  }
  const char* Kb = reinterpret_cast<const char*>(p.kv.K);
  const char* Vb = reinterpret_cast<const char*>(p.kv.V);
  const int64_t page_bytes = p.kv.page_stride * (F8 ? 1 : (int64_t)sizeof(T));
  bool bad_page = false;
  auto issue = [&](int kt0, int slot) __attribute__((always_inline)) {
    char* dst = ring + slot * STAGE;
    int page[NSUB];
#pragma unroll
    for (int j = 0; j < NSUB; ++j) {
      const int key = kt0 + 16 * j;
      page[j] = -1;
      if (key < kend) { page[j] = uniform_page(p, seq, key, shift); bad_page |= page[j] < 0; }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int j = i * RPI / 16, key = kt0 + 16 * j;
      const int64_t at = (int64_t)page[j] * page_bytes + ((int64_t)kvh * p.kv.page_size + (key & (p.kv.page_size - 1)) + (i * RPI) % 16) * RB;
      const char* k = page[j] < 0 ? reinterpret_cast<const char*>(kZeroRows) : Kb + at;
      const char* v = page[j] < 0 ? reinterpret_cast<const char*>(kZeroRows) : Vb + at;
      __builtin_amdgcn_global_load_lds((global_ptr)(k + loff[i % NOFF]), (lds_ptr)(dst + i * 1024), 16, 0, kOnce);
      __builtin_amdgcn_global_load_lds((global_ptr)(v + loff[i % NOFF]), (lds_ptr)(dst + IMG + i * 1024), 16, 0, kOnce);
    }
    if constexpr (F8) {                                // lanes 0 .. KT - 1: the keys' scales, then the values'
      const int l = lane & (2 * KT - 1), key = kt0 + (l & (KT - 1));
      const int pg = NSUB == 1 || (l & 16) == 0 ? page[0] : page[NSUB - 1];
      const float* base = l < KT ? p.kv.k_scale : p.kv.v_scale;
      const float* src = pg < 0 ? reinterpret_cast<const float*>(kZeroRows)
                                : base + (int64_t)pg * p.kv.scale_stride + (int64_t)kvh * p.kv.page_size + (key & (p.kv.page_size - 1));
      __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(dst + 2 * IMG), 4, 0, 0);
    }
  };
  const int first = kbeg + wave * KT, step = NW * KT;
  const int ntile = first < kend ? (kend - first + step - 1) / step : 0;

  // ---- queries: lane = packed row qi, in the element order of the K fragments
  const int r = min(qi, packed - 1), tok = r / G, head = kvh * G + (r - tok * G);
  const int64_t row = sq.q0 + tok;
  const int see = min(first_pos + tok + 1, kmax), see_min = min(first_pos + 1, kmax);
  const T* qp = reinterpret_cast<const T*>(p.Q) + row * p.ldq + (int64_t)head * HD;
  constexpr int NQ = F8 ? HD / 64 : RB / 64;           // 16-byte pieces of a cached row per lane
  constexpr int QE = F8 ? 16 : 16 / (int)sizeof(T);    // elements of a piece
  constexpr int QC = QE * (int)sizeof(T) / 16;
  Chunk16 qf[NQ][QC];
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int e = 0; e < QC; ++e) qf[b][e] = reinterpret_cast<const Chunk16*>(qp + (b * 4 + g) * QE)[e];
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (i < ntile) issue(first + i * step, i);
  // (waited for here, once: inside the loop the wait for them would be one for the ring too)
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int e = 0; e < QC; ++e) asm volatile("" : "+v"(qf[b][e].v));

  auto dim_of = [](int dt, int m) { return sizeof(T) == 4 ? f32_dim(dt, m) : dt * 16 + m; };      // of row m of O^T tile dt
  f32x4 o[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  int slot = 0;                                        // of tile t
  auto tile = [&](int t, auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;      // some row does not see the whole tile, or it ends behind the context
    const int kt0 = first + t * step;
    if (ntile - t >= NS) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VM * (NS - 1)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    char* sK = ring + slot * STAGE;
    char* sV = sK + IMG;
    const float* sc = reinterpret_cast<const float*>(sK + 2 * IMG);
    if (MASKED && kt0 + KT > kend) {                   // rows behind the context: whatever the page holds there must not meet a zero
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (kt0 + i * RPI + lane / NCH >= kend) reinterpret_cast<Chunk16*>(sV + i * 1024)[lane].v = u32x4{0u, 0u, 0u, 0u};
    }

    f32x4 s[NSUB];
    float mt = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NSUB; ++kt) {
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int krow = kt * 16 + qi;
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const Chunk16 kc = *reinterpret_cast<const Chunk16*>(sK + krow * RB + (((b * 4 + g) ^ swizzle<RB>(krow)) << 4));
        if constexpr (!F8) Mma16<T>::run(kc, qf[b][0], s[kt]);
        else if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(e4m3_to_bf16(kc.v[2 * hf]), e4m3_to_bf16(kc.v[2 * hf + 1])), __builtin_bit_cast(bf16x8, qf[b][hf].v), s[kt], 0, 0, 0);
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float x[4];
            e4m3_to_f32(kc.v[w], x);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], __builtin_bit_cast(f32x4, qf[b][w].v)[e], s[kt], 0, 0, 0);
          }
        }
      }
      f32x4 ks = f32x4{p.scale2, p.scale2, p.scale2, p.scale2};
      if constexpr (F8) ks *= *reinterpret_cast<const f32x4*>(sc + kt * 16 + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = s[kt][i] * ks[i];
        if (MASKED && kt0 + kt * 16 + 4 * g + i >= see) v = -INFINITY;
        s[kt][i] = v;
        mt = fmaxf(mt, v);
      }
    }
    mt = max_xor16_32(mt);
    if (__builtin_amdgcn_ballot_w64(mt > m_run) != 0ull) {
      const float alpha = raise_max(m_run, mt);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < NDT; ++i) o[i] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < NSUB; ++kt) {
      f32x4 vs = f32x4{1.f, 1.f, 1.f, 1.f};
      if constexpr (F8) vs = *reinterpret_cast<const f32x4*>(sc + KT + kt * 16 + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float e = __builtin_amdgcn_exp2f(s[kt][i] - m_use);
        sum += e;
        if constexpr (F8) e *= vs[i];
        if (MASKED && kt0 + kt * 16 + 4 * g + i >= see) e = 0.f;
        s[kt][i] = e;
      }
    }
    l_run += sum;

    // infinities and NaN among the values of an edge tile (of several new tokens: a later one's)
    bool odd = false;
    auto v_at = [&](int krow, int d) -> float {
      const int byte = d * (F8 ? 1 : (int)sizeof(T));
      const char* at = sV + krow * RB + (((byte >> 4) ^ swizzle<RB>(krow)) << 4) + (byte & 15);
      if constexpr (F8) { float x[4]; e4m3_to_f32(*reinterpret_cast<const unsigned char*>(at), x); return x[0]; }
      else return to_f32(*reinterpret_cast<const T*>(at));
    };
    if constexpr (MASKED) {
      bool ok = true;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const Chunk16 c = reinterpret_cast<const Chunk16*>(sV + i * 1024)[lane];
        if constexpr (F8) ok = ok && e4m3_finite(c);
        else ok = ok && chunk_finite(c, T());
      }
      odd = __builtin_amdgcn_ballot_w64(!ok) != 0ull;
    }

    if constexpr (sizeof(T) == 2) {
      // The weights as sums of two numbers: a rounding less, and products are not what is short here.  The first is cut off, so that the second has its
      // sign, and the second is never zero beside one that is not: an infinite value stays what it is.
      bf16x8 pf, pl;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = s[i >> 2][i & 3], hi = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, e) & 0xffff0000u);
        pf[i] = (bf16_t)hi;
        pl[i] = (bf16_t)fmaxf(e - hi, e * 0x1p-30f);
      }
      const unsigned vb = lds_address(sV);
#pragma unroll
      for (int d4 = 0; d4 < NDT; d4 += 4) {
        unsigned at[4];
        bf16x8 vf[4];
        if constexpr (F8) {
          const int rr = qi >> 1, krow = rr < 4 ? 4 * g + rr : 12 + 4 * g + rr;
          i32x2 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) at[j] = vb + krow * RB + (((d4 + j) ^ swizzle<RB>(krow)) << 4) + (qi & 1) * 8;
          read_tr8_x4(at, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[j] = join(e4m3_to_bf16((unsigned)w[j][0]), e4m3_to_bf16((unsigned)w[j][1]));
        } else {
          const int qq = qi >> 2, pp = qi & 3, krow = 4 * g + qq;
          u32x4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) at[j] = vb + krow * RB + ((((d4 + j) * 2 + (pp >> 1)) ^ swizzle<RB>(krow)) << 4) + (pp & 1) * 8;
          read_tr16_x4<0, 16 * RB>(at, at, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[j] = __builtin_bit_cast(bf16x8, w[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (MASKED && odd) vf[j] = finite_part(vf[j]);
          o[d4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[j], pf, o[d4 + j], 0, 0, 0);
          o[d4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[j], pl, o[d4 + j], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          float vv[4];
          read_values4<F8, RB>(sV, 4 * g + i, 64 * j + 4 * qi, vv);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (MASKED && odd && !is_finite(vv[w])) vv[w] = 0.f;
            o[4 * j + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[w], s[0][i], o[4 * j + w], 0, 0, 0);
          }
        }
    }
    if (MASKED && __builtin_expect(odd, 0)) {
      for (int k = 0; k < KT; ++k) {
        float e = 0.f;
#pragma unroll
        for (int kt = 0; kt < NSUB; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((k & 3) == i && (k >> 4) == kt) e = s[kt][i];
        e = __shfl(e, ((k >> 2) & 3) * 16 + qi, 64);
        if (kt0 + k < see)
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float vv = v_at(k, dim_of(dt, 4 * g + q));
              if (!is_finite(vv)) o[dt][q] += e * vv;
            }
      }
    }
    if (t + NS < ntile) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this tile has been read
      issue(kt0 + NS * step, slot);
    }
    slot = slot == NS - 1 ? 0 : slot + 1;
  };
  const int t_full = see_min >= first + KT ? min(ntile, (see_min - first - KT) / step + 1) : 0;
  int t = 0;
  for (; t < t_full; ++t) tile(t, std::false_type{});
  for (; t < ntile; ++t) tile(t, std::true_type{});
  if (bad_page && lane == 0) paged_report(p.kv.status, kBadPage);

  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  // ---- the waves' partial results, joined in wave order
  float* so = reinterpret_cast<float*>(ring);          // [HD][RS] O^T, then [16] m, [16] l
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) so[dim_of(dt, 4 * g + i) * RS + qi] = o[dt][i];
  if (g == 0) { so[HD * RS + qi] = m_run; so[HD * RS + 16 + qi] = l_run; }
  __syncthreads();
  for (int i = tid; i < packed * (HD / 4); i += NW * 64) {
    const int pr = i / (HD / 4), d0 = (i - pr * (HD / 4)) * 4, ptok = pr / G, phead = kvh * G + (pr - ptok * G);
    float m = -INFINITY, l = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* x = reinterpret_cast<const float*>(smem + w * RING);
      m = fmaxf(m, x[HD * RS + pr]);
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* x = reinterpret_cast<const float*>(smem + w * RING);
      const float f = __builtin_amdgcn_exp2f(x[HD * RS + pr] - mu);
      l = fmaf(f, x[HD * RS + 16 + pr], l);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(f, x[(d0 + j) * RS + pr], acc[j]);
    }
    const int64_t prow = sq.q0 + ptok;
    const int psee = min(first_pos + ptok + 1, kmax), n = splits_of(p, psee);
    if (split >= n) continue;
    const float inv = inverse_sum(l, n == 1 && psee > 0);
    if (n > 1) {
      const int64_t at = ((int64_t)split * p.b.rows + prow) * p.n_heads + phead;
      if (d0 == 0) p.part_ml[at] = make_float2(m, l);
      *reinterpret_cast<f32x4*>(p.part + at * HD + d0) = acc * inv;
    } else {
      if (p.lse && d0 == 0) p.lse[prow * p.n_heads + phead] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
      T* O = reinterpret_cast<T*>(p.O) + prow * p.ldo + (int64_t)phead * HD + d0;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<bf16x4*>(O) = bf16x4{(bf16_t)(acc[0] * inv), (bf16_t)(acc[1] * inv), (bf16_t)(acc[2] * inv), (bf16_t)(acc[3] * inv)};
      else *reinterpret_cast<f32x4*>(O) = acc * inv;
    }
  }
}

// ---- many rows per sequence: chunks and whole prompts, bf16 ------------------------------------------------------------------------------------
//
// A workgroup of 4 (8) waves takes 128 (256) packed rows of a (sequence, kv head), 32 per wave, on 32x32x16 matrix instructions; tiles of 64 keys are shared by
// the waves.  Bound by the matrix pipe and the vector issue of the softmax together (per tile and wave at head_dim 128: 32 products of 32 cycles, about 200
// vector instructions of 4; at head_dim 64 half the products for the same softmax).  A tile travels through registers into one of two LDS images, one barrier per
// tile, its loads issued a tile ahead: each thread widens 8-bit bytes once for all waves, and the transposing reads of the values, which the compiler would
// hold behind every LDS-DMA in flight, can be requested before the exponentials that hide them (533 us with LDS-DMA and a ring of three, 515 so).
// The kv head is the fastest part of a workgroup's number: workgroups of one kv head then share an XCD (8 of them take the numbers in turn), and its L2
// serves their common keys.  Sequences' tiles are taken from the last to the first, so that a prompt's long rows are not what remains at the end (a prompt
// of 8192, 32 / 8 heads: 642 us in rising order, 576 so, 549 with 256 rows; one level of all sequences at a time: the same there, but 4 chunks over
// 12000 keys 704 us against 447, since the L2 no longer sees a sequence's keys once).  2048 new tokens over 16384: 500 us, 1030 TFLOP/s.
// A wave skips the tiles none of its rows sees, and masks only those that some row sees in part, in a loop of its own.
// A weight is one bf16 number (in 8 bits behind its product with the value's scale): a rounding of 2^-8 of each weight, relative, that the kernel of
// single tokens does not make, and the result's error against 64 bits is 0.0023 where its own rounding alone makes 0.0017.  Two numbers, as there, are half again
// as many products and cost a third: 2048 over 16384 683 us against 514, in 8 bits 743 against 574, 4 prompts of 4096 at 32 / 8 heads x 64 463 against 357.
template <bool F8, int HD, int NW>
__global__ __launch_bounds__(NW * 64, HD == 64 ? 3 : 2) void paged_chunk_kernel(const PagedAttnKArgs p) {
  constexpr int ROWS = NW * 32, RB = HD * 2, IMG = KT * RB, NSTAGE = 2, STAGE = 2 * IMG + (F8 ? 2 * KT * 4 : 0);
  constexpr int NDS = HD / 16, NDT = HD / 32;
  constexpr int CB = F8 ? HD : RB, FB = CB / NW, RW = KT / NW, NC = FB / 16;      // bytes of a cached row, of them per thread; rows per wave; 16-byte loads
  static_assert(FB >= 16, "a thread loads whole 16-byte pieces");
  __shared__ __attribute__((aligned(1024))) char smem[NSTAGE * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ql = lane & 31, h = lane >> 5;
  const int G = p.group, KV = p.kv.n_kv_heads;
  const int kvh = blockIdx.x % KV, unit = blockIdx.x / KV, split = unit / p.tiles;
  if (blockIdx.x == 0 && wave == 0) report_bad_lengths(p.kv, p.b, lane);
  const TileAt at = wave_find_tile<ROWS>(p.b, G, p.tiles - 1 - (unit - split * p.tiles), lane);      // the last rows, which see the most keys, first
  if (at.seq < 0) return;
  const int seq = __builtin_amdgcn_readfirstlane(at.seq), r0 = __builtin_amdgcn_readfirstlane(at.r0);
  const SeqInfo sq = paged_seq(p.b, seq);
  const int packed = sq.nq * G;
  const int first_pos = sq.ctx - sq.nq, kmax = min(sq.ctx, p.b.max_ctx);
  const int kend_all = max(0, min(first_pos + (min(r0 + ROWS, packed) - 1) / G + 1, kmax));
  const int kbeg = p.split ? split * p.split : 0;
  if (split > 0 && kbeg >= kend_all) return;
  const int kend = p.split ? min(kend_all, kbeg + p.split) : kend_all;
  const int ntile = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;

  // ---- this wave's rows
  const int w0 = r0 + wave * 32;                       // first packed row
  const bool rows_here = w0 < packed;
  const int r = w0 + ql, rc = min(r, packed - 1), tok = rc / G, head = kvh * G + (rc - tok * G);
  const int64_t row = sq.q0 + tok;
  const int see = min(first_pos + tok + 1, kmax);
  const int see_min = min(first_pos + min(w0, packed - 1) / G + 1, kmax), see_max = rows_here ? min(first_pos + min(w0 + 31, packed - 1) / G + 1, kmax) : 0;

  // ---- tiles
  const int shift = page_shift_of(p.kv), pmask = p.kv.page_size - 1;
  const char* Kb = reinterpret_cast<const char*>(p.kv.K);
  const char* Vb = reinterpret_cast<const char*>(p.kv.V);
  const int64_t page_bytes = p.kv.page_stride * (F8 ? 1 : 2);
  bool bad_page = false;
  int page;                                            // of this wave's rows of the next tile to fetch
  auto next_page = [&](int kt0) __attribute__((always_inline)) {
    const int key = kt0 + wave * RW;
    page = -1;
    if (key < kend) { page = uniform_page(p, seq, key, shift); bad_page |= page < 0; }
  };
  const char* zero = reinterpret_cast<const char*>(kZeroRows);
  // thread = FB bytes of a row of both images, NW threads a row; 8 bits: the first 2 RW lanes of a wave the scales of its rows
  struct Raw { u32x4 k[NC], v[NC]; float scale; };
  auto fetch = [&](int kt0, Raw& x) __attribute__((always_inline)) {
    const int key = kt0 + wave * RW + lane / NW;
    const bool ok = page >= 0 && key < kend;
    const int64_t at = (int64_t)page * page_bytes + ((int64_t)kvh * p.kv.page_size + (key & pmask)) * CB + (lane % NW) * 16;
    const char *k = ok ? Kb + at : zero, *v = ok ? Vb + at : zero;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      x.k[c] = *reinterpret_cast<const u32x4*>(k + c * NW * 16);
      x.v[c] = *reinterpret_cast<const u32x4*>(v + c * NW * 16);
    }
    if constexpr (F8) {
      const int skey = kt0 + wave * RW + lane % RW;
      const int64_t sat = (int64_t)page * p.kv.scale_stride + (int64_t)kvh * p.kv.page_size + (skey & pmask);
      const float* sp = page >= 0 && skey < kend ? ((lane & RW) ? p.kv.v_scale : p.kv.k_scale) + sat : reinterpret_cast<const float*>(zero);
      x.scale = *sp;
    }
  };
  auto store = [&](const Raw& x, int slot) __attribute__((always_inline)) {
    char* dst = smem + slot * STAGE;
    const int lrow = wave * RW + lane / NW;
    auto put = [&](char* img, int c, u32x4 w) { *reinterpret_cast<u32x4*>(img + lrow * RB + ((c ^ swizzle<RB>(lrow)) << 4)) = w; };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int at = lane % NW + c * NW;
      if constexpr (F8) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          put(dst, 2 * at + w, __builtin_bit_cast(u32x4, join(e4m3_to_bf16(x.k[c][2 * w]), e4m3_to_bf16(x.k[c][2 * w + 1]))));
          put(dst + IMG, 2 * at + w, __builtin_bit_cast(u32x4, join(e4m3_to_bf16(x.v[c][2 * w]), e4m3_to_bf16(x.v[c][2 * w + 1]))));
        }
      } else {
        put(dst, at, x.k[c]);
        put(dst + IMG, at, x.v[c]);
      }
    }
    if (F8 && lane < 2 * RW) reinterpret_cast<float*>(dst + 2 * IMG)[((lane & RW) ? KT : 0) + wave * RW + lane % RW] = (lane & RW) ? x.scale : x.scale * p.scale2;
  };

  // Q^T fragments (B operand: lane = row ql, k-group h): step ds covers d = 16 ds + 8 h .. + 7
  Chunk16 qf[NDS];
  {
    const char* qp = reinterpret_cast<const char*>(reinterpret_cast<const bf16_t*>(p.Q) + row * p.ldq + (int64_t)head * HD);
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) qf[ds] = *reinterpret_cast<const Chunk16*>(qp + ds * 32 + h * 16);
  }
  Raw raw;
  next_page(kbeg);
  if (ntile > 0) { fetch(kbeg, raw); next_page(kbeg + KT); store(raw, 0); }
  if (ntile > 1) { fetch(kbeg + KT, raw); next_page(kbeg + 2 * KT); }
#pragma unroll
  for (int ds = 0; ds < NDS; ++ds) asm volatile("" : "+v"(qf[ds].v));      // waited for here, not in the loop

  // LDS offsets inside a stage.  K (A operand): row ql (+ 32), piece 2 ds + h.  V^T (transposing reads: 16 lanes fetch 4 rows x 16 columns): row 4 h + qq
  // (+ 16 per step, + 8), piece 4 dt + 2 d16 + (pp >> 1); of the row offsets the swizzle sees only the 8, as a bit of its own.
  unsigned kbase[NDS], vbase[NDT];
  {
    const unsigned s0 = lds_address(smem);
    const int qi = lane & 15, d16 = (lane >> 4) & 1, qq = qi >> 2, pp = qi & 3, vrow = 4 * h + qq;
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) kbase[ds] = ql * RB + (((ds * 2 + h) ^ swizzle<RB>(ql)) << 4);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) vbase[dt] = s0 + IMG + vrow * RB + (((dt * 4 + d16 * 2 + (pp >> 1)) ^ swizzle<RB>(vrow)) << 4) + (pp & 1) * 8;
  }

  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  auto compute = [&](int kt0, unsigned so, auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const float* sc = reinterpret_cast<const float*>(smem + so + 2 * IMG);
    unsigned kat[NDS];
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) kat[ds] = so + kbase[ds];
    f32x16 s[2];
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t2][e] = 0.f;
#pragma unroll
      for (int ds = 0; ds < NDS; ++ds) {
        const Chunk16 kf = *reinterpret_cast<const Chunk16*>(smem + kat[ds] + t2 * 32 * RB);
        s[t2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf.v), __builtin_bit_cast(bf16x8, qf[ds].v), s[t2], 0, 0, 0);
      }
    }
    // softmax: the lane's keys are 32 t2 + 8 i + 4 h + r
    if constexpr (F8) {
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 ks = *reinterpret_cast<const f32x4*>(sc + 32 * t2 + 8 * i + 4 * h);
#pragma unroll
          for (int q = 0; q < 4; ++q) s[t2][4 * i + q] *= ks[q];
        }
    }
    int key0 = kt0 + 4 * h;
    if constexpr (MASKED) {
      asm volatile("" : "+v"(key0));
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + 32 * t2 + 8 * (e >> 2) + (e & 3) >= see) s[t2][e] = -INFINITY;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
      for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[t2][e]);
    mt = max_xor32(mt);
    if constexpr (!F8) mt *= p.scale2;                 // scale > 0
    if (__builtin_amdgcn_ballot_w64(mt > m_run) != 0ull) {
      const float alpha = raise_max(m_run, mt);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
    const float nm = m_run == -INFINITY ? 0.f : -m_run;
    bool odd = false;                                  // infinities or NaN among the values of a masked tile
    if constexpr (MASKED) {
      bool ok = true;
#pragma unroll
      for (int i = 0; i < IMG / 1024; ++i) ok = ok && chunk_finite(reinterpret_cast<const Chunk16*>(smem + so + IMG + i * 1024)[lane], bf16_t());
      odd = __builtin_amdgcn_ballot_w64(!ok) != 0ull;
    }
    float sum[2] = {0.f, 0.f};
    auto weights = [&](auto T2) __attribute__((always_inline)) {
      constexpr int t2 = decltype(T2)::value;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float ev = __builtin_amdgcn_exp2f(F8 ? s[t2][e] + nm : fmaf(s[t2][e], p.scale2, nm));
        s[t2][e] = ev;
        sum[e & 1] += ev;
      }
      if constexpr (F8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 vs = *reinterpret_cast<const f32x4*>(sc + KT + 32 * t2 + 8 * i + 4 * h);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            s[t2][4 * i + q] *= vs[q];
            if (MASKED && key0 + 32 * t2 + 8 * i + q >= see) s[t2][4 * i + q] = 0.f;
          }
        }
      }
    };
    if constexpr (MASKED) {
      static_for<0, 2>(weights);
      if (__builtin_expect(odd, 0)) {
        const char* sV = smem + so + IMG;
        for (int k = 0; k < KT; ++k) {
          float pe = 0.f;
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (k >> 5 == t2 && ((k >> 3) & 3) == e >> 2 && (k & 3) == (e & 3)) pe = s[t2][e];
          pe = __shfl(pe, ((k >> 2) & 1) * 32 + ql, 64);
          if (kt0 + k < see)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                const int byte = (32 * dt + 8 * (q >> 2) + 4 * h + (q & 3)) * 2;
                const float vv = (float)*reinterpret_cast<const bf16_t*>(sV + k * RB + (((byte >> 4) ^ swizzle<RB>(k)) << 4) + (byte & 15));
                if (!is_finite(vv)) o[dt][q] += pe * vv;
                if (q & 1) asm volatile("" ::: "memory");      // few of these reads at a time: this code must not cost the common path registers
              }
        }
      }
    }
    unsigned vat[NDT], vat8[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) { vat[dt] = vbase[dt] + so; vat8[dt] = vat[dt] ^ (swizzle<RB>(8) << 4); }
    static_for<0, 2>([&](auto T2) __attribute__((always_inline)) {
      constexpr int t2 = decltype(T2)::value;
      // the values of 32 keys are on their way while the weights are formed
      s16x4 va[2][NDT], vb[2][NDT];
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          va[sl][dt] = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vat[dt] + (2 * t2 + sl) * 16 * RB)));
          vb[sl][dt] = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vat8[dt] + ((2 * t2 + sl) * 16 + 8) * RB)));
        }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!MASKED) weights(T2);
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {
        bf16x8 pf;
#pragma unroll
        for (int q = 0; q < 8; ++q) pf[q] = (bf16_t)s[t2][8 * sl + q];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          bf16x8 vf = join(__builtin_bit_cast(bf16x4, va[sl][dt]), __builtin_bit_cast(bf16x4, vb[sl][dt]));
          if (MASKED && odd) vf = finite_part(vf);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf, o[dt], 0, 0, 0);
        }
      }
    });
    l_run += sum[0] + sum[1];
  };

  int slot = 0;                                        // of tile t
  auto tile = [&](int t, auto masked_tag) __attribute__((always_inline)) {
    const int kt0 = kbeg + t * KT;
    __syncthreads();
    if (t + 1 < ntile) store(raw, 1 - slot);           // (that slot held tile t - 1: every wave is past it)
    if (t + 2 < ntile) { fetch(kt0 + 2 * KT, raw); next_page(kt0 + 3 * KT); }
    if (!decltype(masked_tag)::value || kt0 < see_max) compute(kt0, slot * STAGE, masked_tag);
    slot = slot == NSTAGE - 1 ? 0 : slot + 1;
  };
  // two loops, each with one body: as two branches of one loop the bodies' accumulators met in copies of all of them
  const int t_full = rows_here ? min(ntile, max(0, see_min - kbeg) / KT) : 0;
  int t = 0;
  for (; t < t_full; ++t) tile(t, std::false_type{});
  for (; t < ntile; ++t) tile(t, std::true_type{});
  if (bad_page && lane == 0) paged_report(p.kv.status, kBadPage);

  if (r >= packed) return;
  float l = l_run;
  l += __shfl_xor(l, 32, 64);
  const int n = splits_of(p, see);
  if (split >= n) return;
  const float inv = inverse_sum(l, n == 1 && see > 0);
  if (n > 1) {
    const int64_t at_row = ((int64_t)split * p.b.rows + row) * p.n_heads + head;
    if (h == 0) p.part_ml[at_row] = make_float2(m_run, l);
    float* P = p.part + at_row * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(P + 32 * dt + 8 * i + 4 * h) = f32x4{o[dt][4 * i] * inv, o[dt][4 * i + 1] * inv, o[dt][4 * i + 2] * inv, o[dt][4 * i + 3] * inv};
    return;
  }
  if (p.lse && h == 0) p.lse[row * p.n_heads + head] = l == 0.f ? -INFINITY : (m_run + log2f(l)) * 0.69314718055994530942f;
  bf16_t* O = reinterpret_cast<bf16_t*>(p.O) + row * p.ldo + (int64_t)head * HD;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x4 w;
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = (bf16_t)(o[dt][4 * i + q] * inv);
      *reinterpret_cast<bf16x4*>(O + 32 * dt + 8 * i + 4 * h) = w;
    }
}

// ---- many rows per sequence, f32 ---------------------------------------------------------------------------------------------------------------
//
// The exact-f32 mode: a workgroup of 4 waves takes 64 packed rows, 16 per wave, on 16x16x4 matrix instructions, which bound it (32 cycles for 2048 flop;
// reading the fragments from LDS takes a quarter of that).  Tiles of 32 keys (f32 at head_dim 128: 16, so that three workgroups share a CU: 256 new tokens of 8
// sequences over 4096, 28 / 4 heads 1060 us, 110 TFLOP/s, against 1100 with two of 32 keys) through a ring that the waves share, as cached bytes: 8-bit ones
// are widened where they are read.
template <bool F8, int HD>
__global__ __launch_bounds__(256, 3) void paged_rows_f32_kernel(const PagedAttnKArgs p) {
  constexpr int NW = 4, ROWS = NW * 16, KT = !F8 && HD == 128 ? 16 : 32, NKT = KT / 16, RB = HD * (F8 ? 1 : 4), IMG = KT * RB, STAGE = 2 * IMG + (F8 ? 256 : 0), NSTAGE = F8 ? 4 : 3;
  constexpr int NCH = RB / 16, RPI = 1024 / RB, NI = IMG / 1024, NSEG = 2 * NI / NW, VM = NSEG + (F8 ? 1 : 0), NDT = HD / 16, NQ = HD / (F8 ? 64 : 16);
  __shared__ __attribute__((aligned(1024))) char smem[NSTAGE * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 15, g = lane >> 4;
  const int G = p.group, KV = p.kv.n_kv_heads;
  const int kvh = blockIdx.x % KV, unit = blockIdx.x / KV, split = unit / p.tiles;
  if (blockIdx.x == 0 && wave == 0) report_bad_lengths(p.kv, p.b, lane);
  const TileAt at = wave_find_tile<ROWS>(p.b, G, p.tiles - 1 - (unit - split * p.tiles), lane);      // the last rows, which see the most keys, first
  if (at.seq < 0) return;
  const int seq = __builtin_amdgcn_readfirstlane(at.seq), r0 = __builtin_amdgcn_readfirstlane(at.r0);
  const SeqInfo sq = paged_seq(p.b, seq);
  const int packed = sq.nq * G;
  const int first_pos = sq.ctx - sq.nq, kmax = min(sq.ctx, p.b.max_ctx);
  const int kend_all = max(0, min(first_pos + (min(r0 + ROWS, packed) - 1) / G + 1, kmax));
  const int kbeg = p.split ? split * p.split : 0;
  if (split > 0 && kbeg >= kend_all) return;
  const int kend = p.split ? min(kend_all, kbeg + p.split) : kend_all;
  const int ntile = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;

  const int w0 = r0 + wave * 16;
  const bool rows_here = w0 < packed;
  const int see_min = min(first_pos + min(w0, packed - 1) / G + 1, kmax), see_max = rows_here ? min(first_pos + min(w0 + 15, packed - 1) / G + 1, kmax) : 0;
  const int rc = min(w0 + qi, packed - 1), tok = rc / G, head = kvh * G + (rc - tok * G), see = min(first_pos + tok + 1, kmax);
  const int64_t row = sq.q0 + tok;
  Chunk16 qf[NQ][F8 ? 4 : 1];
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int e = 0; e < (F8 ? 4 : 1); ++e)
      qf[b][e] = reinterpret_cast<const Chunk16*>(reinterpret_cast<const float*>(p.Q) + row * p.ldq + (int64_t)head * HD)[(b * 4 + g) * (F8 ? 4 : 1) + e];

  const int shift = page_shift_of(p.kv), pmask = p.kv.page_size - 1;
  const int64_t page_bytes = p.kv.page_stride * (F8 ? 1 : 4);
  const char* zero = reinterpret_cast<const char*>(kZeroRows);
  bool bad_page = false;
  int page[NKT];                                         // of the two halves of the next tile to fetch
  auto next_pages = [&](int kt0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NKT; ++j) {
      page[j] = -1;
      if (kt0 + 16 * j < kend) { page[j] = uniform_page(p, seq, kt0 + 16 * j, shift); bad_page |= page[j] < 0; }
    }
  };
  auto issue = [&](int kt0, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NSEG; ++j) {
      const int u = wave + NW * j, i = u % NI, key = kt0 + i * RPI, lrow = i * RPI + lane / NCH, pg = i * RPI < 16 ? page[0] : page[NKT - 1];
      const char* base = reinterpret_cast<const char*>(u < NI ? p.kv.K : p.kv.V);
      const char* src = pg < 0 ? zero : base + (int64_t)pg * page_bytes + ((int64_t)kvh * p.kv.page_size + (key & pmask)) * RB;
      if (kt0 + KT > kend && kt0 + lrow >= kend) src = zero;      // behind the context: whatever the page holds must not meet a zero
      src += (lane / NCH) * RB + (((lane % NCH) ^ swizzle<RB>(lrow)) << 4);
      __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(smem + slot * STAGE + u * 1024), 16, 0, 0);
    }
    if constexpr (F8) {                                // (every wave the same 64 scales: one instruction, and the same count of them in every wave)
      const int key = kt0 + (lane & 31), pg = (lane & 16) ? page[NKT - 1] : page[0];
      const float* base = lane < 32 ? p.kv.k_scale : p.kv.v_scale;
      const float* src = pg < 0 || key >= kend ? reinterpret_cast<const float*>(zero)
                                               : base + (int64_t)pg * p.kv.scale_stride + (int64_t)kvh * p.kv.page_size + (key & pmask);
      __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(smem + slot * STAGE + 2 * IMG), 4, 0, 0);
    }
    next_pages(kt0 + KT);
  };
  next_pages(kbeg);
#pragma unroll
  for (int i = 0; i < NSTAGE - 1; ++i)
    if (i < ntile) issue(kbeg + i * KT, i);
#pragma unroll
  for (int b = 0; b < NQ; ++b)
#pragma unroll
    for (int e = 0; e < (F8 ? 4 : 1); ++e) asm volatile("" : "+v"(qf[b][e].v));      // waited for here, not in the loop

  f32x4 o[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  auto compute = [&](int kt0, const char* sK, auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const char* sV = sK + IMG;
    const float* sc = reinterpret_cast<const float*>(sK + 2 * IMG);

    f32x4 s[2];                                        // (of a 16-key tile: the two halves of its sums)
    s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      Chunk16 kc[NKT];
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt) kc[kt] = *reinterpret_cast<const Chunk16*>(sK + (kt * 16 + qi) * RB + (((b * 4 + g) ^ swizzle<RB>(qi)) << 4));      // (+ 16 rows: the same swizzle)
#pragma unroll
      for (int w = 0; w < (F8 ? 4 : 1); ++w) {
        float x[NKT][4];
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt) {
          if constexpr (F8) e4m3_to_f32(kc[kt].v[w], x[kt]);
          else chunk_to_f32<float>(kc[kt], x[kt]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt) {          // chains of products that do not wait for each other
            const int c = NKT == 2 ? kt : e & 1;
            s[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[kt][e], __builtin_bit_cast(f32x4, qf[b][w].v)[e], s[c], 0, 0, 0);
          }
      }
    }
    if constexpr (NKT == 1) s[0] += s[1];
    auto v_at = [&](int krow, int d) -> float {
      const int byte = d * (F8 ? 1 : 4);
      const char* a = sV + krow * RB + (((byte >> 4) ^ swizzle<RB>(krow)) << 4) + (byte & 15);
      if constexpr (F8) { float x[4]; e4m3_to_f32(*reinterpret_cast<const unsigned char*>(a), x); return x[0]; }
      else return *reinterpret_cast<const float*>(a);
    };
    bool odd = false;                                  // infinities or NaN among the values of a masked tile
    if constexpr (MASKED) {
      bool ok = true;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const Chunk16 x = reinterpret_cast<const Chunk16*>(sV + i * 1024)[lane];
        if constexpr (F8) ok = ok && e4m3_finite(x);
        else ok = ok && chunk_finite(x, float());
      }
      odd = __builtin_amdgcn_ballot_w64(!ok) != 0ull;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      f32x4 ks = f32x4{p.scale2, p.scale2, p.scale2, p.scale2};
      if constexpr (F8) ks *= *reinterpret_cast<const f32x4*>(sc + kt * 16 + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = s[kt][i] * ks[i];
        if (MASKED && kt0 + kt * 16 + 4 * g + i >= see) v = -INFINITY;
        s[kt][i] = v;
        mt = fmaxf(mt, v);
      }
    }
    mt = max_xor16_32(mt);
    if (__builtin_amdgcn_ballot_w64(mt > m_run) != 0ull) {
      const float alpha = raise_max(m_run, mt);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < NDT; ++i) o[i] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      f32x4 vs = f32x4{1.f, 1.f, 1.f, 1.f};
      if constexpr (F8) vs = *reinterpret_cast<const f32x4*>(sc + 32 + kt * 16 + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float e = __builtin_amdgcn_exp2f(s[kt][i] - m_use);
        sum += e;
        if constexpr (F8) e *= vs[i];
        if (MASKED && kt0 + kt * 16 + 4 * g + i >= see) e = 0.f;
        s[kt][i] = e;
      }
    }
    l_run += sum;
    if (MASKED && __builtin_expect(odd, 0)) {
      for (int k = 0; k < KT; ++k) {
        float e = 0.f;
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((k & 3) == i && (k >> 4) == kt) e = s[kt][i];
        e = __shfl(e, ((k >> 2) & 3) * 16 + qi, 64);
        if (kt0 + k < see)
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float vv = v_at(k, f32_dim(dt, 4 * g + q));
              if (!is_finite(vv)) o[dt][q] += e * vv;
              if (q & 1) asm volatile("" ::: "memory");
            }
      }
    }
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          float vv[4];
          read_values4<F8, RB>(sV, kt * 16 + 4 * g + i, 64 * j + 4 * qi, vv);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (MASKED && odd && !is_finite(vv[w])) vv[w] = 0.f;
            o[4 * j + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[w], s[kt][i], o[4 * j + w], 0, 0, 0);
          }
        }
  };
  int slot = 0;                                        // of tile t
  auto tile = [&](int t, auto masked_tag) __attribute__((always_inline)) {
    const int kt0 = kbeg + t * KT;
    if (t + NSTAGE - 1 <= ntile) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VM * (NSTAGE - 2)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + NSTAGE - 1 < ntile) issue(kt0 + (NSTAGE - 1) * KT, slot == 0 ? NSTAGE - 1 : slot - 1);      // (that slot held tile t - 1: every wave is past it)
    if (!decltype(masked_tag)::value || kt0 < see_max) compute(kt0, smem + slot * STAGE, masked_tag);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this wave has read the tile when it meets the next barrier
    slot = slot == NSTAGE - 1 ? 0 : slot + 1;
  };
  const int t_full = rows_here ? min(ntile, max(0, see_min - kbeg) / KT) : 0;
  int t = 0;
  for (; t < t_full; ++t) tile(t, std::false_type{});
  for (; t < ntile; ++t) tile(t, std::true_type{});
  if (bad_page && lane == 0) paged_report(p.kv.status, kBadPage);

  if (w0 + qi >= packed) return;
  float l = l_run;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const int n = splits_of(p, see);
  if (split >= n) return;
  const float inv = inverse_sum(l, n == 1 && see > 0);
  float* O = reinterpret_cast<float*>(p.O) + row * p.ldo + (int64_t)head * HD;
  if (n > 1) {
    const int64_t at_row = ((int64_t)split * p.b.rows + row) * p.n_heads + head;
    if (g == 0) p.part_ml[at_row] = make_float2(m_run, l);
    O = p.part + at_row * HD;
  } else if (p.lse && g == 0) p.lse[row * p.n_heads + head] = l == 0.f ? -INFINITY : (m_run + log2f(l)) * 0.69314718055994530942f;
#pragma unroll
  for (int j = 0; j < HD / 64; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4*>(O + f32_dim(4 * j, 4 * g + q)) = f32x4{o[4 * j][q], o[4 * j + 1][q], o[4 * j + 2][q], o[4 * j + 3][q]} * inv;
}

// Joins the splits of the rows whose keys lie in more than one:  out = sum_z w_z O_z / sum_z w_z,  w_z = l_z 2^(m_z - max m).  NG groups of HD / 4 threads share
// a (row, head), each taking every NG-th split, joined in LDS in a fixed order: all of a workgroup's where the splits are many, and one where they are
// at most kFewSplits, with all of them on their way at once.  A row of few splits gets the same bits from both.
constexpr int kFewSplits = 8;
template <typename T, int HD, int NG>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnKArgs p) {
  constexpr int TPG = HD / 4, PER = kThreads / (TPG * NG);      // (row, head) pairs per workgroup: heads of one row
  __shared__ __attribute__((aligned(16))) float acc_s[NG == 1 ? 1 : kThreads / TPG][HD];
  __shared__ float m_s[kThreads / TPG], l_s[kThreads / TPG];
  const int tid = threadIdx.x, lane = tid & 63;
  const int hb = (p.n_heads + PER - 1) / PER, row = blockIdx.x / hb;
  const int sub = tid / TPG, grp = sub % NG, head = (blockIdx.x - row * hb) * PER + sub / NG, d0 = (tid % TPG) * 4;
  const int seq = wave_find_seq(p.b.cu_q, p.b.n_seqs, row, lane);
  const SeqInfo sq = paged_seq(p.b, seq);
  if (row < sq.q0 || row >= sq.q0 + sq.nq) return;
  const int n = splits_of(p, min(sq.ctx - sq.nq + (row - sq.q0) + 1, min(sq.ctx, p.b.max_ctx)));
  if (n <= 1) return;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  if (NG == 1 && head < p.n_heads) {
    float2 ml[kFewSplits];
    f32x4 x[kFewSplits];
#pragma unroll
    for (int z = 0; z < kFewSplits; ++z) {
      ml[z] = make_float2(-INFINITY, 0.f);
      x[z] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (z < n) {
        const int64_t at = ((int64_t)z * p.b.rows + row) * p.n_heads + head;
        ml[z] = p.part_ml[at];
        x[z] = *reinterpret_cast<const f32x4*>(p.part + at * HD + d0);
      }
    }
#pragma unroll
    for (int z = 0; z < kFewSplits; ++z) m = fmaxf(m, ml[z].x);
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int z = 0; z < kFewSplits; ++z) {
      const float w = __builtin_amdgcn_exp2f(ml[z].x - mu);
      l = fmaf(w, ml[z].y, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, ml[z].y * x[z][e], acc[e]);
    }
  }
  if (NG > 1 && head < p.n_heads) {
#pragma unroll 2
    for (int z = grp; z < n; z += NG) {
      const int64_t at = ((int64_t)z * p.b.rows + row) * p.n_heads + head;
      const float2 ml = p.part_ml[at];
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.part + at * HD + d0);
      const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
      const float w0 = __builtin_amdgcn_exp2f(m - mu), w1 = __builtin_amdgcn_exp2f(ml.x - mu) * ml.y;
      l = l * w0 + w1;
      m = mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = acc[e] * w0 + w1 * x[e];
    }
  }
  if constexpr (NG > 1) {
    if (d0 == 0) { m_s[sub] = m; l_s[sub] = l; }
    *reinterpret_cast<f32x4*>(&acc_s[sub][d0]) = acc;
    __syncthreads();
    if (grp > 0) return;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) m = fmaxf(m, m_s[sub + j]);
    const float mu = m == -INFINITY ? 0.f : m;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const float w = __builtin_amdgcn_exp2f(m_s[sub + j] - mu);
      l = fmaf(w, l_s[sub + j], l);
      const f32x4 x = *reinterpret_cast<const f32x4*>(&acc_s[sub + j][d0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, x[e], acc[e]);
    }
  }
  if (head >= p.n_heads) return;
  const float inv = inverse_sum(l, true);
  if (p.lse && d0 == 0) p.lse[(int64_t)row * p.n_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
  T* O = reinterpret_cast<T*>(p.O) + (int64_t)row * p.ldo + (int64_t)head * HD + d0;
  if constexpr (sizeof(T) == 2) *reinterpret_cast<bf16x4*>(O) = bf16x4{(bf16_t)(acc[0] * inv), (bf16_t)(acc[1] * inv), (bf16_t)(acc[2] * inv), (bf16_t)(acc[3] * inv)};
  else *reinterpret_cast<f32x4*>(O) = acc * inv;
}

int cu_count() {
  static const int n = [] { int d = 0, c = 256; (void)hipGetDevice(&d); (void)hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, d); return c; }();
  return n;
}

// How a call is laid out: by its sizes' bounds alone, since the lengths are on the device.
//   decode  up to 16 packed rows per sequence: the streaming kernel.  Workgroups of eight waves where a CU is there for each sequence and kv head, of four,
//           two side by side, where there are more of those (97 rows of 6000 keys, 4 kv heads 121 us, with eight waves 126, two 124; 100 ragged up to 4000
//           in 8 bits 52, 58, 69).
//   chunk   more.  f32: 64 packed rows a workgroup, three side by side.  bf16: 128, two side by side; at head_dim 128 256 rows, which fetch the keys once for
//           twice as many, unless most sequences bring far less than the longest (2048 new tokens over 16384, 32 / 8 heads: 500 us against 543; a prompt
//           of 8192 549 against 578; 8 ragged prompts up to 2000 208 against 218; 6 chunks up to 512 among 24 single tokens 186 against 167).
//   split   keys per workgroup.  Single tokens: as many splits as leave each its CU, two also where they are a little too many (1 sequence of 40000, 8 kv
//           heads: 33 us, in two rounds of them 42; 3 of 131072: 129 against 138; 20 ragged up to 8000: 66 against 76), none for few keys; where
//           workgroups are many, two rounds of them.  bf16 chunks of an even batch: what costs least by the estimate below -- rounds, or for prompts, whose
//           rows see more and more keys and start with the most, the mean share -- with 150 keys' time for the join's launch and 200 for each split's
//           partial results (1024 new tokens over 32768, 40 / 8 heads, 160 workgroups: 8 splits 703 us, unsplit 873; 2048 over 6144 of 3 sequences, 28 / 4
//           heads: unsplit 484, 3 splits 561; 2 prompts of 6000: unsplit 539, 5 splits 743).  The others: two rounds, since a ragged batch's longest
//           sequence else runs on alone (24 sequences, 5 of them chunks of up to 701: 76 us, unsplit 131); in bf16 with a last split that is short, so that
//           only the longest sequences have one and the short work comes last (2.6 % over 15 ragged batches, 0 .. 13 %; the 256 keys' grain already does
//           that to f32's many short ones).  Ragged prompts that fill the chip are not split, as even ones are not (3 of up to 2000, 28 / 4 heads: 117
//           us, in two 141; 4 of up to 1000 56 against 65; 12 of up to 700, 16 / 16 heads x 64: 24 against 33; 8 of up to 1500, 14 / 2 heads x 64: 44
//           against 45; 5 of up to 2000 in 8 bits 157 against 155).  Over far longer contexts they are, for the longest one's sake (4 chunks of up to
//           1000 over 6000: 214 us, unsplit 240; over 3000, where the two rules meet, 118 and 115).
//           At head_dim 64 three workgroups fit side by side, and two are counted: three would take a chunk of 1024 over 32768 at 14 / 2 heads from 226
//           us to 216 in 8 bits, but one of 512 over 8000 at 32 / 8 from 59 to 62, and 24 sequences with 5 chunks in 8 bits from 75 to 82.
struct Plan { int64_t tiles; int split, splits, nw; bool decode; };
Plan plan_of(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a) {
  Plan pl;
  const int G = a.n_heads / kv.n_kv_heads, cus = cu_count();
  const int64_t packed = (int64_t)b.rows * G;
  const bool f32 = kv.dtype == DT_F32;
  const bool even = b.rows >= (int64_t)b.n_seqs * b.max_q;      // all sequences bring max_q tokens
  pl.decode = (int64_t)b.max_q * G <= 16;
  pl.nw = !pl.decode && !f32 && kv.head_dim == 128 && (int64_t)b.max_q * G > 128 && 2ll * b.rows >= (int64_t)b.n_seqs * b.max_q ? 8 : 4;
  const int rows = f32 ? 64 : 32 * pl.nw;
  pl.tiles = pl.decode ? b.n_seqs : std::min<int64_t>(packed / rows + b.n_seqs, b.n_seqs * ceil_div64((int64_t)b.max_q * G, rows));
  const int64_t wgs = std::max<int64_t>(1, pl.tiles * kv.n_kv_heads);
  const int64_t slots = (int64_t)cus * (pl.decode ? 2 : f32 ? 3 : pl.nw == 8 ? 1 : 2);      // workgroups side by side
  pl.split = a.split_keys;
  if (!pl.split) {
    const int64_t up = ceil_div64(2 * slots, wgs), least = f32 ? 256 : 512;
    int64_t tenths = 10 * up;                                   // of as many splits
    if (pl.decode) {
      if (b.max_ctx <= 2 * least) tenths = 10;
      else if (wgs <= cus) tenths = 2 * wgs > cus && 3 * wgs <= 2 * cus ? 20 : 10 * (cus / wgs);
    } else if (!f32 && !even) {
      if (wgs >= slots && 2ll * b.max_ctx <= 5ll * b.max_q) tenths = 10;
      tenths -= tenths > 10 ? 2 : 0;
    } else if (!f32) {
      // in keys: whole rounds, or the mean share and half a workgroup more, whichever is less, and never less than one workgroup; partial results
      const double full = (double)wgs / slots, share = full * (b.max_ctx - 0.5 * std::min(b.max_q, b.max_ctx));
      double best = 1e30;
      for (int i = 1; i <= 64; ++i) {
        const int64_t keys = ceil_div64(ceil_div64(b.max_ctx, i), 256) * 256;
        if (i > 1 && keys < least) break;
        const double half = 0.5 * (i == 1 ? std::max(0, b.max_ctx - b.max_q) : keys);
        const double cost = std::max((double)keys, std::min((double)(ceil_div64(wgs * i, slots) * keys), share + half)) + (i > 1 ? 150 + 200 * i * full : 0);
        if (cost < best) best = cost, tenths = 10 * i;
      }
    }
    pl.split = (int)std::max<int64_t>(least, ceil_div64(ceil_div64(10ll * b.max_ctx, tenths), 256) * 256);
  }
  pl.splits = (int)ceil_div64(b.max_ctx, pl.split);
  if (pl.splits <= 1) pl.split = 0, pl.splits = 1;
  if (pl.decode) pl.nw = a.split_keys || wgs > cus ? 4 : 8;      // (a pinned split: the waves' shares too)
  return pl;
}
uint64_t workspace_of(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a, const Plan& pl) {
  return pl.split ? (uint64_t)pl.splits * b.rows * a.n_heads * (kv.head_dim + 2) * 4 : 0;
}
int check_attn(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a) {
  OAVSR_TRY(check_paged(kv, b, "paged_attention"));
  OAVSR_REQUIRE(a.n_heads > 0 && a.n_heads % kv.n_kv_heads == 0, "paged_attention: heads %d not a multiple of kv heads %d", a.n_heads, kv.n_kv_heads);
  OAVSR_REQUIRE(a.scale > 0.f && a.scale < INFINITY, "paged_attention: scale %g", a.scale);
  OAVSR_REQUIRE(a.split_keys >= 0 && a.split_keys % 256 == 0, "paged_attention: split_keys %d (a multiple of 256)", a.split_keys);
  const int64_t packed = (int64_t)b.rows * a.n_heads;
  OAVSR_REQUIRE(packed < (1ll << 30), "paged_attention: %d rows of %d heads are too many for one launch", b.rows, a.n_heads);
  return 0;
}

template <typename T, bool F8, int HD>
int launch_t(const PagedAttnKArgs& k, const Plan& pl, hipStream_t st) {
  const dim3 line((unsigned)(pl.tiles * k.kv.n_kv_heads * pl.splits));
  if (pl.decode) {
    constexpr int FIT = 17 * 1024 / DecodeShape<T, F8, HD>::STAGE, NS = FIT > 2 ? 2 : FIT;      // a ring of at most 17 KB a wave, 8 waves a CU
    if (pl.nw == 4) hipLaunchKernelGGL((paged_decode_kernel<T, F8, HD, 4, NS>), line, dim3(256), 0, st, k);
    else hipLaunchKernelGGL((paged_decode_kernel<T, F8, HD, 8, NS>), line, dim3(512), 0, st, k);
  } else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((paged_rows_f32_kernel<F8, HD>), line, dim3(256), 0, st, k);
  else {
    if constexpr (HD == 128) {
      if (pl.nw == 8) hipLaunchKernelGGL((paged_chunk_kernel<F8, HD, 8>), line, dim3(512), 0, st, k);
    }
    if (pl.nw == 4) hipLaunchKernelGGL((paged_chunk_kernel<F8, HD, 4>), line, dim3(256), 0, st, k);
  }
  OAVSR_CHECK_HIP(hipGetLastError());
  if (pl.split && k.b.rows) {
    constexpr int ALL = kThreads / (HD / 4);
    static_assert(ALL >= kFewSplits, "groups");
    if (pl.splits > kFewSplits) hipLaunchKernelGGL((paged_merge_kernel<T, HD, ALL>), dim3((unsigned)((int64_t)k.b.rows * k.n_heads)), dim3(kThreads), 0, st, k);
    else hipLaunchKernelGGL((paged_merge_kernel<T, HD, 1>), dim3((unsigned)((int64_t)k.b.rows * ceil_div(k.n_heads, ALL))), dim3(kThreads), 0, st, k);
    OAVSR_CHECK_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace

int64_t paged_attention_workspace(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a) {
  OAVSR_TRY(check_attn(kv, b, a));
  return (int64_t)workspace_of(kv, b, a, plan_of(kv, b, a));
}

int launch_paged_attention(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a, hipStream_t st) {
  OAVSR_TRY(check_attn(kv, b, a));
  const int vec = kv.dtype == DT_F32 ? 4 : 8;
  const int64_t width = (int64_t)a.n_heads * kv.head_dim;
  OAVSR_REQUIRE(a.ldq >= width && a.ldo >= width && a.ldq % vec == 0 && a.ldo % vec == 0, "paged_attention: row strides %lld / %lld", (long long)a.ldq, (long long)a.ldo);
  OAVSR_REQUIRE(b.rows == 0 || (a.Q && a.O), "paged_attention: null rows");
  OAVSR_REQUIRE((((uintptr_t)a.Q | (uintptr_t)a.O | (uintptr_t)a.workspace) & 15) == 0, "paged_attention: pointers must be 16-byte aligned");
  if (nothing_to_do(kv, b)) return 0;
  const Plan pl = plan_of(kv, b, a);
  const uint64_t need = workspace_of(kv, b, a, pl);
  OAVSR_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "paged_attention: a workspace of %llu bytes is needed, %llu given", (unsigned long long)need,
                (unsigned long long)(a.workspace ? a.workspace_bytes : 0));
  const int64_t joins = pl.split ? (int64_t)b.rows * (pl.splits > kFewSplits ? a.n_heads : ceil_div(a.n_heads, kThreads / (kv.head_dim / 4))) : 0;
  OAVSR_REQUIRE(pl.splits <= 65535 && pl.tiles * kv.n_kv_heads * pl.splits <= kMaxThreads / (pl.nw * 64) && joins <= kMaxThreads / kThreads,
                "paged_attention: too many workgroups (%lld tiles, %d splits, %d rows)", (long long)pl.tiles, pl.splits, b.rows);
  PagedAttnKArgs k;
  k.kv = kv; k.b = b; k.Q = a.Q; k.ldq = a.ldq; k.O = a.O; k.ldo = a.ldo; k.lse = a.lse; k.scale2 = a.scale * 1.44269504088896340736f;
  k.n_heads = a.n_heads; k.group = a.n_heads / kv.n_kv_heads; k.split = pl.split; k.tiles = (int)pl.tiles;
  k.part = reinterpret_cast<float*>(a.workspace);
  k.part_ml = reinterpret_cast<float2*>(k.part + (size_t)pl.splits * b.rows * a.n_heads * kv.head_dim);
  const bool f8 = kv.format == KV_E4M3;
  if (kv.dtype == DT_F32) {
    if (kv.head_dim == 64) return f8 ? launch_t<float, true, 64>(k, pl, st) : launch_t<float, false, 64>(k, pl, st);
    return f8 ? launch_t<float, true, 128>(k, pl, st) : launch_t<float, false, 128>(k, pl, st);
  }
  if (kv.head_dim == 64) return f8 ? launch_t<bf16_t, true, 64>(k, pl, st) : launch_t<bf16_t, false, 64>(k, pl, st);
  return f8 ? launch_t<bf16_t, true, 128>(k, pl, st) : launch_t<bf16_t, false, 128>(k, pl, st);
}

}  // namespace oavsr
