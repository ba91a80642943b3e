// Attention of a batch's new tokens over a paged cache (include/omni_avsr.h: oavsr_op_paged_attention).
//
// A kv head serves a group of G = n_heads / n_kv_heads query heads, so the (new token, head of the group) pairs of a sequence are the rows of one problem:
// packed row r = token * G + head, all against the same keys and values, which a workgroup fetches once for its rows.  Softmax in one pass over the keys:
// running maximum m, sum l and O, rescaled when m grows, in base 2 (scale * log2 e folded into the scores).
//
// S^T = K Q^T and O^T = V^T P^T on 16x16 matrix instructions: a lane then owns one query column, its softmax is lane-local but for two exchanges, and the
// accumulator registers of S^T are the B operand of the second product.
//
// Keys behind a sequence's context are never fetched.  A tile that some of the workgroup's rows see only in part (an edge tile) is masked; P = 0 there
// does not suffice, since 0 * NaN and 0 * infinity are NaN: where such a tile's values hold one (rare), its second product runs without those values, and
// they are then added for the rows that see them.
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
  int n_heads, group, split, tile_is_seq;            // split: keys per workgroup (0: all); tile_is_seq: every sequence fits one tile
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

// 16 bytes of T from the cache: element e of a token's row
template <typename T, bool F8>
__device__ __forceinline__ Chunk16 cache_chunk(const void* base, int64_t at) {
  if constexpr (!F8) return *reinterpret_cast<const Chunk16*>(reinterpret_cast<const T*>(base) + at);
  else {
    constexpr int VEC = TypeInfo<T>::kVec;
    float x[VEC];
    const unsigned* w = reinterpret_cast<const unsigned*>(reinterpret_cast<const char*>(base) + at);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) e4m3_to_f32(w[i], x + 4 * i);
    return chunk_from_f32<T>(x);                     // exact: three bits of mantissa
  }
}

template <typename T, bool F8, int HD>
__global__ __launch_bounds__(kThreads) void paged_attn_kernel(const PagedAttnKArgs p) {
  constexpr int RB = HD * (int)sizeof(T), NCH = RB / 16, SWZ = RB == 128 ? 7 : 15, NBLK = RB / 64, NDT = HD / 16, NLD = KT * NCH / kThreads;
  __shared__ __attribute__((aligned(16))) char sK[KT * RB];
  __shared__ __attribute__((aligned(16))) char sV[KT * RB];
  __shared__ float s_ks[KT], s_vs[KT];
  __shared__ int s_odd;                                // the V tile holds an infinity or a NaN

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, qi = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.y, G = p.group;
  const TileAt at = p.tile_is_seq ? TileAt{(int)blockIdx.x, 0} : wave_find_tile<64>(p.b, G, blockIdx.x, lane);
  if (at.seq < 0) return;
  const SeqInfo sq = paged_seq(p.b, at.seq);
  if (sq.bad && tid == 0) paged_report(p.kv.status, kBadLength);
  const int packed = sq.nq * G;
  if (at.r0 >= packed) return;
  const int last_tok = (min(at.r0 + 64, packed) - 1) / G;
  const int first_pos = sq.ctx - sq.nq;                // place of the sequence's first new token
  const int kmax = min(sq.ctx, p.b.max_ctx);
  const int kend_all = max(0, min(first_pos + last_tok + 1, kmax));
  const int kbeg = p.split ? min(kend_all, (int)blockIdx.z * p.split) : 0;
  if (p.split && blockIdx.z > 0 && kbeg >= kend_all) return;
  const int kend = p.split ? min(kend_all, kbeg + p.split) : kend_all;

  const int r = at.r0 + wave * 16 + qi, rc = min(r, packed - 1), tok = rc / G, head = kvh * G + (rc - tok * G);
  const int64_t row = sq.q0 + tok;
  const int see = min(first_pos + tok + 1, kmax);      // keys this row sees
  const int tok0 = min(at.r0 + wave * 16, packed - 1) / G, see0 = min(first_pos + tok0 + 1, kmax);      // ... and the wave's first row

  Chunk16 qf[NBLK];
  {
    const char* qp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.Q) + row * p.ldq + (int64_t)head * HD);
#pragma unroll
    for (int b = 0; b < NBLK; ++b) qf[b] = *reinterpret_cast<const Chunk16*>(qp + b * 64 + g * 16);
  }
  f32x4 o[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  const int shift = page_shift_of(p.kv);

  for (int kt0 = kbeg; kt0 < kend; kt0 += KT) {
    __syncthreads();
    if (tid == 0) s_odd = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int id = tid + j * kThreads, krow = id / NCH, c = id - krow * NCH, key = kt0 + krow;
      Chunk16 ck, cv;
      ck.v = cv.v = u32x4{0u, 0u, 0u, 0u};
      float ks = 0.f, vs = 0.f;
      if (key < kend) {
        const int page = paged_page(p.kv, p.b, at.seq, key, shift);
        if (page >= 0) {
          const int64_t t = (int64_t)kvh * p.kv.page_size + (key & (p.kv.page_size - 1));
          const int64_t e = (int64_t)page * p.kv.page_stride + t * HD + c * TypeInfo<T>::kVec;
          ck = cache_chunk<T, F8>(p.kv.K, e);
          cv = cache_chunk<T, F8>(p.kv.V, e);
          if constexpr (F8) {
            ks = p.kv.k_scale[(int64_t)page * p.kv.scale_stride + t];
            vs = p.kv.v_scale[(int64_t)page * p.kv.scale_stride + t];
          }
        } else if (c == 0) paged_report(p.kv.status, kBadPage);
      }
      const int off = krow * RB + ((c ^ (krow & SWZ)) << 4);
      *reinterpret_cast<Chunk16*>(sK + off) = ck;
      *reinterpret_cast<Chunk16*>(sV + off) = cv;
      if (!chunk_finite(cv, T())) s_odd = 1;
      if (F8 && c == 0) { s_ks[krow] = ks; s_vs[krow] = vs; }
    }
    __syncthreads();

    const bool edge = kt0 + KT > see0;                 // some row of the wave does not see the whole tile
    f32x4 s[4];
    float mt = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int krow = kt * 16 + qi;
#pragma unroll
      for (int b = 0; b < NBLK; ++b) Mma16<T>::run(*reinterpret_cast<const Chunk16*>(sK + krow * RB + (((b * 4 + g) ^ (krow & SWZ)) << 4)), qf[b], s[kt]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = kt * 16 + 4 * g + i;
        float v = s[kt][i] * p.scale2;
        if (F8) v *= s_ks[k];
        if (edge && kt0 + k >= see) v = -INFINITY;
        s[kt][i] = v;
        mt = fmaxf(mt, v);
      }
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float m_new = fmaxf(m_run, mt), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m_run - m_use);
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = kt * 16 + 4 * g + i;
        float e = exp2f(s[kt][i] - m_use);
        sum += e;
        if (F8) e *= s_vs[k];
        if (edge && kt0 + k >= see) e = 0.f;
        s[kt][i] = e;
      }
    l_run = l_run * alpha + sum;
    m_run = m_new;
#pragma unroll
    for (int i = 0; i < NDT; ++i) o[i] *= alpha;

    const bool odd = edge && s_odd;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        bf16x8 pf;
#pragma unroll
        for (int i = 0; i < 4; ++i) { pf[i] = (bf16_t)s[2 * u][i]; pf[4 + i] = (bf16_t)s[2 * u + 1][i]; }
        const int qq = qi >> 2, pp = qi & 3;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const int c = dt * 2 + (pp >> 1), row0 = 32 * u + 4 * g + qq, row1 = row0 + 16;
          const bf16x4 v0 = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(sV + row0 * RB + ((c ^ (row0 & SWZ)) << 4) + (pp & 1) * 8)));
          const bf16x4 v1 = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(sV + row1 * RB + ((c ^ (row1 & SWZ)) << 4) + (pp & 1) * 8)));
          bf16x8 vf;
#pragma unroll
          for (int i = 0; i < 4; ++i) { vf[i] = v0[i]; vf[4 + i] = v1[i]; }
          if (odd) vf = finite_part(vf);
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, o[dt], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const int c = dt * 4 + (qi >> 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int krow = kt * 16 + 4 * g + i;
            float vv = *reinterpret_cast<const float*>(sV + krow * RB + ((c ^ (krow & SWZ)) << 4) + (qi & 3) * 4);
            if (odd && !is_finite(vv)) vv = 0.f;
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv, s[kt][i], o[dt], 0, 0, 0);
          }
        }
    }
    if (odd) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          for (int gg = 0; gg < 4; ++gg) {
            const float e = __shfl(s[kt][i], gg * 16 + qi, 64);
            const int krow = kt * 16 + 4 * gg + i;
            if (kt0 + krow < see)
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const int byte = (dt * 16 + 4 * g + q) * (int)sizeof(T);
                  const float vv = to_f32(*reinterpret_cast<const T*>(sV + krow * RB + (((byte >> 4) ^ (krow & SWZ)) << 4) + (byte & 15)));
                  if (!is_finite(vv)) o[dt][q] += e * vv;
                }
          }
    }
  }

  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (r >= packed) return;
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // (a NaN sum stays one)
  if (p.split) {
    const int64_t at_row = ((int64_t)blockIdx.z * p.b.rows + row) * p.n_heads + head;
    if (g == 0) p.part_ml[at_row] = make_float2(m_run, l_run);
    float* P = p.part + at_row * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(P + dt * 16 + 4 * g) = o[dt] * inv;
    return;
  }
  if (p.lse && g == 0) p.lse[row * p.n_heads + head] = l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * 0.69314718055994530942f;
  T* O = reinterpret_cast<T*>(p.O) + row * p.ldo + (int64_t)head * HD;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    if constexpr (sizeof(T) == 2) {
      bf16x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (bf16_t)(o[dt][i] * inv);
      *reinterpret_cast<bf16x4*>(O + dt * 16 + 4 * g) = w;
    } else *reinterpret_cast<f32x4*>(O + dt * 16 + 4 * g) = o[dt] * inv;
  }
}

// Joins the splits of a row's keys: a wave per (row, head), the splits in order.  out = sum_z w_z O_z / sum_z w_z,  w_z = l_z 2^(m_z - max m).
template <typename T, int HD>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnKArgs p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * 4 + wave;
  if (i >= (int64_t)p.b.rows * p.n_heads) return;
  const int row = (int)(i / p.n_heads), head = (int)(i - (int64_t)row * p.n_heads);
  const int seq = wave_find_seq(p.b.cu_q, p.b.n_seqs, row, lane);
  const SeqInfo sq = paged_seq(p.b, seq);
  if (row < sq.q0 || row >= sq.q0 + sq.nq) return;
  const int see = min(sq.ctx - sq.nq + (row - sq.q0) + 1, min(sq.ctx, p.b.max_ctx));
  const int n = see > 0 ? (see - 1) / p.split + 1 : 0;
  constexpr int E = HD / 64;
  float acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int z = 0; z < n; ++z) {
    const int64_t at = ((int64_t)z * p.b.rows + row) * p.n_heads + head;
    const float2 ml = p.part_ml[at];
    const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
    const float w0 = exp2f(m - mu), w1 = exp2f(ml.x - mu) * ml.y;
    l = l * w0 + w1;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + w1 * p.part[at * HD + lane * E + e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (p.lse && lane == 0) p.lse[i] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
  T* O = reinterpret_cast<T*>(p.O) + row * p.ldo + (int64_t)head * HD;
#pragma unroll
  for (int e = 0; e < E; ++e) O[lane * E + e] = from_f32<T>(acc[e] * inv);
}

int cu_count() {
  static const int n = [] { int d = 0, c = 256; (void)hipGetDevice(&d); (void)hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, d); return c; }();
  return n;
}

// How a call is laid out: tiles of packed rows, keys per workgroup.
struct Plan { int64_t tiles; int split, splits, tile_is_seq; };
Plan plan_of(const PagedKv& kv, const PagedBatch& b, const PagedAttnArgs& a) {
  Plan pl;
  const int G = a.n_heads / kv.n_kv_heads;
  pl.tile_is_seq = (int64_t)b.max_q * G <= 64;
  pl.tiles = pl.tile_is_seq ? b.n_seqs : (int64_t)b.rows * G / 64 + b.n_seqs;
  pl.split = a.split_keys;
  if (!pl.split) {
    const int64_t wgs = pl.tiles * kv.n_kv_heads, want = 4 * cu_count();
    int64_t n = want / (wgs > 0 ? wgs : 1);
    int64_t k = n > 1 ? ceil_div64(b.max_ctx, n) : b.max_ctx;
    k = (k + 255) / 256 * 256;
    pl.split = (int)(k < 256 ? 256 : k);
  }
  pl.splits = b.max_ctx > 0 ? ceil_div(b.max_ctx, pl.split) : 1;
  if (pl.splits <= 1) pl.split = 0, pl.splits = 1;
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
  hipLaunchKernelGGL((paged_attn_kernel<T, F8, HD>), dim3((unsigned)pl.tiles, k.kv.n_kv_heads, pl.splits), dim3(kThreads), 0, st, k);
  OAVSR_CHECK_HIP(hipGetLastError());
  if (pl.split) {
    hipLaunchKernelGGL((paged_merge_kernel<T, HD>), dim3((unsigned)ceil_div64((int64_t)k.b.rows * k.n_heads, 4)), dim3(kThreads), 0, st, k);
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
  if (b.rows == 0 || b.n_seqs == 0) return 0;
  const Plan pl = plan_of(kv, b, a);
  const uint64_t need = workspace_of(kv, b, a, pl);
  OAVSR_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "paged_attention: a workspace of %llu bytes is needed, %llu given", (unsigned long long)need,
                (unsigned long long)(a.workspace ? a.workspace_bytes : 0));
  OAVSR_REQUIRE(pl.tiles < (1ll << 31) && pl.splits <= 65535, "paged_attention: too many workgroups (%lld tiles, %d splits)", (long long)pl.tiles, pl.splits);
  PagedAttnKArgs k;
  k.kv = kv; k.b = b; k.Q = a.Q; k.ldq = a.ldq; k.O = a.O; k.ldo = a.ldo; k.lse = a.lse; k.scale2 = a.scale * 1.44269504088896340736f;
  k.n_heads = a.n_heads; k.group = a.n_heads / kv.n_kv_heads; k.split = pl.split; k.tile_is_seq = pl.tile_is_seq;
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
