// Attention over a paged K/V cache held in 8 bits with a scale for each block and head.
//
// For query row i of head h with visible tokens t (K codes kc_t, V codes vc_t in a block b whose
// scales are ks_b, vs_b):
//     s_t = scale * ks_b * (q . kc_t),   out = sum_t e^(s_t) vs_b vc_t / sum_t e^(s_t).
// A scale is one number for a tile of tokens, so neither product multiplies a cached element by
// it: ks_b goes onto the score, and vs_b into the exponent. With base-2 scores s' = s log2 e and
//     w_t = 2^(s'_t + log2 vs_b - M),  M the running maximum of s'_t + log2 vs_b,
// out = sum w_t vc_t / sum (w_t / vs_b). Both sums and M are float32; w is at most 2^8 and is
// rounded to half precision for its product alone (float32 queries: to a pair of halves).
//
// The codes are exact in half precision, so both products run on m16n8k16 half-precision tensor
// instructions with float32 sums. A query row is scaled by a power of two into [-1, 1] (its
// exponent returns with ks_b); bfloat16 queries are then exact halves down to 2^-14 of the row's
// largest, float32 ones are split into two halves.
//
// Bound: HBM, 2 D bytes a token and K/V head. What the layout buys: the fragments' index maps are
// free to choose, because q . kc sums over dims in any order and the softmax over tokens in any
// order. A lane's 16 dims of K are 16 neighbouring bytes, its V values 8 neighbouring bytes of
// four tokens, the score fragments are the weight fragments of the second product: no shuffle,
// no transposition through shared memory, about 1.4 integer operations a code to make halves.
//
// One CTA takes a request, a K/V head, up to 8 query rows (those of the heads that share the K/V
// head, of all the request's query tokens) and a range of 16-token tiles. Each warp streams its
// own tiles through its own ring of cp.async stages; the warps' partial sums meet in shared
// memory at the end. Long contexts of few requests are split over CTAs, and a dependent launch
// adds the pieces.
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"

namespace vfl {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;             // query rows of a CTA
constexpr int kSmemPerSM = 227 * 1024;
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100: smaller V scales count as it
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.f;

struct Int8AttnParams {
  const void* q;
  int64_t q_stride;
  const int8_t* k_cache;
  const int8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  int64_t num_blocks;
  void* out;
  int64_t out_stride;
  const int32_t* qsl;
  const int32_t* seq_lens;
  const int32_t* table;
  int64_t table_stride;
  int32_t table_cols;
  int num_heads, num_kv_heads, block_size, causal, total_q, max_seq_len;
  int tiles_per_split, num_splits;
  float scale_log2;
  float* ws_acc;  // [total_q * num_heads, num_splits, D]
  float2* ws_ml;  // [total_q * num_heads, num_splits]
  unsigned int* err;
};

// A request's query rows, its cached tokens (clamped to what its table and plan hold), or
// rows < 0 where query_start_loc is out of order.
struct RequestSpan {
  int q_begin, rows, len;
  bool clamped;
};

__device__ __forceinline__ RequestSpan request_span(const Int8AttnParams& p, int r) {
  RequestSpan s;
  s.q_begin = __ldg(p.qsl + r);
  const int q_end = __ldg(p.qsl + r + 1);
  const int len = __ldg(p.seq_lens + r);
  s.rows = s.q_begin < 0 || q_end < s.q_begin || q_end > p.total_q ? -1 : q_end - s.q_begin;
  const int64_t cap = min((int64_t)p.table_cols * p.block_size, (int64_t)p.max_seq_len);
  s.clamped = len > cap;
  s.len = max(s.clamped ? (int)cap : len, 0);
  return s;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where the 32-byte unit `u` of row `row` of a 16 x D byte tile lies: the units of a 128-byte
// line are permuted so that the eight rows (K) and four rows (V) that a warp reads together
// fall into different banks.
template <int D>
__device__ __forceinline__ int tile_offset(int row, int byte) {
  if (D == 64) {
    const int line = row >> 1, in_line = (row & 1) * 64 + byte;
    return line * 128 + (in_line ^ ((line & 3) << 5));
  }
  if (D % 128 == 0) {
    const int x = (row & 3) ^ ((row >> 1) & 2);
    return row * D + (byte ^ (x << 5));
  }
  return row * D + byte;
}

// Bytes 0, 2 (shift 0) or 1, 3 (shift 8) of `w`, signed, as two halves: 0x6400 | (b ^ 0x80) is
// 1024 + b + 128, from which 1152 leaves b exactly.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w) {
  const uint32_t biased = (w & 0x00ff00ffu) ^ 0x64806480u;
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), bias);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// c[0..1] (rows 0-7 of the product) += A . B with rows 8-15 of A zero: those rows' sums are
// zeros that nothing keeps.
__device__ __forceinline__ void mma_half_rows8(float& c0, float& c1, uint32_t a0, uint32_t a2, uint32_t b0,
                                               uint32_t b1) {
  float d2, d3;
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%10,%10};"
      : "+f"(c0), "+f"(c1), "=f"(d2), "=f"(d3)
      : "r"(a0), "r"(0u), "r"(a2), "r"(0u), "r"(b0), "r"(b1), "f"(0.f));
}

// What a warp knows of 32 of its tiles, one a lane: the tile's block and its scales.
struct TileMeta {
  int64_t head_row;  // (block * num_kv_heads + head): row of the scale tables
  float ks, lv, inv_vs;
};

template <typename T, int D>
struct Shape {
  static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;  // halves that make up a query element
  static constexpr int kSteps = D / 16;                  // k16 steps of q . kc
  static constexpr int kTiles = D / 8;                   // n8 tiles of the output
  static constexpr int kStageBytes = 2 * 16 * D;
  static constexpr int kStages = D <= 64 ? 6 : (D <= 128 ? 4 : (D <= 256 ? 3 : 2));
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kMergeFloats = kWarps * kRows * (D + 2);
  static constexpr int kSmem = kWarps * kRingBytes > kMergeFloats * 4 ? kWarps * kRingBytes : kMergeFloats * 4;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&f)[4]) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[4]) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
  f[0] = __uint_as_float(v.x << 16);
  f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16);
  f[3] = __uint_as_float(v.y & 0xffff0000u);
}

__device__ __forceinline__ void store_elem(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_elem(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Factor of a piece with maximum `m` in a sum with maximum `m_all`. A piece without a maximum
// holds zeros (nothing visible) or NaNs (every score a NaN), and either is to be kept.
__device__ __forceinline__ float merge_factor(float m, float m_all) {
  return m == -INFINITY ? 1.f : exp2_approx(m - m_all);
}

// First dim of the word (4 codes) of k16 step s that lane group thread tq holds: whole groups of
// 64 dims give a thread 16 neighbouring bytes, the rest 4.
template <int D>
__device__ __forceinline__ int k_dim(int s, int tq) {
  constexpr int kWhole = D / 64 * 4;
  return s < kWhole ? (s >> 2) * 64 + tq * 16 + (s & 3) * 4 : kWhole * 16 + (s - kWhole) * 16 + tq * 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_attention_int8_kernel(const Int8AttnParams p) {
  using S = Shape<T, D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int r = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - r * p.num_kv_heads;
  const int split = blockIdx.z;
  const RequestSpan req = request_span(p, r);
  if (req.rows < 0) {
    if (threadIdx.x == 0 && kvh == 0 && blockIdx.y == 0 && split == 0) report(p.err, VFL_DEVERR_QUERY);
    return;
  }
  if (req.clamped && threadIdx.x == 0 && kvh == 0 && blockIdx.y == 0 && split == 0)
    report(p.err, VFL_DEVERR_CONTEXT);
  // the request's rows of this K/V head: query token j of group head e is row j * group + e
  const int group = p.num_heads / p.num_kv_heads;
  const int row0 = blockIdx.y * kRows;
  const int nrows = min(kRows, req.rows * group - row0);
  if (nrows <= 0) return;
  const int L = req.len;
  const int tiles_all = ceil_div(L, 16);
  const int n_splits = max(1, ceil_div(tiles_all, p.tiles_per_split));
  if (split >= n_splits) return;
  // visible tokens of row i (causal rows end at successive positions)
  auto visible = [&](int i) {
    return i < nrows ? max(p.causal ? L - (req.rows - 1 - (row0 + i) / group) : L, 0) : 0;
  };
  const int vis_max = visible(nrows - 1);
  const int tile_begin = split * p.tiles_per_split;
  const int tile_end = min(tile_begin + p.tiles_per_split, ceil_div(vis_max, 16));
  const int bs = p.block_size, tpb = bs / 16;

  // ---- this lane's query row, scaled into [-1, 1], as the A fragments of q . kc
  const bool row_on = g < nrows;
  const int token = row_on ? (row0 + g) / group : 0;
  const int head = kvh * group + (row_on ? (row0 + g) % group : 0);
  const int64_t q_row = req.q_begin + token;
  uint32_t qa[S::kTerms][S::kSteps][2];
  float q_scale = 1.f;
  {
    const T* src = static_cast<const T*>(p.q) + q_row * p.q_stride + (int64_t)head * D;
    float amax = 0.f;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (row_on) load4(src + k_dim<D>(s, tq), f);
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(f[i]));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^e >= amax > 2^(e-1); an infinity stays one in the products, as it would unscaled
    int e = 0;
    if (amax > 0.f && amax <= FLT_MAX) frexpf(amax, &e);
    e = max(-125, min(126, e));
    q_scale = ldexpf(1.f, e);
    const float q_inv = ldexpf(1.f, -e);
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (row_on) load4(src + k_dim<D>(s, tq), f);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] *= q_inv;
      qa[0][s][0] = pack_half2(f[0], f[2]);
      qa[0][s][1] = pack_half2(f[1], f[3]);
      if (S::kTerms == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] -= __half2float(__float2half_rn(f[i]));
        qa[S::kTerms - 1][s][0] = pack_half2(f[0], f[2]);
        qa[S::kTerms - 1][s][1] = pack_half2(f[1], f[3]);
      }
    }
  }
  const float s_mul = q_scale * p.scale_log2;
  const int vis = visible(g);

  // ---- this warp's tiles: tile_begin + warp + kWarps * i
  const int first = tile_begin + warp;
  const int count = tile_end > first ? ceil_div(tile_end - first, kWarps) : 0;
  uint8_t* ring = smem + warp * S::kRingBytes;
  const uint32_t ring_u32 = smem_u32(ring);
  auto load_meta = [&](int i) {  // of tile i of this warp
    TileMeta m{0, 0.f, 0.f, 1.f};
    if (i < count) {
      int b = __ldg(p.table + (int64_t)r * p.table_stride + (first + kWarps * i) / tpb);
      if (b < 0 || b >= p.num_blocks) {
        report(p.err, VFL_DEVERR_BLOCK_ID);
        b = 0;
      }
      m.head_row = (int64_t)b * p.num_kv_heads + kvh;
      m.ks = __ldg(p.k_scale + m.head_row);
      const float vs = __ldg(p.v_scale + m.head_row);
      const float vs_used = vs > 0.f ? fmaxf(vs, kMinScale) : 1.f;  // a zero scale's codes are zeros
      m.lv = log2f(vs_used);
      m.inv_vs = 1.f / vs_used;
    }
    return m;
  };
  TileMeta meta = load_meta(lane), ahead = load_meta(32 + lane);  // tiles base..base+31, base+32..base+63
  int base = 0;
  auto issue = [&](int i) {  // copies tile i into its stage (a group of its own, empty past the end)
    if (i < count) {
      const int64_t row = __shfl_sync(0xffffffffu, i < base + 32 ? meta.head_row : ahead.head_row, i & 31);
      const int tile = first + kWarps * i;
      const int64_t src = (row * bs + (tile % tpb) * 16) * D;
      const uint32_t dst = ring_u32 + (i % S::kStages) * S::kStageBytes;
#pragma unroll
      for (int j = 0; j < (D + 31) / 32; ++j) {
        const int c = j * 32 + lane;  // 16-byte piece of the 16 x D tile
        if (D % 32 == 0 || c < D) {
          const int trow = c / (D / 16), byte = (c % (D / 16)) * 16;
          const uint32_t at = dst + tile_offset<D>(trow, byte);
          cp_async16(at, p.k_cache + src + c * 16);
          cp_async16(at + 16 * D, p.v_cache + src + c * 16);
        }
      }
    }
    cp_async_commit();
  };

  float m_run = -INFINITY, l_run = 0.f;
  float acc[S::kTiles][2];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) acc[t][0] = acc[t][1] = 0.f;

#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    if (i == base + 32) {
      base += 32;
      meta = ahead;
      ahead = load_meta(base + 32 + lane);
    }
    issue(i + S::kStages - 1);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    const uint8_t* kt = ring + (i % S::kStages) * S::kStageBytes;
    const uint8_t* vt = kt + 16 * D;

    // scores of rows g over tokens tq, tq + 4 (tile 0 of n8) and tq + 8, tq + 12 (tile 1)
    float sc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int krow = (g >> 1) + 4 * (g & 1) + 8 * nt;
#pragma unroll
      for (int c = 0; c < (S::kSteps + 3) / 4; ++c) {
        uint32_t w[4];
        if (c < D / 64) {
          const uint4 v = *reinterpret_cast<const uint4*>(kt + tile_offset<D>(krow, c * 64 + tq * 16));
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < S::kSteps - 4 * c && j < 4; ++j)
            w[j] = *reinterpret_cast<const uint32_t*>(kt + tile_offset<D>(krow, c * 64 + j * 16 + tq * 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = 4 * c + j;
          if (s < S::kSteps) {
            const uint32_t b0 = codes_to_half2(w[j]), b1 = codes_to_half2(w[j] >> 8);
#pragma unroll
            for (int term = 0; term < S::kTerms; ++term)
              mma_half_rows8(sc[nt][0], sc[nt][1], qa[term][s][0], qa[term][s][1], b0, b1);
          }
        }
      }
    }

    // weights
    const float ks = __shfl_sync(0xffffffffu, meta.ks, i & 31) * s_mul;
    const float lv = __shfl_sync(0xffffffffu, meta.lv, i & 31);
    const float inv_vs = __shfl_sync(0xffffffffu, meta.inv_vs, i & 31);
    const int tok0 = (first + kWarps * i) * 16;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = tok0 + tq + 4 * e;
      x[e] = tok < vis ? fmaf(sc[e >> 1][e & 1], ks, lv) : -INFINITY;
    }
    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if (__any_sync(0xffffffffu, top > m_run + kRescaleSlack)) {
      float mx = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (mx > m_run + kRescaleSlack) {
        const float alpha = m_run == -INFINITY ? 0.f : exp2_approx(m_run - mx);
        m_run = mx;
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
          acc[t][0] *= alpha;
          acc[t][1] *= alpha;
        }
      }
    }
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // a row that has seen no token yet has m = -inf, and x - m would be a NaN
      w[e] = x[e] == -INFINITY ? 0.f : exp2_approx(x[e] - m_run);
      l_run = fmaf(w[e], inv_vs, l_run);
    }
    uint32_t pa[S::kTerms][2];
    pa[0][0] = pack_half2(w[0], w[1]);
    pa[0][1] = pack_half2(w[2], w[3]);
    if (S::kTerms == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] -= __half2float(__float2half_rn(w[e]));
      pa[S::kTerms - 1][0] = pack_half2(w[0], w[1]);
      pa[S::kTerms - 1][1] = pack_half2(w[2], w[3]);
    }

    // out += w . vc: n8 tile `t` holds, of each group of 8 * span dims, dims span * g + (t - t0)
    constexpr int kSpan16 = D / 128, kSpan8 = (D % 128) / 64, kSpan4 = (D % 64) / 32, kSpan2 = (D % 32) / 16;
    auto product = [&](const uint32_t (&word)[4], int t) {  // 4 dims of the four tokens
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // tokens tq, tq + 4 side by side: (dim, dim + 1) of one, then of the other
        const uint32_t lo = __byte_perm(word[0], word[1], half ? 0x7632 : 0x5410);
        const uint32_t hi = __byte_perm(word[2], word[3], half ? 0x7632 : 0x5410);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const uint32_t b0 = codes_to_half2(lo >> (8 * d)), b1 = codes_to_half2(hi >> (8 * d));
          const int n = t + 2 * half + d;
          if (n < S::kTiles) {
#pragma unroll
            for (int term = 0; term < S::kTerms; ++term)
              mma_half_rows8(acc[n][0], acc[n][1], pa[term][0], pa[term][1], b0, b1);
          }
        }
      }
    };
#pragma unroll
    for (int c = 0; c < kSpan16; ++c) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint4*>(vt + tile_offset<D>(tq + 4 * e, c * 128 + g * 16));
      const uint32_t w0[4] = {v[0].x, v[1].x, v[2].x, v[3].x}, w1[4] = {v[0].y, v[1].y, v[2].y, v[3].y};
      const uint32_t w2[4] = {v[0].z, v[1].z, v[2].z, v[3].z}, w3[4] = {v[0].w, v[1].w, v[2].w, v[3].w};
      product(w0, 16 * c);
      product(w1, 16 * c + 4);
      product(w2, 16 * c + 8);
      product(w3, 16 * c + 12);
    }
    if (kSpan8) {
      constexpr int b = kSpan16 * 128;
      uint2 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint2*>(vt + tile_offset<D>(tq + 4 * e, b + g * 8));
      const uint32_t w0[4] = {v[0].x, v[1].x, v[2].x, v[3].x}, w1[4] = {v[0].y, v[1].y, v[2].y, v[3].y};
      product(w0, b / 8);
      product(w1, b / 8 + 4);
    }
    if (kSpan4) {
      constexpr int b = kSpan16 * 128 + kSpan8 * 64;
      uint32_t w0[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w0[e] = *reinterpret_cast<const uint32_t*>(vt + tile_offset<D>(tq + 4 * e, b + g * 4));
      product(w0, b / 8);
    }
    if (kSpan2) {
      constexpr int b = kSpan16 * 128 + kSpan8 * 64 + kSpan4 * 32;
      uint32_t w0[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w0[e] = *reinterpret_cast<const uint16_t*>(vt + tile_offset<D>(tq + 4 * e, b + g * 2));
      product(w0, b / 8);  // its upper two tiles do not exist
    }
    __syncwarp();  // every lane is done with the stage before it is filled again
  }
  cp_async_wait<0>();

  // ---- the warps' sums meet: m, l, acc per row, then one thread per (row, dim)
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  __syncthreads();  // the rings are free
  float* ml = reinterpret_cast<float*>(smem);          // [warp][row][2]
  float* sum = ml + kWarps * kRows * 2;                // [warp][row][D]
  if (row_on) {
    if (tq == 0) {
      ml[(warp * kRows + g) * 2] = m_run;
      ml[(warp * kRows + g) * 2 + 1] = l_run;
    }
    float* dst = sum + (warp * kRows + g) * D;
    constexpr int kSpan16 = D / 128, kSpan8 = (D % 128) / 64, kSpan4 = (D % 64) / 32;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) {
      // tile t's column n is dim start + span * n + (t - start / 8)
      const int start = t < kSpan16 * 16 ? t / 16 * 128
                        : t < kSpan16 * 16 + kSpan8 * 8 ? kSpan16 * 128
                        : t < kSpan16 * 16 + kSpan8 * 8 + kSpan4 * 4 ? kSpan16 * 128 + kSpan8 * 64
                                                                     : kSpan16 * 128 + kSpan8 * 64 + kSpan4 * 32;
      const int span = t < kSpan16 * 16 ? 16 : t < kSpan16 * 16 + kSpan8 * 8 ? 8
                       : t < kSpan16 * 16 + kSpan8 * 8 + kSpan4 * 4 ? 4 : 2;
#pragma unroll
      for (int e = 0; e < 2; ++e) dst[start + span * (2 * tq + e) + (t - start / 8)] = acc[t][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * D; i += kThreads) {
    const int row = i / D, d = i - row * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[(w * kRows + row) * 2]);
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = merge_factor(ml[(w * kRows + row) * 2], m);
      l = fmaf(f, ml[(w * kRows + row) * 2 + 1], l);
      o = fmaf(f, sum[(w * kRows + row) * D + d], o);
    }
    const int64_t out_row = req.q_begin + (row0 + row) / group;
    const int out_head = kvh * group + (row0 + row) % group;
    if (n_splits == 1) {
      // l is a NaN where a score was: the row then is one, as in a plain softmax
      store_elem(static_cast<T*>(p.out) + out_row * p.out_stride + (int64_t)out_head * D + d, l == 0.f ? 0.f : o / l);
    } else {
      const int64_t item = (out_row * p.num_heads + out_head) * p.num_splits + split;
      p.ws_acc[item * D + d] = o;
      if (d == 0) p.ws_ml[item] = make_float2(m, l);
    }
  }
}

// Adds the pieces of rows that were split. grid: (requests, query tokens of the longest request,
// heads); one thread a dim.
template <typename T>
__global__ void combine_int8_kernel(const Int8AttnParams p, int D) {
  griddep_wait();
  const RequestSpan req = request_span(p, blockIdx.x);
  if ((int)blockIdx.y >= req.rows) return;
  const int tiles_all = ceil_div(req.len, 16);
  const int n_splits = max(1, ceil_div(tiles_all, p.tiles_per_split));
  if (n_splits == 1) return;
  const int h = blockIdx.z;
  const int64_t row = req.q_begin + blockIdx.y;
  const int64_t item = (row * p.num_heads + h) * p.num_splits;
  float m = -INFINITY;
  for (int s = 0; s < n_splits; ++s) m = fmaxf(m, p.ws_ml[item + s].x);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float l = 0.f, o = 0.f;
    for (int s = 0; s < n_splits; ++s) {
      const float2 ml = p.ws_ml[item + s];
      const float f = merge_factor(ml.x, m);
      l = fmaf(f, ml.y, l);
      o = fmaf(f, p.ws_acc[(item + s) * D + d], o);
    }
    store_elem(static_cast<T*>(p.out) + row * p.out_stride + (int64_t)h * D + d, l == 0.f ? 0.f : o / l);
  }
}

int64_t acc_bytes(int64_t items, int D) { return ceil_div(items * D * 4, (int64_t)256) * 256; }

int64_t workspace_of(const vfl_attention_int8_plan* plan) {
  if (plan->num_splits <= 1) return 0;
  const int64_t items = (int64_t)plan->total_q * plan->num_heads * plan->num_splits;
  return acc_bytes(items, plan->head_dim) + items * 8;
}

int row_chunks(const vfl_attention_int8_plan* plan) {
  return static_cast<int>(ceil_div((int64_t)plan->max_q_len * (plan->num_heads / plan->num_kv_heads), (int64_t)kRows));
}

int smem_bytes(int dtype, int D) {
  const int stage = 32 * D, stages = D <= 64 ? 6 : (D <= 128 ? 4 : (D <= 256 ? 3 : 2));
  const int ring = kWarps * stage * stages, merge = kWarps * kRows * (D + 2) * 4;
  (void)dtype;
  return ring > merge ? ring : merge;
}

template <typename T, int D>
int launch(const Int8AttnParams& p, dim3 grid, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  auto kern = paged_attention_int8_kernel<T, D>;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), Shape<T, D>::kSmem, smem_done);
  if (st) return st;
  kern<<<grid, kThreads, Shape<T, D>::kSmem, stream>>>(p);
  return cuda_status(cudaGetLastError(), "attention_with_kv_cache_int8 launch");
}

template <typename T>
int launch_dim(const Int8AttnParams& p, int D, dim3 grid, cudaStream_t s) {
  switch (D) {
    case 32: return launch<T, 32>(p, grid, s);
    case 48: return launch<T, 48>(p, grid, s);
    case 64: return launch<T, 64>(p, grid, s);
    case 80: return launch<T, 80>(p, grid, s);
    case 96: return launch<T, 96>(p, grid, s);
    case 112: return launch<T, 112>(p, grid, s);
    case 128: return launch<T, 128>(p, grid, s);
    case 160: return launch<T, 160>(p, grid, s);
    case 192: return launch<T, 192>(p, grid, s);
    case 224: return launch<T, 224>(p, grid, s);
    case 256: return launch<T, 256>(p, grid, s);
    default: return launch<T, 512>(p, grid, s);
  }
}

// A plan is caller memory: what the kernels rely on is checked again.
int check_plan(const vfl_attention_int8_plan* plan) {
  if (plan == nullptr || plan->magic != VFL_INT8_PLAN_MAGIC)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan was not made by vfl_plan_attention_int8");
  if (plan->num_reqs < 0 || plan->num_heads <= 0 || plan->num_kv_heads <= 0 ||
      plan->num_heads % plan->num_kv_heads != 0 || plan->total_q < 0 || plan->max_q_len < 0 || plan->max_seq_len < 0 ||
      (plan->causal != 0 && plan->causal != 1))
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan counts out of range");
  if (!dtype_ok(plan->dtype) || !head_dim_supported(plan->head_dim) || plan->block_size < 16 ||
      plan->block_size > 1024 || plan->block_size % 16 != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan dtype / head_dim / block_size not built");
  if (plan->num_splits < 1 || plan->num_splits > 65535 || plan->tiles_per_split < 1 ||
      (int64_t)plan->num_splits * plan->tiles_per_split < ceil_div((int64_t)plan->max_seq_len, (int64_t)16))
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan splits do not cover max_seq_len %d", plan->max_seq_len);
  if (row_chunks(plan) > 65535 || (int64_t)plan->num_reqs * plan->num_kv_heads > INT32_MAX ||
      plan->max_q_len > 65535 || plan->num_heads > 65535)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan launch grid too large");
  if (plan->workspace_bytes < workspace_of(plan))
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan workspace_bytes %lld < the %lld its splits need",
                (long long)plan->workspace_bytes, (long long)workspace_of(plan));
  return VFL_OK;
}

}  // namespace
}  // namespace vfl

using namespace vfl;

extern "C" {

int vfl_plan_attention_int8(int num_reqs, int num_heads, int num_kv_heads, int head_dim, int block_size, int dtype,
                            int causal, const int32_t* seq_lens_host, const int32_t* query_start_loc_host,
                            vfl_attention_int8_plan* plan) {
  if (plan == nullptr) return fail(VFL_ERR_INVALID_ARGUMENT, "plan is NULL");
  plan->magic = 0;
  if (num_reqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: num_reqs %d, num_heads %d, num_kv_heads %d", num_reqs,
                num_heads, num_kv_heads);
  char isa[8];
  int st = vfl_get_isa(dtype, block_size, head_dim, isa, sizeof(isa));
  if (st) return st;
  if (num_reqs > 0 && seq_lens_host == nullptr) return fail(VFL_ERR_INVALID_ARGUMENT, "seq_lens_host is NULL");
  if (query_start_loc_host && query_start_loc_host[0] < 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "query_start_loc[0] < 0");
  const int group = num_heads / num_kv_heads;
  int64_t max_q = 0, max_seq = 0, items = 0;
  for (int r = 0; r < num_reqs; ++r) {
    const int64_t n = seq_lens_host[r];
    const int64_t ql = query_start_loc_host ? (int64_t)query_start_loc_host[r + 1] - query_start_loc_host[r] : 1;
    if (n < 0) return fail(VFL_ERR_INVALID_ARGUMENT, "seq_lens[%d] = %lld < 0", r, (long long)n);
    if (ql < 0) return fail(VFL_ERR_INVALID_ARGUMENT, "query_start_loc decreases at %d", r);
    max_q = ql > max_q ? ql : max_q;
    max_seq = n > max_seq ? n : max_seq;
    items += ceil_div(ql * group, (int64_t)kRows) * num_kv_heads;
  }
  const int64_t total_q = num_reqs == 0 ? 0 : (query_start_loc_host ? query_start_loc_host[num_reqs] : num_reqs);
  if (total_q > INT32_MAX / 2) return fail(VFL_ERR_UNSUPPORTED, "too many query rows (%lld)", (long long)total_q);
  plan->num_reqs = num_reqs;
  plan->num_heads = num_heads;
  plan->num_kv_heads = num_kv_heads;
  plan->head_dim = head_dim;
  plan->block_size = block_size;
  plan->dtype = dtype;
  plan->causal = causal != 0;
  plan->total_q = static_cast<int32_t>(total_q);
  plan->max_q_len = static_cast<int32_t>(max_q);
  plan->max_seq_len = static_cast<int32_t>(max_seq);

  // Splits: as many as give every CTA slot an item, each of at least two tiles a warp.
  int per_sm = kSmemPerSM / (smem_bytes(dtype, head_dim) + 1024);
  per_sm = per_sm < 1 ? 1 : per_sm;
  const int64_t slots = (int64_t)kNumSMs * per_sm;
  const int64_t tiles = ceil_div(max_seq, (int64_t)16);
  int64_t splits = 1;
  if (items > 0 && 2 * items <= slots) {
    const int64_t by_len = tiles / (2 * kWarps);
    splits = slots / items;
    splits = splits < by_len ? splits : by_len;
    splits = splits < 1 ? 1 : splits;
  }
  int64_t per = ceil_div(tiles < 1 ? (int64_t)1 : tiles, splits);
  per = ceil_div(per, (int64_t)kWarps) * kWarps;
  plan->tiles_per_split = static_cast<int32_t>(per);
  plan->num_splits = static_cast<int32_t>(tiles < 1 ? 1 : ceil_div(tiles, per));
  plan->workspace_bytes = workspace_of(plan);
  plan->magic = VFL_INT8_PLAN_MAGIC;
  st = check_plan(plan);
  if (st) plan->magic = 0;
  return st;
}

int vfl_attention_with_kv_cache_int8(const vfl_attention_int8_plan* plan, const void* query, int64_t query_token_stride,
                                     const void* k_cache, const void* v_cache, const float* k_scale,
                                     const float* v_scale, int64_t num_blocks, void* output,
                                     int64_t output_token_stride, const int32_t* query_start_loc,
                                     const int32_t* seq_lens, const int32_t* block_table, int64_t table_stride,
                                     int32_t table_cols, float scale, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  int st = check_plan(plan);
  if (st) return st;
  if (plan->num_reqs == 0 || plan->total_q == 0) return VFL_OK;
  if (!query || !k_cache || !v_cache || !k_scale || !v_scale || !output || !query_start_loc || !seq_lens ||
      (!block_table && table_cols > 0))
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: NULL pointer");
  const int D = plan->head_dim, H = plan->num_heads;
  const int64_t es = static_cast<int64_t>(dtype_size(plan->dtype));
  if (num_blocks <= 0 || num_blocks > INT32_MAX || table_cols < 0 || table_stride < table_cols)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: num_blocks %lld, table_stride %lld, table_cols %d",
                (long long)num_blocks, (long long)table_stride, table_cols);
  if (query_token_stride < (int64_t)H * D || output_token_stride < (int64_t)H * D)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: token stride smaller than a token");
  if (!aligned16(query) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(output) ||
      (query_token_stride * es) % 16 != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: tensors and the query stride must be 16-byte aligned");
  if (!(scale == scale) || fabsf(scale) > FLT_MAX)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: scale is not finite");
  if (plan->workspace_bytes > 0 &&
      (workspace == nullptr || !aligned16(workspace) || workspace_bytes < (size_t)plan->workspace_bytes))
    return fail(VFL_ERR_WORKSPACE, "attention_int8: needs %lld workspace bytes (16-byte aligned), got %zu",
                (long long)plan->workspace_bytes, workspace_bytes);
  Int8AttnParams p;
  st = device_error_word(&p.err);
  if (st) return st;
  p.q = query;
  p.q_stride = query_token_stride;
  p.k_cache = static_cast<const int8_t*>(k_cache);
  p.v_cache = static_cast<const int8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.num_blocks = num_blocks;
  p.out = output;
  p.out_stride = output_token_stride;
  p.qsl = query_start_loc;
  p.seq_lens = seq_lens;
  p.table = block_table;
  p.table_stride = table_stride;
  p.table_cols = table_cols;
  p.num_heads = H;
  p.num_kv_heads = plan->num_kv_heads;
  p.block_size = plan->block_size;
  p.causal = plan->causal;
  p.total_q = plan->total_q;
  p.max_seq_len = plan->max_seq_len;
  p.tiles_per_split = plan->tiles_per_split;
  p.num_splits = plan->num_splits;
  p.scale_log2 = scale * kLog2e;
  const int64_t items = (int64_t)plan->total_q * H * plan->num_splits;
  p.ws_acc = static_cast<float*>(workspace);
  p.ws_ml = plan->num_splits > 1
                ? reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + acc_bytes(items, D)) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(plan->num_reqs * plan->num_kv_heads, row_chunks(plan), plan->num_splits);
  st = plan->dtype == VFL_DTYPE_F32 ? launch_dim<float>(p, D, grid, s) : launch_dim<__nv_bfloat16>(p, D, grid, s);
  if (st || plan->num_splits == 1) return st;
  const dim3 cgrid(plan->num_reqs, plan->max_q_len, H);
  const int threads = D <= 64 ? 64 : 128;
  if (plan->dtype == VFL_DTYPE_F32)
    combine_int8_kernel<float><<<cgrid, threads, 0, s>>>(p, D);
  else
    combine_int8_kernel<__nv_bfloat16><<<cgrid, threads, 0, s>>>(p, D);
  return cuda_status(cudaGetLastError(), "attention_int8 combine launch");
}

}  // extern "C"
