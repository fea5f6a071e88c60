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
// order. Scores are taken as K q^T (16 tokens x 8 query rows) and outputs as V^T w^T (16 dims x 8
// rows), so that the cached elements fill the instruction's 16-row side and a few query rows its
// 8-column side. A lane's 16 dims of K are 16 neighbouring bytes, its V values 8 neighbouring
// bytes of four tokens; two 8 x 8 transpositions in registers turn scores into weights. Per tile
// of 16 tokens and D = 64 that is about 90 integer and half operations a lane to make halves of
// the codes, 8 tensor instructions, and 25 for the softmax.
//
// One CTA takes a request, a K/V head, 8 or 16 query rows (those of the heads that share the K/V
// head, of all the request's query tokens) and a range of 16-token tiles. Each warp streams its
// own tiles through its own ring of cp.async stages; the warps' partial sums meet in shared
// memory at the end. Long contexts of few requests are cut over a cluster of up to 8 CTAs, whose
// sums meet in distributed shared memory, and over more clusters where that is not enough: then
// a dependent launch adds the clusters' pieces.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;
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
  int num_splits, cluster;  // CTAs on an item; of them in a cluster
  float scale_log2;
  float* ws_acc;  // [total_q * num_heads, clusters, D]
  float2* ws_ml;  // [total_q * num_heads, clusters]
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

__device__ __forceinline__ void mma_half(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 x 8 half matrix whose row g the four lanes of group g hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// NT: n8 tiles of query rows.
template <typename T, int D, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;  // halves that make up a query element
  static constexpr int kSteps = D / 16;                  // k16 steps of K q^T
  static constexpr int kTiles = D / 16;                  // m16 tiles of the output
  static constexpr int kStageBytes = 2 * 16 * D;
  static constexpr int kStages = D <= 128 ? 4 : (D <= 256 ? 3 : 2);
  static constexpr int kRingBytes = kStages * kStageBytes;
  // query fragments stay in registers up to this many, in shared memory past it
  static constexpr bool kQueryInSmem = kTerms * NT * kSteps * 2 > 32;
  static constexpr int kQueryBytes = kQueryInSmem ? kTerms * NT * kSteps * 32 * 8 : 0;
  static constexpr int kMetaBytes = kWarps * 64 * 16;
  // sums of the warps [warp][row][D], of the CTA [row][D], and their (m, l)
  static constexpr int kMergeBytes = ((kWarps + 1) * kRows * (D + 2)) * 4;
  static constexpr int kRegion = kWarps * kRingBytes > kMergeBytes ? kWarps * kRingBytes : kMergeBytes;
  static constexpr int kSmem = kRegion + kMetaBytes + kQueryBytes;
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

// The V dims of a lane: column n of [0, D / 8) is dim start + span * g + (n - start / 8), where
// spans of 16, 8, 4 and 2 neighbouring dims cover groups of 128, 64, 32 and 16.
template <int D>
__device__ __forceinline__ int v_dim(int n, int g) {
  constexpr int k16 = D / 128, k8 = (D % 128) / 64, k4 = (D % 64) / 32;
  const int start = n < k16 * 16 ? n / 16 * 128
                    : n < k16 * 16 + k8 * 8 ? k16 * 128
                    : n < k16 * 16 + k8 * 8 + k4 * 4 ? k16 * 128 + k8 * 64
                                                     : k16 * 128 + k8 * 64 + k4 * 32;
  const int span = n < k16 * 16 ? 16 : n < k16 * 16 + k8 * 8 ? 8 : n < k16 * 16 + k8 * 8 + k4 * 4 ? 4 : 2;
  return start + span * g + (n - start / 8);
}

// One query row's four dims of k16 step s as the two B registers of each term.
template <int kTerms>
__device__ __forceinline__ void query_halves(float (&f)[4], float inv, uint32_t (&b)[kTerms][2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= inv;
#pragma unroll
  for (int term = 0; term < kTerms; ++term) {
    b[term][0] = pack_half2(f[0], f[2]);
    b[term][1] = pack_half2(f[1], f[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] -= __half2float(__float2half_rn(f[i]));
  }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) paged_attention_int8_kernel(const Int8AttnParams p) {
  using S = Shape<T, D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int r = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - r * p.num_kv_heads;
  const int split = blockIdx.z;
  const int bs = p.block_size, tpb = bs >> 4;
  const RequestSpan req = request_span(p, r);
  if (req.rows < 0) {
    if (threadIdx.x == 0 && kvh == 0 && blockIdx.y == 0 && split == 0) report(p.err, VFL_DEVERR_QUERY);
    return;
  }
  if (req.clamped && threadIdx.x == 0 && kvh == 0 && blockIdx.y == 0 && split == 0)
    report(p.err, VFL_DEVERR_CONTEXT);
  // the request's rows of this K/V head: query token j of group head e is row j * group + e
  const int group = p.num_heads / p.num_kv_heads;
  const int row0 = blockIdx.y * S::kRows;
  const int nrows = min(S::kRows, req.rows * group - row0);
  if (nrows <= 0) return;
  const int L = req.len;
  // visible tokens of row i (causal rows end at successive positions)
  auto visible = [&](int i) { return max(p.causal ? L - (req.rows - 1 - (row0 + i) / group) : L, 0); };
  // the context's tiles in equal ranges over the item's CTAs, whatever length was planned for
  const int tiles_all = ceil_div(L, 16);
  const int per = ceil_div(tiles_all, p.num_splits);
  const int tile_begin = split * per;
  const int tile_end = min(tile_begin + per, ceil_div(visible(nrows - 1), 16));

  // ---- this warp's tiles: tile_begin + warp + kWarps * i. A lane keeps the position of one of
  // 32 tiles in units of 16 tokens of the pools, and of the next 32.
  const int first = tile_begin + warp;
  const int count = tile_end > first ? ceil_div(tile_end - first, kWarps) : 0;
  auto locate = [&](int i) {
    if (i >= count) return 0;
    const int tile = first + kWarps * i;
    const int col = tpb == 1 ? tile : tile / tpb;
    int b = __ldg(p.table + (int64_t)r * p.table_stride + col);
    if (b < 0 || b >= p.num_blocks) {
      report(p.err, VFL_DEVERR_BLOCK_ID);
      b = 0;
    }
    return (b * p.num_kv_heads + kvh) * tpb + (tile - col * tpb);  // the host checked that it fits
  };
  int place = locate(lane), place_next = 0;
  uint8_t* ring = smem + warp * S::kRingBytes;
  const uint32_t ring_u32 = smem_u32(ring);
  // where this lane's 16-byte pieces of a tile go, within a stage
  constexpr int kPieces = (D + 31) / 32;
  uint32_t piece_at[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int c = j * 32 + lane;
    piece_at[j] = ring_u32 + tile_offset<D>(c / (D / 16), (c % (D / 16)) * 16);
  }
  int base = 0;  // `place` is of tiles base .. base + 31
  auto issue = [&](int i, int stage) {  // copies tile i into `stage` (a group of its own, empty past the end)
    if (i < count) {
      const int at = __shfl_sync(0xffffffffu, i < base + 32 ? place : place_next, i & 31);
      const int64_t src = (int64_t)at * (16 * D) + lane * 16;
      const uint32_t to = stage * S::kStageBytes;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        if (D % 32 == 0 || j * 32 + lane < D) {
          cp_async16(piece_at[j] + to, p.k_cache + src + j * 512);
          cp_async16(piece_at[j] + to + 16 * D, p.v_cache + src + j * 512);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i, i);

  // ---- the tiles' scales: (ks, log2 vs, 1 / vs), 64 tiles of them in shared memory
  float4* meta = reinterpret_cast<float4*>(smem + S::kRegion) + warp * 64;
  float ks_next = 0.f, vs_next = 1.f;
  auto load_scales = [&](int i, int at) {
    if (i < count) {
      const int row = tpb == 1 ? at : at / tpb;
      ks_next = __ldg(p.k_scale + row);
      vs_next = __ldg(p.v_scale + row);
    }
  };
  auto keep_scales = [&](int i) {
    const float vs = vs_next > 0.f ? fmaxf(vs_next, kMinScale) : 1.f;  // a zero scale's codes are zeros
    meta[i & 63] = make_float4(ks_next, log2f(vs), 1.f / vs, 0.f);
  };
  load_scales(lane, place);

  // ---- the query rows, scaled into [-1, 1], as the B fragments of K q^T
  uint2* q_smem = reinterpret_cast<uint2*>(smem + S::kRegion + S::kMetaBytes);
  uint32_t qb[S::kQueryInSmem ? 1 : NT][S::kQueryInSmem ? 1 : S::kSteps][S::kTerms][2];
  float s_mul[NT][2];  // of the rows 2 tq, 2 tq + 1 whose scores this lane holds
  int vis[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = nt * 8 + g;
    const bool on = row < nrows;
    const int vrow = row0 + (on ? row : 0);
    const int token = vrow / group, head = kvh * group + vrow - token * group;
    const T* src = static_cast<const T*>(p.q) + (int64_t)(req.q_begin + token) * p.q_stride + (int64_t)head * D;
    float amax = 0.f;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (on) load4(src + k_dim<D>(s, tq), f);
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(f[i]));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^e > amax >= 2^(e-1); an infinity stays one in the products, as it would unscaled
    int e = 0;
    if (amax > 0.f && amax <= FLT_MAX) frexpf(amax, &e);
    e = max(-125, min(126, e));
    const float inv = ldexpf(1.f, -e);
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (on) load4(src + k_dim<D>(s, tq), f);
      uint32_t b[S::kTerms][2];
      query_halves<S::kTerms>(f, inv, b);
#pragma unroll
      for (int term = 0; term < S::kTerms; ++term) {
        if (S::kQueryInSmem) {
          if (s % kWarps == warp)
            q_smem[((term * NT + nt) * S::kSteps + s) * 32 + lane] = make_uint2(b[term][0], b[term][1]);
        } else {
          qb[S::kQueryInSmem ? 0 : nt][S::kQueryInSmem ? 0 : s][term][0] = b[term][0];
          qb[S::kQueryInSmem ? 0 : nt][S::kQueryInSmem ? 0 : s][term][1] = b[term][1];
        }
      }
    }
    const float mul = ldexpf(1.f, e) * p.scale_log2;
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
      s_mul[nt][e2] = __shfl_sync(0xffffffffu, mul, (2 * tq + e2) * 4);
      // columns without a row have scores of zero; as rows that see everything they stay on the
      // common path
      const int row2 = nt * 8 + 2 * tq + e2;
      vis[nt][e2] = row2 < nrows ? visible(row2) : INT32_MAX;
    }
  }
  const int vis_all = visible(0);  // tokens that every row sees
  keep_scales(lane);
  if (S::kQueryInSmem) __syncthreads();

  float m_run[NT][2], l_run[NT][2];
  float acc[NT][S::kTiles][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt][0] = m_run[nt][1] = -INFINITY;
    l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][t][e] = 0.f;
  }
  const int krow = (g >> 1) + 4 * (g & 1);  // token of score row g; row g + 8 holds token krow + 8

  int stage = 0;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    if ((i & 31) == 0) {
      if (i > 0) place = place_next;
      base = i;
      place_next = locate(i + 32 + lane);
    }
    if ((i & 31) == 8) load_scales(i - 8 + 32 + lane, place_next);
    if ((i & 31) == 24) keep_scales(i - 24 + 32 + lane);
    const int ahead = i + S::kStages - 1;
    issue(ahead, stage == 0 ? S::kStages - 1 : stage - 1);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    const uint8_t* kt = ring + stage * S::kStageBytes;
    const uint8_t* vt = kt + 16 * D;

    // ---- scores: c[0..1] token g of rows 2 tq, 2 tq + 1; c[2..3] token g + 8
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = 0.f;
#pragma unroll
    for (int c = 0; c < (S::kSteps + 3) / 4; ++c) {
      uint32_t w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (c < D / 64) {
          const uint4 v = *reinterpret_cast<const uint4*>(kt + tile_offset<D>(krow + 8 * h, c * 64 + tq * 16));
          w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < S::kSteps - 4 * c && j < 4; ++j)
            w[h][j] = *reinterpret_cast<const uint32_t*>(kt + tile_offset<D>(krow + 8 * h, c * 64 + j * 16 + tq * 4));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = 4 * c + j;
        if (s < S::kSteps) {
          const uint32_t a[4] = {codes_to_half2(w[0][j]), codes_to_half2(w[1][j]), codes_to_half2(w[0][j] >> 8),
                                 codes_to_half2(w[1][j] >> 8)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int term = 0; term < S::kTerms; ++term) {
              if (S::kQueryInSmem) {
                const uint2 b = q_smem[((term * NT + nt) * S::kSteps + s) * 32 + lane];
                mma_half(sc[nt], a, b.x, b.y);
              } else {
                const auto& b = qb[S::kQueryInSmem ? 0 : nt][S::kQueryInSmem ? 0 : s][term];
                mma_half(sc[nt], a, b[0], b[1]);
              }
            }
        }
      }
    }

    // ---- weights
    const float4 mt = meta[i & 63];
    const int tok0 = (first + kWarps * i) * 16;
    const bool partial = tok0 + 16 > vis_all;
    uint32_t pb[NT][S::kTerms][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mul[2] = {mt.x * s_mul[nt][0], mt.x * s_mul[nt][1]};
      float x[4];  // base-2 exponents against the running maximum
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(sc[nt][e], mul[e & 1], mt.y - m_run[nt][e & 1]);
      if (partial) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tok0 + krow + 8 * (e >> 1) >= vis[nt][e & 1]) x[e] = -INFINITY;
      }
      // NaN - as for a row that has no maximum yet - compares false: such rows come here too
      const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      if (__any_sync(0xffffffffu, !(top <= kRescaleSlack))) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float y0 = tok0 + krow < vis[nt][e] ? fmaf(sc[nt][e], mul[e], mt.y) : -INFINITY;
          const float y1 = tok0 + krow + 8 < vis[nt][e] ? fmaf(sc[nt][e + 2], mul[e], mt.y) : -INFINITY;
          float mx = fmaxf(y0, y1);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          float& m = m_run[nt][e];
          if (mx > m + kRescaleSlack) {
            const float alpha = m == -INFINITY ? 0.f : exp2_approx(m - mx);
            m = mx;
            l_run[nt][e] *= alpha;
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
              acc[nt][t][e] *= alpha;
              acc[nt][t][e + 2] *= alpha;
            }
          }
          // a row that has seen no token yet has m = -inf, and -inf - m would be a NaN
          x[e] = y0 == -INFINITY ? -INFINITY : y0 - m;
          x[e + 2] = y1 == -INFINITY ? -INFINITY : y1 - m;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = exp2_approx(x[e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) l_run[nt][e] = fmaf(x[e] + x[e + 2], mt.z, l_run[nt][e]);
#pragma unroll
      for (int term = 0; term < S::kTerms; ++term) {
        pb[nt][term][0] = transpose8(pack_half2(x[0], x[1]));
        pb[nt][term][1] = transpose8(pack_half2(x[2], x[3]));
        if (term + 1 < S::kTerms) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] -= __half2float(__float2half_rn(x[e]));
        }
      }
    }

    // ---- out^T += V^T w^T. `word`: 4 neighbouring dims (columns n .. n + 3) of the tokens
    // tq, tq + 4, tq + 8, tq + 12
    auto product = [&](uint32_t t0, uint32_t t1, uint32_t t2, uint32_t t3, int n) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tile = n / 2 + half;
        if (tile < S::kTiles) {
          // two tokens side by side: (dim, dim + 1) of one, then of the other
          const uint32_t lo = __byte_perm(t0, t1, half ? 0x7632 : 0x5410);
          const uint32_t hi = __byte_perm(t2, t3, half ? 0x7632 : 0x5410);
          const uint32_t a[4] = {codes_to_half2(lo), codes_to_half2(lo >> 8), codes_to_half2(hi), codes_to_half2(hi >> 8)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int term = 0; term < S::kTerms; ++term) mma_half(acc[nt][tile], a, pb[nt][term][0], pb[nt][term][1]);
        }
      }
    };
    constexpr int k16 = D / 128, k8 = (D % 128) / 64, k4 = (D % 64) / 32, k2 = (D % 32) / 16;
#pragma unroll
    for (int c = 0; c < k16; ++c) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint4*>(vt + tile_offset<D>(tq + 4 * e, c * 128 + g * 16));
      product(v[0].x, v[1].x, v[2].x, v[3].x, 16 * c);
      product(v[0].y, v[1].y, v[2].y, v[3].y, 16 * c + 4);
      product(v[0].z, v[1].z, v[2].z, v[3].z, 16 * c + 8);
      product(v[0].w, v[1].w, v[2].w, v[3].w, 16 * c + 12);
    }
    if (k8) {
      constexpr int b = k16 * 128;
      uint2 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint2*>(vt + tile_offset<D>(tq + 4 * e, b + g * 8));
      product(v[0].x, v[1].x, v[2].x, v[3].x, b / 8);
      product(v[0].y, v[1].y, v[2].y, v[3].y, b / 8 + 4);
    }
    if (k4) {
      constexpr int b = k16 * 128 + k8 * 64;
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint32_t*>(vt + tile_offset<D>(tq + 4 * e, b + g * 4));
      product(v[0], v[1], v[2], v[3], b / 8);
    }
    if (k2) {
      constexpr int b = k16 * 128 + k8 * 64 + k4 * 32;
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint16_t*>(vt + tile_offset<D>(tq + 4 * e, b + g * 2));
      product(v[0], v[1], v[2], v[3], b / 8);
    }
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    __syncwarp();  // every lane is done with the stage before it is filled again
  }
  cp_async_wait<0>();

  // ---- the warps' sums meet: m, l, acc per row, then one thread per (row, dim)
  __syncthreads();  // the rings are free
  float* sums = reinterpret_cast<float*>(smem);            // [warp][row][D]
  float* ml = sums + kWarps * S::kRows * D;                // [warp][row][2]
  float* cta_sum = ml + kWarps * S::kRows * 2;             // [row][D]
  float* cta_ml = cta_sum + S::kRows * D;                  // [row][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[nt][e];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int row = nt * 8 + 2 * tq + e;
      if (row < nrows) {
        if (g == 0) *reinterpret_cast<float2*>(ml + (warp * S::kRows + row) * 2) = make_float2(m_run[nt][e], l);
        float* dst = sums + (warp * S::kRows + row) * D;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
          dst[v_dim<D>(2 * t, g)] = acc[nt][t][e];
          dst[v_dim<D>(2 * t + 1, g)] = acc[nt][t][e + 2];
        }
      }
    }
  __syncthreads();
  const int clusters = p.num_splits / p.cluster;
  auto finish = [&](int row, int d, float m, float l, float o) {
    const int vrow = row0 + row, token = vrow / group;
    const int64_t out_row = req.q_begin + token;
    const int head = kvh * group + vrow - token * group;
    if (clusters == 1) {
      // l is a NaN where a score was: the row then is one, as in a plain softmax
      store_elem(static_cast<T*>(p.out) + out_row * p.out_stride + (int64_t)head * D + d, l == 0.f ? 0.f : o / l);
    } else {
      const int64_t item = (out_row * p.num_heads + head) * clusters + split / p.cluster;
      p.ws_acc[item * D + d] = o;
      if (d == 0) p.ws_ml[item] = make_float2(m, l);
    }
  };
  for (int i = threadIdx.x; i < nrows * D; i += kThreads) {
    const int row = i / D, d = i - row * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[(w * S::kRows + row) * 2]);
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = merge_factor(ml[(w * S::kRows + row) * 2], m);
      l = fmaf(f, ml[(w * S::kRows + row) * 2 + 1], l);
      o = fmaf(f, sums[(w * S::kRows + row) * D + d], o);
    }
    if (p.cluster == 1) {
      finish(row, d, m, l, o);
    } else {
      cta_sum[i] = o;
      if (d == 0) *reinterpret_cast<float2*>(cta_ml + 2 * row) = make_float2(m, l);
    }
  }
  if (p.cluster == 1) return;

  // ---- the cluster's sums meet: each CTA finishes a share of the (row, dim) pairs
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int rank = split % p.cluster;
  for (int i = rank * kThreads + threadIdx.x; i < nrows * D; i += p.cluster * kThreads) {
    const int row = i / D, d = i - row * D;
    float m = -INFINITY;
    float2 part[kMaxCluster];
    float val[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      if (c < p.cluster) {
        part[c] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(cta_ml, c) + 2 * row);
        val[c] = cluster.map_shared_rank(cta_sum, c)[i];
        m = fmaxf(m, part[c].x);
      }
    }
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      if (c < p.cluster) {
        const float f = merge_factor(part[c].x, m);
        l = fmaf(f, part[c].y, l);
        o = fmaf(f, val[c], o);
      }
    }
    finish(row, d, m, l, o);
  }
  cluster.sync();  // no CTA leaves while another still reads its sums
}

// Adds the clusters' pieces of the rows. grid: (requests, query tokens of the longest one, heads);
// one thread a dim.
template <typename T>
__global__ void combine_int8_kernel(const Int8AttnParams p, int D) {
  griddep_wait();
  const RequestSpan req = request_span(p, blockIdx.x);
  if ((int)blockIdx.y >= req.rows) return;
  const int h = blockIdx.z;
  const int64_t row = req.q_begin + blockIdx.y;
  const int clusters = p.num_splits / p.cluster;
  const int64_t item = (row * p.num_heads + h) * clusters;
  float m = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < clusters; ++s) m = fmaxf(m, p.ws_ml[item + s].x);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float l = 0.f, o = 0.f;
#pragma unroll 4
    for (int s = 0; s < clusters; ++s) {
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
  const int64_t clusters = plan->num_splits / plan->cluster;
  if (clusters <= 1) return 0;
  const int64_t items = (int64_t)plan->total_q * plan->num_heads * clusters;
  return acc_bytes(items, plan->head_dim) + items * 8;
}

int64_t row_chunks(const vfl_attention_int8_plan* plan) {
  return ceil_div((int64_t)plan->max_q_len * (plan->num_heads / plan->num_kv_heads), (int64_t)plan->rows_per_cta);
}

// Whether 16 query rows a CTA are built: past 128 dims their sums do not fit the registers.
bool rows16_built(int head_dim) { return head_dim <= 128; }

template <typename T, int D, int NT>
int launch(const Int8AttnParams& p, dim3 grid, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  auto kern = paged_attention_int8_kernel<T, D, NT>;
  constexpr int kSmem = Shape<T, D, NT>::kSmem;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), kSmem, smem_done);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = p.cluster;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "attention_with_kv_cache_int8 launch");
}

template <typename T, int NT>
int launch_dim(const Int8AttnParams& p, int D, dim3 grid, cudaStream_t s) {
  switch (D) {
    case 32: return launch<T, 32, NT>(p, grid, s);
    case 48: return launch<T, 48, NT>(p, grid, s);
    case 64: return launch<T, 64, NT>(p, grid, s);
    case 80: return launch<T, 80, NT>(p, grid, s);
    case 96: return launch<T, 96, NT>(p, grid, s);
    case 112: return launch<T, 112, NT>(p, grid, s);
    case 128: return launch<T, 128, NT>(p, grid, s);
    default: break;
  }
  if constexpr (NT == 1) {
    switch (D) {
      case 160: return launch<T, 160, 1>(p, grid, s);
      case 192: return launch<T, 192, 1>(p, grid, s);
      case 224: return launch<T, 224, 1>(p, grid, s);
      case 256: return launch<T, 256, 1>(p, grid, s);
      default: return launch<T, 512, 1>(p, grid, s);
    }
  }
  return fail(VFL_ERR_UNSUPPORTED, "attention_int8: 16 rows a CTA at head_dim %d", D);
}

template <typename T>
int launch_rows(const Int8AttnParams& p, int D, int rows, dim3 grid, cudaStream_t s) {
  return rows == 16 ? launch_dim<T, 2>(p, D, grid, s) : launch_dim<T, 1>(p, D, grid, s);
}

// Dynamic shared memory of a CTA (upper bound over the types).
int smem_bytes(int D, int rows) {
  const int ring = kWarps * 32 * D * (D <= 128 ? 4 : (D <= 256 ? 3 : 2));
  const int merge = (kWarps + 1) * rows * (D + 2) * 4;
  return (ring > merge ? ring : merge) + kWarps * 64 * 16 + (2 * rows * D > 1024 ? 4 * rows * D : 0);
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
  const int c = plan->cluster;
  if (!(c == 1 || c == 2 || c == 4 || c == kMaxCluster) || plan->num_splits < 1 || plan->num_splits > 65535 ||
      plan->num_splits % c != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan splits %d in clusters of %d", plan->num_splits, c);
  if (!(plan->rows_per_cta == 8 || (plan->rows_per_cta == 16 && rows16_built(plan->head_dim))))
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan rows_per_cta %d", plan->rows_per_cta);
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
  const int64_t group = num_heads / num_kv_heads;
  int64_t max_q = 0, max_seq = 0;
  for (int r = 0; r < num_reqs; ++r) {
    const int64_t n = seq_lens_host[r];
    const int64_t ql = query_start_loc_host ? (int64_t)query_start_loc_host[r + 1] - query_start_loc_host[r] : 1;
    if (n < 0) return fail(VFL_ERR_INVALID_ARGUMENT, "seq_lens[%d] = %lld < 0", r, (long long)n);
    if (ql < 0) return fail(VFL_ERR_INVALID_ARGUMENT, "query_start_loc decreases at %d", r);
    max_q = ql > max_q ? ql : max_q;
    max_seq = n > max_seq ? n : max_seq;
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

  plan->rows_per_cta = max_q * group > 8 && rows16_built(head_dim) ? 16 : 8;
  int64_t items = 0;
  for (int r = 0; r < num_reqs; ++r) {
    const int64_t ql = query_start_loc_host ? (int64_t)query_start_loc_host[r + 1] - query_start_loc_host[r] : 1;
    if (seq_lens_host[r] > 0) items += ceil_div(ql * group, (int64_t)plan->rows_per_cta) * num_kv_heads;
  }

  // Splits: as many as give every CTA slot an item, each of at least a tile a warp.
  int per_sm = kSmemPerSM / (smem_bytes(head_dim, plan->rows_per_cta) + 1024);
  per_sm = per_sm < 1 ? 1 : (per_sm > 4 ? 4 : per_sm);
  const int64_t slots = (int64_t)kNumSMs * per_sm;
  const int64_t tiles = ceil_div(max_seq, (int64_t)16);
  int64_t splits = 1;
  if (items > 0) {
    const int64_t by_len = tiles / kWarps;
    splits = slots / items;
    splits = splits < by_len ? splits : by_len;
  }
  int cluster = 1;
  while (cluster < kMaxCluster && 2 * cluster <= splits) cluster *= 2;
  plan->cluster = cluster;
  plan->num_splits = static_cast<int32_t>(cluster < kMaxCluster ? cluster : splits / kMaxCluster * kMaxCluster);
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
  if (num_blocks > 0 && num_blocks * plan->num_kv_heads > INT32_MAX / (plan->block_size / 16))
    return fail(VFL_ERR_UNSUPPORTED, "attention_int8: %lld blocks are more than the kernel indexes", (long long)num_blocks);
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
  p.num_splits = plan->num_splits;
  p.cluster = plan->cluster;
  p.scale_log2 = scale * kLog2e;
  const int clusters = plan->num_splits / plan->cluster;
  const int64_t items = (int64_t)plan->total_q * H * clusters;
  p.ws_acc = static_cast<float*>(workspace);
  p.ws_ml = clusters > 1
                ? reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + acc_bytes(items, D)) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(plan->num_reqs * plan->num_kv_heads, (unsigned)row_chunks(plan), plan->num_splits);
  st = plan->dtype == VFL_DTYPE_F32 ? launch_rows<float>(p, D, plan->rows_per_cta, grid, s)
                                    : launch_rows<__nv_bfloat16>(p, D, plan->rows_per_cta, grid, s);
  if (st || clusters == 1) return st;
  const dim3 cgrid(plan->num_reqs, plan->max_q_len, H);
  const int threads = D <= 64 ? 64 : 128;
  if (plan->dtype == VFL_DTYPE_F32)
    combine_int8_kernel<float><<<cgrid, threads, 0, s>>>(p, D);
  else
    combine_int8_kernel<__nv_bfloat16><<<cgrid, threads, 0, s>>>(p, D);
  return cuda_status(cudaGetLastError(), "attention_int8 combine launch");
}

}  // extern "C"
