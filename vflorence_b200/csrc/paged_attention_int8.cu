// Attention over a paged K/V cache held in 8 bits with a scale for each block and head.
//
// For query row i of head h with visible tokens t (K codes kc_t, V codes vc_t in a block b whose
// scales are ks_b, vs_b):
//     s_t = scale * ks_b * (q . kc_t),   out = sum_t e^(s_t) vs_b vc_t / sum_t e^(s_t).
// A scale is one number for a tile of tokens, so neither product multiplies a cached element by
// it: ks_b goes onto the score, and vs_b into the exponent. With base-2 scores s' = s log2 e and
//     w_t = 2^(s'_t + log2 vs_b - M),  M below the running maximum of s'_t + log2 vs_b,
// out = sum w_t vc_t / sum (w_t / vs_b). Both sums and M are float32. w is rounded to half precision for
// its product alone (float32 queries: to a pair of halves, 2^-22 of it). M is kept 7 to 15 below the
// maximum, so that the largest weight is near the upper end of a half's range and every weight is held
// to 2^-32 of it or better: n tokens that small beside a large one are off by n 2^-32 of the largest |v|.
//
// Scores: K's codes enter m16n8k32 integer instructions as they are. A query row is brought to
// whole numbers of 2^-22 (bfloat16) or 2^-30 (float32) of a power of two above its largest
// element, held as 3 or 4 planes of 8 bits: elements down to 2^-15 (2^-7) of the row's largest are
// exact, smaller ones are rounded to 2^-23 (2^-31) of that power, 13 (21) bits beside a channel a
// thousand times larger. The sums are exact integers. A plane less takes 3 to 8 % off the times below
// and leaves 5 (13) bits. Outputs: V's codes are exact in half precision and meet w in m16n8k16 half
// instructions with float32 sums.
//
// Bound: HBM, 2 D bytes a token and K/V head, and close behind it the integer pipe that turns V's
// codes into halves. What the layout buys: scores are taken as K q^T (16 tokens x 8 query rows)
// and outputs as V^T w^T (16 dims x 8 rows), so that the cached elements fill the instructions'
// 16-row side and a few query rows their 8-column side. The index maps are free to choose,
// because q . kc sums over dims in any order and the softmax over tokens in any order: a lane's
// K operands are 16 neighbouring bytes of two tokens, its V operands come transposed out of a
// byte matrix load, and two 8 x 8 transpositions in registers turn scores into weights.
//
// One CTA takes a request, a K/V head, 8 or 16 query rows (those of the heads that share the K/V
// head, of all the request's query tokens) and a range of 16-token tiles. Each warp streams its
// own tiles through its own ring of cp.async stages; the warps' partial sums meet in shared
// memory at the end. Long contexts of few requests are cut over a cluster of up to 8 CTAs, whose
// sums meet in distributed shared memory, and over more clusters where that is not enough: then
// a second launch adds the clusters' pieces.
//
// Measured, bfloat16, head_dim 64: 256 requests of 1 to 4096 tokens x 16 heads 180 us, 1079 MB at 6.0
// TB/s (0.93 of a plain copy; 0.68 of the issue slots); 64 requests of 585 x 12 heads, three rows each,
// 17.5 us (58 MB), one request of 577 6.2 us: start, joins and drain.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kMaxWarps = 4;
constexpr int kMaxCluster = 8;
constexpr int kSmemPerSM = 227 * 1024;
constexpr float kMinScale = 7.888609052210118e-31f;     // 2^-100: smaller V scales count as it
constexpr float kScaleRange = 8.077935669463161e-28f;   // 2^-90: also those this much below the largest
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLift = 7.f;            // log2 of the largest weight when its token sets the maximum
constexpr float kRescaleSlack = 15.f;   // and the most before another one does: 2^15 is a half
constexpr float kSumUnit = 0.000244140625f;  // 2^-12, of the sums of w / vs: 2^15 times 2^100 times a context's tokens is past float32

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

// Where byte `byte` of row `row` of a 16 x D byte tile lies: the 16-byte chunks of a 128-byte line
// are permuted so that the rows that one phase of a warp's loads reads (pairs of K rows 2 apart,
// eight neighbouring V rows) fall into different banks.
template <int D>
__device__ __forceinline__ int tile_offset(int row, int byte) {
  int x = 0;
  if (D % 128 == 0) x = ((row & 2) << 1) | ((row & 4) >> 1) | (row & 1);
  if (D == 64) x = ((row >> 1) & 3) | ((row & 2) << 1);
  if (D == 32) x = (row >> 2) & 1;
  return (row * D + byte) ^ (x << 4);
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

// Whole numbers: A 16 x 32 (or 16 x 16) of K codes, B of 8-bit query digits.
__device__ __forceinline__ void mma_int_k32(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first of a chain: its sums start at `from`.
__device__ __forceinline__ void mma_int_k32_from(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1, int from) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(from));
}
__device__ __forceinline__ void mma_int_k16(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(b0));
}

// 16 x 16 byte matrices whose rows the lanes 0-15 (16-31) address, transposed: lane 4g + tq gets
// rows 4 tq .. 4 tq + 3 of column g in r[0] (r[2]) and of column g + 8 in r[1] (r[3]).
__device__ __forceinline__ void load_bytes_trans_x2(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void load_bytes_trans_x1(uint32_t addr, uint32_t& r0, uint32_t& r1) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x1.trans.shared.b8 {%0,%1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
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
  static constexpr int kPlanes = sizeof(T) == 4 ? 4 : 3;  // 8-bit digits of a query element
  static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;   // halves that make up a weight
  static constexpr int kWords = D / 16;                   // 4-dim words a lane holds of a row
  static constexpr int kTiles = D / 16;                   // m16 tiles of the output
  static constexpr int kStageBytes = 2 * 16 * D;
  static constexpr int kStages = D <= 128 ? 4 : 2;
  static constexpr int kRingBytes = kStages * kStageBytes;
  // CTAs of four warps that an SM's registers are to hold (96, 128 and 168 a lane)
  static constexpr int kMinCtas = D * NT <= 64 ? 5 : (D * NT <= 128 ? (sizeof(T) == 4 ? 3 : 4) : (D <= 128 ? 2 : 1));
  // query digits stay in registers up to this many, in shared memory past it
  static constexpr bool kQueryInSmem = kPlanes * NT * kWords > 32;
  // the warps' rings, later their sums [warp][row][D], the CTA's [row][D] and all their (m, l)
  __device__ __forceinline__ static int region(int warps) {
    const int merge = (warps + 1) * kRows * (D + 2) * 4;
    return warps * kRingBytes > merge ? warps * kRingBytes : merge;
  }
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

__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}
__device__ __forceinline__ void add_scaled(float4& o, float f, const float4& v) {
  o.x = fmaf(f, v.x, o.x);
  o.y = fmaf(f, v.y, o.y);
  o.z = fmaf(f, v.z, o.z);
  o.w = fmaf(f, v.w, o.w);
}

// Root of the factor of a piece with maximum `m` in a sum with maximum `m_all`. The sums of weights take
// it twice: theirs may be within range where the factor is not (blocks of zeros before others). A piece
// without a maximum holds zeros (nothing visible) or NaNs (every score a NaN), and either is to be kept.
__device__ __forceinline__ float merge_root(float m, float m_all) {
  return m == -INFINITY ? 1.f : exp2_approx(0.5f * (m - m_all));
}

// First dim of word `w` (4 dims) of a row that lane group thread tq holds: whole groups of 64 dims
// give a thread 16 neighbouring bytes, a group of 32 gives 8, one of 16 gives 4.
template <int D>
__device__ __forceinline__ int k_dim(int w, int tq) {
  constexpr int k64 = D / 64, k32 = (D % 64) / 32;
  if (w < 4 * k64) return (w >> 2) * 64 + tq * 16 + (w & 3) * 4;
  if (w < 4 * k64 + 2 * k32) return k64 * 64 + tq * 8 + (w - 4 * k64) * 4;
  return k64 * 64 + k32 * 32 + tq * 4;
}

// 2^e for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// A lane's place in the fragments.
struct Lane {
  int lane, g, tq, krow;  // krow: token of score row g; row g + 8 holds token krow + 1
  __device__ __forceinline__ Lane() : lane(threadIdx.x & 31), g(lane >> 2), tq(lane & 3), krow(2 * g) {}
};

// What a lane knows of the query rows: their digits (or where in shared memory they are), the
// factor of their scores, the tokens they see.
template <typename T, int D, int NT>
struct Query {
  using S = Shape<T, D, NT>;
  uint32_t digits[S::kQueryInSmem ? 1 : NT * S::kPlanes * S::kWords];
  const uint32_t* smem;
  float mul[NT][2];  // of the rows 2 tq, 2 tq + 1 whose scores this lane holds
  int vis[NT][2];
  int vis_all;       // tokens that every row sees

  // word `w` of row g of n8 tile nt, plane `plane` (0: the highest digits)
  __device__ __forceinline__ uint32_t word(int nt, int plane, int w, int lane) const {
    const int at = (nt * S::kPlanes + plane) * S::kWords + w;
    return S::kQueryInSmem ? smem[at * 32 + lane] : digits[S::kQueryInSmem ? 0 : at];
  }

  // Rows row0 .. row0 + nrows of a request's rows of one K/V head. `visible(i)`: tokens that row i
  // of these sees. Warp `warp` stores its share of the digits where they go to shared memory (the
  // caller syncs).
  template <typename V>
  __device__ __forceinline__ void load(const Int8AttnParams& p, const Lane& ln, int warp, int warps, int q_begin, int kvh,
                                       int group, int row0, int nrows, const V& visible, uint32_t* q_smem) {
    smem = q_smem;
    vis_all = visible(0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + ln.g;
      const bool on = row < nrows;
      const int vrow = row0 + (on ? row : 0);
      const int token = vrow / group, head = kvh * group + vrow - token * group;
      const T* src = static_cast<const T*>(p.q) + (int64_t)(q_begin + token) * p.q_stride + (int64_t)head * D;
      constexpr int kHeld = S::kWords <= 8 ? S::kWords : 1;  // long rows are read twice
      float f[kHeld][4];
      float amax = 0.f;
      bool odd = false;  // an infinity or a NaN
      auto look = [&](const float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          amax = fmaxf(amax, fabsf(v[i]));
          odd |= !(fabsf(v[i]) <= FLT_MAX);
        }
      };
#pragma unroll
      for (int w = 0; w < S::kWords; ++w) {
        float(&v)[4] = f[w < kHeld ? w : 0];
        v[0] = v[1] = v[2] = v[3] = 0.f;
        if (on) load4(src + k_dim<D>(w, ln.tq), v);
        if (kHeld == 1) look(v);
      }
      if (kHeld > 1) {
#pragma unroll
        for (int w = 0; w < kHeld; ++w) look(f[w]);
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const bool bad = ((__ballot_sync(0xffffffffu, odd) >> (ln.lane & ~3)) & 15u) != 0;  // in this lane's row
      // 2^e > amax >= 2^(e-1), from the exponent bits
      const int e = max(-90, static_cast<int>(__float_as_uint(amax) >> 23) - 126);
      constexpr int kBits = 8 * S::kPlanes - 2;
      const float to_int = power_of_two(kBits - e);
#pragma unroll
      for (int w = 0; w < S::kWords; ++w) {
        if (S::kQueryInSmem && w % warps != warp) continue;
        float(&v)[4] = f[w < kHeld ? w : 0];
        if (kHeld == 1) {
          v[0] = v[1] = v[2] = v[3] = 0.f;
          if (on) load4(src + k_dim<D>(w, ln.tq), v);
        }
        // digits base 256 in [-128, 127]: with 128 added to each they are the bytes of a plain number, and
        // a byte loses the 128 again by flipping its top bit. Up to 2^22 adding 1.5 * 2^23 leaves the
        // whole number in the sum's mantissa
        constexpr uint32_t kBias = S::kPlanes == 4 ? 0x80808080u : 0x808080u;
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t whole = S::kPlanes == 4 ? (uint32_t)__float2int_rn(v[i] * to_int)
                                                 : __float_as_uint(fmaf(v[i], to_int, 12582912.f)) - 0x4b400000u;
          c[i] = (whole + kBias) ^ kBias;
        }
#pragma unroll
        for (int plane = 0; plane < S::kPlanes; ++plane) {
          constexpr uint32_t kPick[4] = {0x0040, 0x0051, 0x0062, 0x0073};  // byte 0, 1, 2, 3 of two words
          const uint32_t pick = kPick[S::kPlanes - 1 - plane];
          const uint32_t packed = __byte_perm(__byte_perm(c[0], c[1], pick), __byte_perm(c[2], c[3], pick), 0x5410);
          const int at = (nt * S::kPlanes + plane) * S::kWords + w;
          if (S::kQueryInSmem) {
            q_smem[at * 32 + ln.lane] = packed;
          } else {
            digits[S::kQueryInSmem ? 0 : at] = packed;
          }
        }
      }
      // a row with an infinity or a NaN scores NaN
      const float row_mul = bad ? NAN : p.scale_log2 * power_of_two(e - kBits);
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        mul[nt][e2] = __shfl_sync(0xffffffffu, row_mul, (2 * ln.tq + e2) * 4);
        // columns without a row have scores of zero; as rows that see everything they stay on
        // the common path
        const int row2 = nt * 8 + 2 * ln.tq + e2;
        vis[nt][e2] = row2 < nrows ? visible(row2) : INT32_MAX;
      }
    }
  }
};

// Running sums of a warp: maximum and sum of the rows 2 tq, 2 tq + 1 and out^T.
template <typename T, int D, int NT>
struct Sums {
  using S = Shape<T, D, NT>;
  float m[NT][2], l[NT][2];  // l in units of 2^12
  float acc[NT][S::kTiles][4];

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][t][e] = 0.f;
    }
  }

  // l over the lanes that share a row
  __device__ __forceinline__ void reduce() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
  }

  // One 16-token tile in shared memory: K codes at kt, V codes at vt (a shared address); mt = (ks,
  // log2 vs, 1 / vs); tok0: the tile's first position.
  __device__ __forceinline__ void tile(const uint8_t* kt, uint32_t vt, const float4& mt, int tok0,
                                       const Query<T, D, NT>& q, const Lane& ln) {
    const int tq = ln.tq, krow = ln.krow;
    // ---- scores: c[0..1] token krow of rows 2 tq, 2 tq + 1; c[2..3] token krow + 1
    // A plane's sum is below 2^22 up to 256 dims: started at the bits of 1.5 * 2^23, it is that float's mantissa,
    // and a subtraction turns it into a number where a conversion runs at a quarter of the rate (512 x 577
    // float32 125 -> 121 us; bfloat16, with fewer planes, 103 -> 106). Otherwise the two highest planes are
    // converted as one integer (2^14 * 127 * 512 < 2^31).
    constexpr bool kMantissa = sizeof(T) == 4 && D <= 256;
    constexpr int kFrom = kMantissa ? 0x4b400000 : 0;
    auto number = [](int sum) { return kMantissa ? __int_as_float(sum) - 12582912.f : (float)sum; };
    int si[NT][S::kPlanes][4];
    constexpr int k64 = D / 64, k32 = (D % 64) / 32, k16 = (D % 32) / 16;
    auto pair = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, int w) {  // words w, w + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pl = 0; pl < S::kPlanes; ++pl) {
          if (w == 0)
            mma_int_k32_from(si[nt][pl], a0, a1, a2, a3, q.word(nt, pl, w, ln.lane), q.word(nt, pl, w + 1, ln.lane), kFrom);
          else
            mma_int_k32(si[nt][pl], a0, a1, a2, a3, q.word(nt, pl, w, ln.lane), q.word(nt, pl, w + 1, ln.lane));
        }
    };
#pragma unroll
    for (int c = 0; c < k64; ++c) {
      const uint4 a = *reinterpret_cast<const uint4*>(kt + tile_offset<D>(krow, c * 64 + tq * 16));
      const uint4 b = *reinterpret_cast<const uint4*>(kt + tile_offset<D>(krow + 1, c * 64 + tq * 16));
      pair(a.x, b.x, a.y, b.y, 4 * c);
      pair(a.z, b.z, a.w, b.w, 4 * c + 2);
    }
    if (k32) {
      const uint2 a = *reinterpret_cast<const uint2*>(kt + tile_offset<D>(krow, k64 * 64 + tq * 8));
      const uint2 b = *reinterpret_cast<const uint2*>(kt + tile_offset<D>(krow + 1, k64 * 64 + tq * 8));
      pair(a.x, b.x, a.y, b.y, 4 * k64);
    }
    if (k16) {
      const uint32_t a = *reinterpret_cast<const uint32_t*>(kt + tile_offset<D>(krow, k64 * 64 + k32 * 32 + tq * 4));
      const uint32_t b = *reinterpret_cast<const uint32_t*>(kt + tile_offset<D>(krow + 1, k64 * 64 + k32 * 32 + tq * 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pl = 0; pl < S::kPlanes; ++pl)
          mma_int_k16(si[nt][pl], a, b, q.word(nt, pl, 4 * k64 + 2 * k32, ln.lane));
    }
    // digits to scores
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[nt][e] = kMantissa ? fmaf(number(si[nt][0][e]), 256.f, number(si[nt][1][e]))
                              : (float)(si[nt][0][e] * 256 + si[nt][1][e]);
#pragma unroll
        for (int pl = 2; pl < S::kPlanes; ++pl) sc[nt][e] = fmaf(sc[nt][e], 256.f, number(si[nt][pl][e]));
      }

    // ---- weights
    const bool partial = tok0 + 16 > q.vis_all;
    uint32_t pb[NT][S::kTerms][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mul[2] = {mt.x * q.mul[nt][0], mt.x * q.mul[nt][1]};
      float x[4];  // base-2 exponents against the running maximum
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(sc[nt][e], mul[e & 1], mt.y - m[nt][e & 1]);
      if (partial) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tok0 + krow + (e >> 1) >= q.vis[nt][e & 1]) x[e] = -INFINITY;
      }
      // NaN - as for a row that has no maximum yet - compares false: such rows come here too
      const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      if (__any_sync(0xffffffffu, !(top <= kRescaleSlack))) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float y0 = tok0 + krow < q.vis[nt][e] ? fmaf(sc[nt][e], mul[e], mt.y) : -INFINITY;
          const float y1 = tok0 + krow + 1 < q.vis[nt][e] ? fmaf(sc[nt][e + 2], mul[e], mt.y) : -INFINITY;
          float mx = fmaxf(y0, y1);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          float& mr = m[nt][e];
          if (mx > mr + kRescaleSlack) {
            const float to = mx - kLift;
            const float root = mr == -INFINITY ? 0.f : exp2_approx(0.5f * (mr - to)), alpha = root * root;
            mr = to;
            l[nt][e] = l[nt][e] * root * root;
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
              acc[nt][t][e] *= alpha;
              acc[nt][t][e + 2] *= alpha;
            }
          }
          // a row that has seen no token yet has m = -inf, and -inf - m would be a NaN
          x[e] = y0 == -INFINITY ? -INFINITY : y0 - mr;
          x[e + 2] = y1 == -INFINITY ? -INFINITY : y1 - mr;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = exp2_approx(x[e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) l[nt][e] = fmaf((x[e] + x[e + 2]) * kSumUnit, mt.z, l[nt][e]);
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

    // ---- out^T += V^T w^T. A lane's word holds tokens 4 tq .. 4 tq + 3 of a dim: bytes 0 and 2 are
    // the tokens of score rows 2 tq, 2 tq + 1, bytes 1 and 3 those of rows 2 tq + 8, 2 tq + 9
    auto product = [&](uint32_t lo, uint32_t hi, int t) {  // dims g and g + 8 of m16 tile t
      const uint32_t a[4] = {codes_to_half2(lo), codes_to_half2(hi), codes_to_half2(lo >> 8), codes_to_half2(hi >> 8)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int term = 0; term < S::kTerms; ++term) mma_half(acc[nt][t], a, pb[nt][term][0], pb[nt][term][1]);
    };
#pragma unroll
    for (int t = 0; t + 1 < S::kTiles; t += 2) {  // lanes 0-15 address the rows of tile t, 16-31 of t + 1
      uint32_t r[4];
      load_bytes_trans_x2(vt + tile_offset<D>(ln.lane & 15, t * 16 + (ln.lane & 16)), r);
      product(r[0], r[1], t);
      product(r[2], r[3], t + 1);
    }
    if (S::kTiles % 2) {
      uint32_t r0, r1;
      load_bytes_trans_x1(vt + tile_offset<D>(ln.lane & 15, (S::kTiles - 1) * 16), r0, r1);
      product(r0, r1, S::kTiles - 1);
    }
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kMaxWarps * 32, Shape<T, D, NT>::kMinCtas) paged_attention_int8_kernel(const Int8AttnParams p) {
  using S = Shape<T, D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const Lane ln;
  const int warp = threadIdx.x >> 5, lane = ln.lane, warps = blockDim.x >> 5;
  const int region = S::region(warps);
  const int r = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - r * p.num_kv_heads;
  const int split = blockIdx.z;
  const int bs = p.block_size, tpb = bs >> 4;
  const RequestSpan req = request_span(p, r);
  // an unsplit context's first tiles do not depend on its length: their table entries come with it
  const int32_t* table = p.table + (int64_t)r * p.table_stride;
  int entry = 0;
  if (p.num_splits == 1) {
    const int col = (warp + warps * lane) / tpb;
    if (col < p.table_cols) entry = __ldg(table + col);
  }
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

  // ---- this warp's tiles: tile_begin + warp + warps * i. A lane keeps the position of one of
  // 32 tiles in units of 16 tokens of the pools, and of the next 32.
  const int first = tile_begin + warp;
  const int count = tile_end > first ? ceil_div(tile_end - first, warps) : 0;
  auto locate = [&](int i, bool have_entry) {
    if (i >= count) return 0;
    const int tile = first + warps * i;
    const int col = tpb == 1 ? tile : tile / tpb;
    int b = have_entry ? entry : __ldg(table + col);
    if (b < 0 || b >= p.num_blocks) {
      report(p.err, VFL_DEVERR_BLOCK_ID);
      b = 0;
    }
    return (b * p.num_kv_heads + kvh) * tpb + (tile - col * tpb);  // the host checked that it fits
  };
  int place = locate(lane, p.num_splits == 1), place_next = 0;
  uint8_t* ring = smem + warp * S::kRingBytes;
  const uint32_t ring_u32 = smem_u32(ring);
  // where this lane's 16-byte pieces of a tile go, within a stage
  constexpr int kPieces = (D + 31) / 32;
  const int8_t* k_lane = p.k_cache + lane * 16;
  const int8_t* v_lane = p.v_cache + lane * 16;
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
      const int8_t* ks = k_lane + (int64_t)at * (16 * D);
      const int8_t* vs = v_lane + (int64_t)at * (16 * D);
      const uint32_t to = stage * S::kStageBytes;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        if (D % 32 == 0 || j * 32 + lane < D) {
          cp_async16(piece_at[j] + to, ks + j * 512);
          cp_async16(piece_at[j] + to + 16 * D, vs + j * 512);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i, i);

  // ---- the tiles' scales: (ks, log2 vs, 1 / vs), 64 tiles of them in shared memory
  float4* meta = reinterpret_cast<float4*>(smem + region) + warp * 64;
  float ks_next = 0.f, vs_next = 0.f, largest_vs = 0.f;
  auto load_scales = [&](int i, int at) {
    ks_next = vs_next = 0.f;
    if (i < count) {
      const int row = tpb == 1 ? at : at / tpb;
      ks_next = __ldg(p.k_scale + row);
      vs_next = __ldg(p.v_scale + row);
    }
  };
  auto keep_scales = [&](int i) {
    // A block of zeros has scale 0. Its tokens weigh in the sum of the weights alone: with a scale far
    // below the others' they leave the maximum to the blocks that the output comes from, and their weights
    // are still within range of it.
    largest_vs = fmaxf(largest_vs, __uint_as_float(__reduce_max_sync(
        0xffffffffu, vs_next > 0.f && vs_next <= FLT_MAX ? __float_as_uint(vs_next) : 0u)));
    const float least = fmaxf(kMinScale, largest_vs * kScaleRange);
    const float vs = vs_next < least ? least : vs_next;  // a NaN stays one
    meta[i & 63] = make_float4(ks_next, log2f(vs), 1.f / vs, 0.f);
  };
  load_scales(lane, place);

  // ---- the query rows
  Query<T, D, NT> query;
  query.load(p, ln, warp, warps, req.q_begin, kvh, group, row0, nrows, visible,
             reinterpret_cast<uint32_t*>(smem + region + warps * 64 * 16));
  keep_scales(lane);
  if (S::kQueryInSmem) __syncthreads();
  Sums<T, D, NT> sum;
  sum.reset();

  // batches of 32 tiles (their places and scales come one batch ahead), in them turns of the ring
#pragma unroll 1
  for (; base < count; base += 32) {
    if (base > 0) place = place_next;
    place_next = locate(base + 32 + lane, false);
#pragma unroll 1
    for (int i0 = base; i0 < min(base + 32, count); i0 += S::kStages) {
      if (i0 - base == 8) load_scales(base + 32 + lane, place_next);
      if (i0 - base == 24) keep_scales(base + 32 + lane);
      const float4* mt = meta + (i0 & 63);
      const int tok0 = (first + warps * i0) * 16;
#pragma unroll
      for (int st = 0; st < S::kStages; ++st) {
        if (i0 + st < count) {
          issue(i0 + st + S::kStages - 1, (st + S::kStages - 1) % S::kStages);
          cp_async_wait<S::kStages - 1>();
          __syncwarp();
          sum.tile(ring + st * S::kStageBytes, ring_u32 + st * S::kStageBytes + 16 * D, mt[st],
                   tok0 + st * (warps * 16), query, ln);
          __syncwarp();  // every lane is done with the stage before it is filled again
        }
      }
    }
  }
  cp_async_wait<0>();

  // ---- the warps' sums meet: m, l, acc per row, then one thread per (row, dim)
  __syncthreads();  // the rings are free
  sum.reduce();
  float* sums = reinterpret_cast<float*>(smem);            // [warp][row][D]
  float* cta_sum = sums + warps * S::kRows * D;            // [row][D]
  float* ml = cta_sum + S::kRows * D;                      // [warp][row][2]
  float* cta_ml = ml + warps * S::kRows * 2;               // [row][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = nt * 8 + 2 * ln.tq + e;
      if (row < nrows) {
        if (ln.g == 0)
          *reinterpret_cast<float2*>(ml + (warp * S::kRows + row) * 2) = make_float2(sum.m[nt][e], sum.l[nt][e]);
        float* dst = sums + (warp * S::kRows + row) * D;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
          dst[16 * t + ln.g] = sum.acc[nt][t][e];
          dst[16 * t + ln.g + 8] = sum.acc[nt][t][e + 2];
        }
      }
    }
  __syncthreads();
  const int clusters = p.num_splits / p.cluster;
  // one row's sums, four dims a lane: the output, or the cluster's piece
  auto finish = [&](int row, float m, float l, auto&& sum_at) {
    const int vrow = row0 + row, token = vrow / group;
    const int64_t out_row = req.q_begin + token;
    const int head = kvh * group + vrow - token * group;
    if (clusters == 1) {
      T* dst = static_cast<T*>(p.out) + out_row * p.out_stride + (int64_t)head * D;
      // l is a NaN where a score was: the row then is one, as in a plain softmax
      const float inv = l == 0.f ? 0.f : 1.f / l;
      constexpr float c = kSumUnit;
      for (int d = lane * 4; d < D; d += 128) {
        const float4 o = sum_at(d);
        store4(dst + d, o.x * inv * c, o.y * inv * c, o.z * inv * c, o.w * inv * c);
      }
    } else {
      const int64_t item = (out_row * p.num_heads + head) * clusters + split / p.cluster;
      for (int d = lane * 4; d < D; d += 128) *reinterpret_cast<float4*>(p.ws_acc + item * D + d) = sum_at(d);
      if (lane == 0) p.ws_ml[item] = make_float2(m, l);
    }
  };
  for (int row = warp; row < nrows; row += warps) {
    float m = -INFINITY, l = 0.f, f[kMaxWarps];
#pragma unroll
    for (int w = 0; w < kMaxWarps; ++w)
      if (w < warps) m = fmaxf(m, ml[(w * S::kRows + row) * 2]);
#pragma unroll
    for (int w = 0; w < kMaxWarps; ++w)
      if (w < warps) {
        const float root = merge_root(ml[(w * S::kRows + row) * 2], m);
        f[w] = root * root;
        l = fmaf(root, root * ml[(w * S::kRows + row) * 2 + 1], l);
      }
    auto sum_at = [&](int d) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kMaxWarps; ++w)
        if (w < warps) add_scaled(o, f[w], *reinterpret_cast<const float4*>(sums + (w * S::kRows + row) * D + d));
      return o;
    };
    if (p.cluster == 1) {
      finish(row, m, l, sum_at);
    } else {
      for (int d = lane * 4; d < D; d += 128) *reinterpret_cast<float4*>(cta_sum + row * D + d) = sum_at(d);
      if (lane == 0) *reinterpret_cast<float2*>(cta_ml + 2 * row) = make_float2(m, l);
    }
  }
  if (p.cluster == 1) return;

  // ---- the cluster's sums meet: each warp of the cluster finishes a share of the rows. The tiles'
  // scales are done with: their place holds the factors of a row's pieces
  float* row_factor = reinterpret_cast<float*>(smem + region);
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int row = (split % p.cluster) * warps + warp; row < nrows; row += p.cluster * warps) {
    float2 part = make_float2(-INFINITY, 0.f);  // lane c: of CTA c
    if (lane < p.cluster) part = *reinterpret_cast<const float2*>(cluster.map_shared_rank(cta_ml, lane) + 2 * row);
    float m = part.x;
#pragma unroll
    for (int o = kMaxCluster / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    const float root = lane < p.cluster ? merge_root(part.x, m) : 0.f;
    float l = root * part.y * root;
#pragma unroll
    for (int o = kMaxCluster / 2; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    l = __shfl_sync(0xffffffffu, l, 0);
    if (lane < kMaxCluster) row_factor[warp * kMaxCluster + lane] = root * root;
    __syncwarp();
    finish(row, m, l, [&](int d) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int c = 0; c < p.cluster; ++c)
        add_scaled(o, row_factor[warp * kMaxCluster + c],
                   *reinterpret_cast<const float4*>(cluster.map_shared_rank(cta_sum, c) + row * D + d));
      return o;
    });
    __syncwarp();
  }
  cluster.sync();  // no CTA leaves while another still reads its sums
}

// Adds the clusters' pieces of the rows. grid: (requests, query tokens of the longest one, heads);
// one thread a dim.
template <typename T>
__global__ void combine_int8_kernel(const Int8AttnParams p, int D) {
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
      const float root = merge_root(ml.x, m);
      l = fmaf(root, root * ml.y, l);
      o = fmaf(root * root, p.ws_acc[(item + s) * D + d], o);
    }
    store_elem(static_cast<T*>(p.out) + row * p.out_stride + (int64_t)h * D + d, l == 0.f ? 0.f : o / l * kSumUnit);
  }
}

// Dynamic shared memory of a CTA, as the kernel lays it out.
int smem_bytes(int dtype, int D, int rows, int warps) {
  const int ring = warps * 32 * D * (D <= 128 ? 4 : 2), merge = (warps + 1) * rows * (D + 2) * 4;
  const int words = (dtype == VFL_DTYPE_F32 ? 4 : 3) * rows / 8 * (D / 16);
  return (ring > merge ? ring : merge) + warps * 64 * 16 + (words > 32 ? words * 128 : 0);
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

// About `splits` CTAs a context: a power of two up to a cluster's 8, multiples of 8 past it.
void set_splits(vfl_attention_int8_plan* plan, int64_t splits) {
  int cluster = 1;
  while (cluster < kMaxCluster && 2 * cluster <= splits) cluster *= 2;
  plan->cluster = cluster;
  plan->num_splits = static_cast<int32_t>(cluster < kMaxCluster ? cluster : splits / kMaxCluster * kMaxCluster);
}

// Warps and CTAs of an item. Measured on B200 (device time, bfloat16, head_dim 64; items = requests
// x K/V heads x row chunks):
//   * more items than slots: the CTA's start (about 5 us, five CTAs of four warps an SM) is spread
//     over fewer warps. 8192 items of 9 tiles: 1, 2, 4 warps take 36, 49, 69 us; 4096 items of 32
//     tiles: 54, 51, 60; 4096 of 1 to 256: 245, 198, 180. Hence one warp up to 16 tiles, two up to 64.
//   * items that four warps run in little more than one wave, and two warps in one, run two (768
//     items of 37 tiles: 17.4 against 20.8 us);
//   * fewer items: the context is cut until the slots are full, over a cluster at most (one of 8
//     takes 9.1 us for 16 items of 256 tiles, four clusters and the adding launch 9.9), past 512
//     tiles over more.
void choose_shape(vfl_attention_int8_plan* plan, int64_t items, int64_t tiles_sum) {
  const int64_t mean = items > 0 ? tiles_sum / items : 0;
  const int64_t longest = ceil_div((int64_t)plan->max_seq_len, (int64_t)16);
  const int by_smem = kSmemPerSM / (smem_bytes(plan->dtype, plan->head_dim, plan->rows_per_cta, 4) + 1024);
  const int lanes = plan->head_dim * plan->rows_per_cta;  // of a CTA's sums; see Shape::kMinCtas
  const int by_regs = lanes <= 512 ? 5 : (lanes <= 1024 ? (plan->dtype == VFL_DTYPE_F32 ? 3 : 4) : 2);
  const int per_sm = by_smem < 1 ? 1 : (by_smem < by_regs ? by_smem : by_regs);
  const int64_t slots = (int64_t)kNumSMs * per_sm;  // of CTAs of four warps
  plan->warps = 4;
  int64_t splits = 1;
  if (items > 2 * slots) {
    plan->warps = mean <= 16 ? 1 : (mean <= 64 ? 2 : 4);
  } else if (items > slots) {
    plan->warps = mean <= 64 ? 2 : 4;
  } else if (items > 0) {
    splits = slots / items;
    if (splits == 1 && 14 * items < 10 * slots && mean >= 64) splits = 2;
    const int64_t by_len = ceil_div(longest, (int64_t)2 * plan->warps);
    splits = splits < by_len ? splits : by_len;
    if (longest <= 512 && splits > kMaxCluster) splits = kMaxCluster;
    // clusters do not fill every GPC (with two CTAs an SM 71 of 4 and 33 of 8 were measured to fit):
    // one more is a second wave (72 float32 items of 16 rows: 20.4 us over clusters of 4, 17 of 2)
    if (splits >= 8 && splits < 16 && 100 * items > 89 * (slots / 8)) splits = 4;
    if (splits >= 4 && splits < 8 && 100 * items > 96 * (slots / 4)) splits = 2;
  }
  set_splits(plan, splits);
}

// Whether 16 query rows a CTA are built: past 128 dims their sums do not fit the registers.
bool rows16_built(int head_dim) { return head_dim <= 128; }

struct Launch {
  dim3 grid;
  int threads, smem;
  cudaStream_t stream;
};

template <typename T, int D, int NT>
int launch(const Int8AttnParams& p, const Launch& l) {
  static int smem_done[kMaxDevices] = {};
  auto kern = paged_attention_int8_kernel<T, D, NT>;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), l.smem, smem_done);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = l.grid;
  cfg.blockDim = dim3(l.threads, 1, 1);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = l.stream;
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
int launch_dim(const Int8AttnParams& p, int D, const Launch& l) {
  switch (D) {
    case 32: return launch<T, 32, NT>(p, l);
    case 48: return launch<T, 48, NT>(p, l);
    case 64: return launch<T, 64, NT>(p, l);
    case 80: return launch<T, 80, NT>(p, l);
    case 96: return launch<T, 96, NT>(p, l);
    case 112: return launch<T, 112, NT>(p, l);
    case 128: return launch<T, 128, NT>(p, l);
    default: break;
  }
  if constexpr (NT == 1) {
    switch (D) {
      case 160: return launch<T, 160, 1>(p, l);
      case 192: return launch<T, 192, 1>(p, l);
      case 224: return launch<T, 224, 1>(p, l);
      case 256: return launch<T, 256, 1>(p, l);
      default: return launch<T, 512, 1>(p, l);
    }
  }
  return fail(VFL_ERR_UNSUPPORTED, "attention_int8: 16 rows a CTA at head_dim %d", D);
}

template <typename T>
int launch_rows(const Int8AttnParams& p, int D, int rows, const Launch& l) {
  return rows == 16 ? launch_dim<T, 2>(p, D, l) : launch_dim<T, 1>(p, D, l);
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
  if (!(plan->warps == 1 || plan->warps == 2 || plan->warps == kMaxWarps) ||
      smem_bytes(plan->dtype, plan->head_dim, plan->rows_per_cta, plan->warps) > kSmemPerSM)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: plan warps %d", plan->warps);
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
  int64_t items = 0, tiles_sum = 0;
  for (int r = 0; r < num_reqs; ++r) {
    const int64_t ql = query_start_loc_host ? (int64_t)query_start_loc_host[r + 1] - query_start_loc_host[r] : 1;
    const int64_t n = ceil_div(ql * group, (int64_t)plan->rows_per_cta) * num_kv_heads;
    if (seq_lens_host[r] > 0) items += n;
    tiles_sum += n * ceil_div((int64_t)seq_lens_host[r], (int64_t)16);
  }

  choose_shape(plan, items, tiles_sum);
  plan->workspace_bytes = workspace_of(plan);
  plan->magic = VFL_INT8_PLAN_MAGIC;
  st = check_plan(plan);
  if (st) plan->magic = 0;
  return st;
}

int vfl_plan_attention_int8_shape(vfl_attention_int8_plan* plan, int warps, int num_splits) {
  int st = check_plan(plan);
  if (st) return st;
  vfl_attention_int8_plan next = *plan;
  if (warps != 0) next.warps = warps;
  if (num_splits < 0 || num_splits > 65535)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: num_splits %d", num_splits);
  if (num_splits > 0) set_splits(&next, num_splits);
  next.workspace_bytes = workspace_of(&next);
  st = check_plan(&next);
  if (st) return st;
  *plan = next;
  return VFL_OK;
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
  if (plan->num_reqs == 0 || plan->max_q_len == 0) return VFL_OK;  // rows before the first request's are nobody's
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
      (query_token_stride * es) % 16 != 0 || (output_token_stride * es) % 16 != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: tensors and token strides must be 16-byte aligned");
  if (!(scale == scale) || fabsf(scale) > FLT_MAX)
    return fail(VFL_ERR_INVALID_ARGUMENT, "attention_int8: scale is not finite");
  if (plan->workspace_bytes > 0 &&
      (workspace == nullptr || !aligned16(workspace) || workspace_bytes < (size_t)plan->workspace_bytes))
    return fail(VFL_ERR_WORKSPACE, "attention_int8: needs %lld workspace bytes (16-byte aligned), got %zu",
                (long long)plan->workspace_bytes, workspace_bytes);
  Int8AttnParams p = {};
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
  Launch l;
  l.grid = dim3(plan->num_reqs * plan->num_kv_heads, (unsigned)row_chunks(plan), plan->num_splits);
  l.threads = plan->warps * 32;
  l.smem = smem_bytes(plan->dtype, D, plan->rows_per_cta, plan->warps);
  l.stream = s;
  st = plan->dtype == VFL_DTYPE_F32 ? launch_rows<float>(p, D, plan->rows_per_cta, l)
                                    : launch_rows<__nv_bfloat16>(p, D, plan->rows_per_cta, l);
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
