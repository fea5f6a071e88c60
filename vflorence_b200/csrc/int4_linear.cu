// Linear layer with 4-bit weights and group scales for the few rows of a decode step:
//     y[m, n] = act(sum_g s[n, g] sum_{k in group g} x[m, k] (c[n, k] - 8) + b[n]).
// Codes c are packed two a byte along k, the lower nibble first, rows of a torch.nn.Linear weight;
// s has the type of x.
//
// Bound: HBM, half a byte a weight: every weight meets each of the few rows of x once. The
// products run on m16n8k16 bfloat16 tensor instructions with float32 sums: a nibble n becomes the
// bfloat16 0x4300 | n = 128 + n by one logic instruction a pair, and one subtraction of 136 leaves
// c - 8 exactly. bfloat16 x is used as it is; float32 x is the sum of three bfloat16 terms, which
// hold its 24 bits. Products are exact; a group's sum is taken in float32 before its scale.
//
// The 16 x k operand needs no re-packing: the order of k inside a product is free as long as both
// operands share it. Of each chunk of 128 k a lane takes 32 codes of a weight row, as many
// neighbouring ones as a scale group allows (16 bytes for groups of 128 and more). A word's nibbles
// i and i + 4 make a pair, and x is staged in shared memory in that order, so that a lane's
// operands for two steps are one 16-byte read, shared by two tiles of 16 weight rows.
//
// Work split: a CTA, or a cluster of 4 that shares out a long k so that a CTA stages its part of x
// only, takes a number of 32-row weight tiles. A CTA's (tile, chunk) units form one line that its 8
// warps cut evenly; each streams its stretch through its own ring of cp.async stages, from one tile
// into the next, and leaves a piece a tile. Pieces and CTAs are summed in a fixed order.
//
// Measured: 8 x 16384 x 8192 bfloat16 24 us, 69 MB at 2.9 TB/s. The same stream without its products
// takes 17.5 us; they are 340 instructions a unit, most of them shifts and logic at half rate, which 16
// warps an SM (121 registers) do not hide behind the stream: 0.47 of the issue slots are used. 1 x 1024 x
// 1024: 4.2 us, start and staging. Past 32 rows every 32 rows read and convert the weights anew: the
// bfloat16 GEMM of the library is as fast at 16 to 32 rows and faster past them (1024 x 1024: 8 rows 4.7
// against 4.5 us, 32 rows 9.9 against 4.1; 16384 x 8192: 8 rows 27 against 44, 32 rows 65 against 43).
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 128;      // k of a unit
constexpr int kTileRows = 32;    // weight rows of a unit
constexpr int kStageBytes = kTileRows * kChunk / 2;  // a unit's codes
constexpr int kStages = 3;
constexpr int kMaxRows = 32;     // rows of x a CTA takes; more rows are more CTAs
constexpr int kCluster = 4;      // CTAs that share out a long k
constexpr int kMaxClusters = 66; // that the GPU holds at once, two CTAs an SM (measured: they do not fill every GPC)
constexpr int kMaxTiles = 48;    // weight tiles of a CTA times n8 tiles of x rows: their sums fit the rings
constexpr int kHalfSmem = 112 * 1024;  // of a CTA that shares its SM with another
constexpr int kMaxSmem = 226 * 1024;

struct Int4LinearParams {
  const void* x;
  int64_t x_stride;
  const uint8_t* codes;
  const void* scales;
  const void* bias;
  void* y;
  int64_t y_stride;
  int rows, n, k, group, act;
  int cluster, clusters, chunks_per_cta, tiles_per_cluster;
  int segment;  // chunks whose x is staged at a time
};

__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Nibbles kShift / 4 and kShift / 4 + 4 of w, less 8, as two bfloat16.
template <int kShift>
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
  uint32_t biased;  // one instruction, which the compiler would split in two
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(biased) : "r"(w >> kShift), "r"(0x000f000f), "r"(0x43004300));
  const __nv_bfloat162 bias = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), bias);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_bf16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// kBytes (4, 8, 16) of neighbouring scales.
template <int kBytes, typename T, int kCount>
__device__ __forceinline__ void load_scales(const T* from, T (&to)[kCount]) {
  if constexpr (kBytes == 16) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(from));
    memcpy(to, &v, 16);
  } else if constexpr (kBytes == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(from));
    memcpy(to, &v, 8);
  } else {
    const uint32_t v = __ldg(reinterpret_cast<const unsigned int*>(from));
    memcpy(to, &v, sizeof(to) < 4 ? sizeof(to) : 4);
  }
}

// Where quarter q of the 64 bytes of row g (mod 8) lies: turned so that the lanes' reads of
// load_words, whose rows are 64 bytes apart, meet every bank once.
template <int kWords>
__device__ __forceinline__ int place(int g, int q) {
  return (q ^ (kWords == 1 ? g >> 1 : (kWords == 2 ? g & 2 : 0))) * 16;
}

// A lane's words of a row's 64 bytes: kWords neighbouring ones of each scale group.
template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t* row, int g, int tq, uint32_t (&w)[4]) {
  if (kWords == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + tq * 16);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if (kWords == 2) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + place<2>(g, j + (tq >> 1)) + (tq & 1) * 8);
      w[j] = v.x; w[j + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(row + place<1>(g, j) + tq * 4);
  }
}

// 8 neighbouring x of a row, as loaded; zeros where there is none.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, bool there) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) {
      a = __ldg(reinterpret_cast<const float4*>(p));
      b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool there) {
    a = there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack16(a, f, __nv_bfloat16()); }
};

// 8 x as 16 bytes in the order of a word's nibble pairs: (0, 4) (1, 5) (2, 6) (3, 7).
__device__ __forceinline__ uint4 pair_order(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[4]), pack_bf16x2(f[1], f[5]), pack_bf16x2(f[2], f[6]),
                    pack_bf16x2(f[3], f[7]));
}

// The shared memory of a CTA that stages `chunks` chunks of x at a time and has `tiles` weight tiles.
template <typename T, int NT>
struct Layout {
  static constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
  static constexpr int kChunkX = NT * kTerms * 2048;  // a chunk of x: [word][n8][term][lane] 16 bytes
  int x, pieces, total;
  __host__ __device__ Layout(int chunks, int tiles) {
    x = kWarps * kStages * kStageBytes;
    pieces = x + chunks * kChunkX;  // [tile + warp][8 * NT][32] float
    total = pieces + (tiles + kWarps) * kTileRows * 8 * NT * 4;
  }
};

// NT: n8 tiles of x rows (8 * NT rows). kWords: words of a lane inside one scale group of a chunk
// (4: groups of 128 and more, 2: of 64, 1: of 32).
template <typename T, int NT, int kWords>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) int4_linear_kernel(const Int4LinearParams p) {
  using L = Layout<T, NT>;
  constexpr int kTerms = L::kTerms, kBlocks = 4 / kWords;  // scale groups of a chunk
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int rank = blockIdx.x % p.cluster;
  const int tile0 = blockIdx.x / p.cluster * p.tiles_per_cluster;
  const int tiles = max(0, min(p.tiles_per_cluster, ceil_div(p.n, kTileRows) - tile0));
  const int m0 = blockIdx.y * (8 * NT);
  const int rows = min(8 * NT, p.rows - m0);
  const int k_begin = rank * p.chunks_per_cta * kChunk, k_end = min(k_begin + p.chunks_per_cta * kChunk, p.k);
  const int seg = p.segment;
  const L at(seg, p.tiles_per_cluster);
  const int64_t row_bytes = p.k / 2;
  const int groups = p.k / p.group;
  // a chunk's scales by one load where every row's are aligned for it (8 x 8192 x 8192 in groups of 32
  // bfloat16: 16.6 us, one by one 22.1)
  const bool wide_scales = groups % kBlocks == 0 && reinterpret_cast<uintptr_t>(p.scales) % (kBlocks * sizeof(T)) == 0;
  const int group_chunks = kWords == 4 ? p.group / kChunk : 1;

  // ---- this warp's stretch of the CTA's units, tile after tile; the same for every segment of k
  const int units = tiles * seg;
  const int first = units * warp / kWarps, last = units * (warp + 1) / kWarps;
  uint8_t* ring = smem + warp * (kStages * kStageBytes);
  const uint32_t ring_at = smem_u32(ring) + g * 64 + place<kWords>(g, tq);
  float* pieces = reinterpret_cast<float*>(smem + at.pieces);
  constexpr int kTile = kTileRows * 8 * NT;

  for (int s0 = k_begin; s0 == k_begin || s0 < k_end; s0 += seg * kChunk) {
    // the next fetch: its tile, place in k, this lane's codes and scales
    int f_tile = 0, f_k = 0, f_left = 0, f_group = 0, f_group_left = 0;
    const uint8_t* pc[4] = {};  // of rows g, g + 8, g + 16, g + 24
    const T* ps = nullptr;      // of row `lane`
    T scale[kStages][kBlocks];
    auto aim = [&](int tile, int chunk) {
      f_tile = tile;
      f_left = seg - chunk;
      f_k = s0 + chunk * kChunk;
      const int n0 = (tile0 + tile) * kTileRows;
      const uint8_t* base = p.codes + f_k / 2 + tq * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) pc[i] = base + min(n0 + g + 8 * i, p.n - 1) * row_bytes;  // rows past the end repeat the last
      ps = static_cast<const T*>(p.scales) + (int64_t)min(n0 + lane, p.n - 1) * groups;
      if (kWords == 4) {
        f_group = f_k / kChunk / group_chunks;
        f_group_left = (f_group + 1) * group_chunks - f_k / kChunk;
      } else {
        f_group = f_k / kChunk * kBlocks;
      }
    };
    if (first < last) aim(first / seg, first % seg);
    auto fetch = [&](int unit, int stage) {  // a group of its own, empty past the end
      if (unit < last) {
        // k is a multiple of 32: a piece is all there, or all past the end and zeros
        const int bytes = f_k + tq * 32 < k_end ? 16 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring_at + stage * kStageBytes + i * 512),
                       "l"(pc[i]), "r"(bytes)
                       : "memory");
          pc[i] += kChunk / 2;
        }
        if (kBlocks > 1 && wide_scales) {
          load_scales<kBlocks * sizeof(T)>(ps + min(f_group, groups - kBlocks), scale[stage]);  // past k: the last ones
        } else {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) scale[stage][b] = __ldg(ps + min(f_group + b, groups - 1));
        }
        f_k += kChunk;
        if (kWords < 4) {
          f_group += kBlocks;
        } else if (--f_group_left == 0) {
          ++f_group;
          f_group_left = group_chunks;
        }
        if (--f_left == 0 && unit + 1 < last) aim(f_tile + 1, 0);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(first + i, i);

    // ---- x in the order of the nibbles (columns without a row keep whatever is there: nothing
    // reads their sums)
    if (s0 > k_begin) __syncthreads();
    // a batch of loads is in flight before the first is used: one at a time, each turn of the CTA's
    // threads cost its latency (16 x 1024 x 4096 bfloat16: 9.4 us)
    constexpr int kBatch = sizeof(T) == 4 ? 4 : 8;
    const int items = rows * seg * 16;  // of 8 elements
    const uint32_t inverse = (1u << 20) / seg + 1;  // (i * inverse) >> 20 = i / seg while i * seg < 2^20
    for (int i0 = threadIdx.x; i0 < items; i0 += kBatch * kThreads) {
      Raw8<T> raw[kBatch];
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        const int i = i0 + r * kThreads, mc = i >> 4, m = mc * inverse >> 20, c = mc - m * seg;
        const int kb = s0 + c * kChunk + (i & 15) * 8;
        raw[r].load(static_cast<const T*>(p.x) + (m0 + m) * p.x_stride + kb, i < items && kb < k_end);
      }
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        const int i = i0 + r * kThreads, mc = i >> 4, m = mc * inverse >> 20, c = mc - m * seg, u = i & 15;
        if (i >= items) break;
        float f[8];
        raw[r].get(f);
        // unit u is word `word` of lane group `q`
        const int word = u / (4 * kWords) * kWords + (u & (kWords - 1)), q = (u / kWords) & 3;
        uint8_t* dst = smem + at.x + c * L::kChunkX + (word * NT + (m >> 3)) * (kTerms * 512) + ((m & 7) * 4 + q) * 16;
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
          if (term + 1 < kTerms) {  // the upper 8 bits, cut off: what is left is exact (an infinity leaves nothing)
            float top[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              top[e] = __uint_as_float(__float_as_uint(f[e]) & 0xffff0000u);
              f[e] = fabsf(f[e]) == INFINITY ? 0.f : f[e] - top[e];
            }
            *reinterpret_cast<uint4*>(dst + term * 512) = pair_order(top);
          } else {
            *reinterpret_cast<uint4*>(dst + term * 512) = pair_order(f);
          }
        }
      }
    }
    __syncthreads();

    // ---- the stretch
    float acc[NT][2][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][h][e] = 0.f;
    int tile = first < last ? first / seg : 0, chunk = first - tile * seg;
    const uint8_t* xd = smem + at.x + chunk * L::kChunkX + lane * 16;
    auto leave = [&]() {  // this tile's piece [x row][32]
      float* dst = pieces + (tile + warp) * kTile;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* at_e = dst + (t * 8 + 2 * tq + (e & 1)) * kTileRows + h * 16 + (e >> 1) * 8 + g;
            *at_e = s0 > k_begin ? *at_e + acc[t][h][e] : acc[t][h][e];
            acc[t][h][e] = 0.f;
          }
    };
#pragma unroll 1
    for (int u0 = first; u0 < last; u0 += kStages) {
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        if (u0 + st < last) {
          fetch(u0 + st + kStages - 1, (st + kStages - 1) % kStages);
          asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
          __syncwarp();
          const uint8_t* wr = ring + st * kStageBytes + g * 64;
          uint32_t w[4][4];  // rows g + 8 i: words in the order of the scale groups
#pragma unroll
          for (int i = 0; i < 4; ++i) load_words<kWords>(wr + i * 512, g, tq, w[i]);
#pragma unroll
          for (int j0 = 0; j0 < kBlocks; ++j0) {
            float part[NT][2][4];
#pragma unroll
            for (int j = j0 * kWords; j < (j0 + 1) * kWords; ++j) {
              uint32_t lo[2][4], hi[2][4];  // the word's pairs 0, 1 and 2, 3
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                lo[h][0] = nibbles<0>(w[2 * h][j]); lo[h][1] = nibbles<0>(w[2 * h + 1][j]);
                lo[h][2] = nibbles<4>(w[2 * h][j]); lo[h][3] = nibbles<4>(w[2 * h + 1][j]);
                hi[h][0] = nibbles<8>(w[2 * h][j]); hi[h][1] = nibbles<8>(w[2 * h + 1][j]);
                hi[h][2] = nibbles<12>(w[2 * h][j]); hi[h][3] = nibbles<12>(w[2 * h + 1][j]);
              }
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                  const uint4 x = *reinterpret_cast<const uint4*>(xd + ((j * NT + t) * kTerms + term) * 512);
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    if (j == j0 * kWords && term == 0)
                      mma_bf16_first(part[t][h], lo[h], x.x, x.y);
                    else
                      mma_bf16(part[t][h], lo[h], x.x, x.y);
                    mma_bf16(part[t][h], hi[h], x.z, x.w);
                  }
                }
            }
            const float s = as_float(scale[st][j0]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float fa = __shfl_sync(0xffffffffu, s, h * 16 + g), fb = __shfl_sync(0xffffffffu, s, h * 16 + 8 + g);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                acc[t][h][0] = fmaf(fa, part[t][h][0], acc[t][h][0]);
                acc[t][h][1] = fmaf(fa, part[t][h][1], acc[t][h][1]);
                acc[t][h][2] = fmaf(fb, part[t][h][2], acc[t][h][2]);
                acc[t][h][3] = fmaf(fb, part[t][h][3], acc[t][h][3]);
              }
            }
          }
          __syncwarp();  // every lane is done with the stage before it is filled again
          xd += L::kChunkX;
          if (++chunk == seg) {
            leave();
            xd -= seg * L::kChunkX;
            chunk = 0;
            ++tile;
          }
        }
      }
    }
    if (first < last && chunk > 0) leave();
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __syncthreads();

  // ---- a tile's pieces in the order of its warps, then the cluster's parts in the order of its
  // CTAs. The rings are free: the CTA's sums [tile][x row][32] take their place
  float* sums = reinterpret_cast<float*>(smem);
  constexpr int kPer = kTile / 32;  // elements of a tile a lane takes: its weight row, every x row
  auto store = [&](int t, const float (&v)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int m = j, n = (tile0 + t) * kTileRows + lane;
      if (m < rows && n < p.n) {
        float o = v[j];
        if (p.bias != nullptr) o += as_float(static_cast<const T*>(p.bias)[n]);
        if (p.act == VFL_ACT_GELU) o = gelu(o);
        put(static_cast<T*>(p.y) + (m0 + m) * p.y_stride + n, o);
      }
    }
  };
  for (int t = warp; t < tiles; t += kWarps) {
    float v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = 0.f;
    for (int w = 0; w < kWarps; ++w) {
      const int b = units * w / kWarps, e = units * (w + 1) / kWarps;
      if (b < e && b < (t + 1) * seg && e > t * seg) {
        const float* piece = pieces + (t + w) * kTile + lane;
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] += piece[j * 32];
      }
    }
    if (p.cluster == 1) {
      store(t, v);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) sums[t * kTile + j * 32 + lane] = v[j];
    }
  }
  if (p.cluster == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int t = rank * kWarps + warp; t < tiles; t += p.cluster * kWarps) {
    float v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = 0.f;
    for (int r = 0; r < p.cluster; ++r) {
      const float* part = cluster.map_shared_rank(sums, r) + t * kTile + lane;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] += part[j * 32];
    }
    store(t, v);
  }
  cluster.sync();  // no CTA leaves while another still reads its sums
}

// CTAs of a launch. Every CTA stages its part of x before its first product, in every launch anew,
// so a long k is cut over a cluster of 4 as soon as staging is what counts: from k = 4096, or 384
// rows' chunks and terms. Clusters of 1 / 2 / 4 / 8 measured, in us:
//     8 x 65536 x 2048 bfloat16    20.9 / 22.0 / 25.9 / 43.5
//     8 x 16384 x 8192 bfloat16    31.9 / 26.4 / 24.8 / 27.7
//     4 x 4096 x 16384 bfloat16    23.2 / 19.7 / 17.1 / 17.4
//     16 x 4096 x 1024 float32      9.2 /  8.7 /  8.3 / 12.6
//     16 x 51289 x 1024 float32    29.3 / 30.5 / 47.8 / 71.2  (more tiles than one wave of clusters holds)
template <typename T, int NT>
int choose(Int4LinearParams* p) {
  using L = Layout<T, NT>;
  const int tiles = ceil_div(p->n, kTileRows), chunks = ceil_div(p->k, kChunk);
  const int rows = p->rows < 8 * NT ? p->rows : 8 * NT;
  const bool cut = (chunks >= 32 || (chunks >= kCluster && chunks * rows * L::kTerms >= 384)) &&
                   tiles <= kMaxClusters * (kMaxTiles / NT);
  const int c = cut ? kCluster : 1;
  p->cluster = c;
  p->chunks_per_cta = ceil_div(chunks, c);
  const int64_t units = (int64_t)tiles * p->chunks_per_cta;
  int64_t clusters = ceil_div(units, (int64_t)kWarps);
  const int64_t most = cut ? kMaxClusters : 2 * kNumSMs;  // one more would be a second wave
  clusters = clusters < most ? clusters : most;
  clusters = clusters < tiles ? clusters : tiles;
  const int64_t least = ceil_div(tiles, kMaxTiles / NT);
  clusters = clusters < least ? least : clusters;
  p->tiles_per_cluster = static_cast<int>(ceil_div((int64_t)tiles, clusters));
  p->clusters = ceil_div(tiles, p->tiles_per_cluster);
  // segments of equal length whose x lets two CTAs share an SM, or one fit at all
  const int fixed = L(0, p->tiles_per_cluster).total;
  int room = (kHalfSmem - fixed) / L::kChunkX;
  if (room < 4) room = (kMaxSmem - fixed) / L::kChunkX;
  p->segment = ceil_div(p->chunks_per_cta, ceil_div(p->chunks_per_cta, room));
  return L(p->segment, p->tiles_per_cluster).total;
}

template <typename T, int NT, int kWords>
int launch(Int4LinearParams p, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  const int smem = choose<T, NT>(&p);
  auto kern = int4_linear_kernel<T, NT, kWords>;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), smem, smem_done);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.clusters * p.cluster, ceil_div(p.rows, 8 * NT), 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "linear_int4 launch");
}

template <typename T, int NT>
int launch_group(const Int4LinearParams& p, cudaStream_t s) {
  if (p.group == 32) return launch<T, NT, 1>(p, s);
  if (p.group == 64) return launch<T, NT, 2>(p, s);
  return launch<T, NT, 4>(p, s);
}

template <typename T>
int launch_rows(const Int4LinearParams& p, cudaStream_t s) {
  if (p.rows <= 8) return launch_group<T, 1>(p, s);
  if (p.rows <= 16) return launch_group<T, 2>(p, s);
  return launch_group<T, kMaxRows / 8>(p, s);
}

}  // namespace
}  // namespace vfl

using namespace vfl;

extern "C" int vfl_linear_int4(const void* x, int64_t x_stride, const void* codes, const void* scales, const void* bias,
                               void* y, int64_t y_stride, int32_t rows, int32_t n, int32_t k, int32_t group_size,
                               int32_t dtype, int32_t activation, void* stream) {
  if (!dtype_ok(dtype)) return fail(VFL_ERR_UNSUPPORTED, "linear_int4: dtype %d", dtype);
  if (activation != VFL_ACT_NONE && activation != VFL_ACT_GELU)
    return fail(VFL_ERR_INVALID_ARGUMENT, "linear_int4: activation %d", activation);
  if (rows < 0 || n <= 0 || k <= 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "linear_int4: rows %d, n %d, k %d", rows, n, k);
  if (group_size != 32 && group_size != 64 && (group_size <= 0 || group_size % kChunk != 0))
    return fail(VFL_ERR_UNSUPPORTED, "linear_int4: group_size %d (32, 64 or a multiple of 128)", group_size);
  if (k % group_size != 0)
    return fail(VFL_ERR_UNSUPPORTED, "linear_int4: k %d is not a multiple of the group size %d", k, group_size);
  if (rows == 0) return VFL_OK;
  if (ceil_div(rows, kMaxRows) > 65535) return fail(VFL_ERR_UNSUPPORTED, "linear_int4: too many rows (%d)", rows);
  if (!x || !codes || !scales || !y) return fail(VFL_ERR_INVALID_ARGUMENT, "linear_int4: NULL pointer");
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  if (!aligned16(x) || (x_stride * es) % 16 != 0 || !aligned16(codes) || x_stride < k || y_stride < n)
    return fail(VFL_ERR_INVALID_ARGUMENT,
                "linear_int4: x, its rows and the codes must be 16-byte aligned, x_stride >= k, y_stride >= n");
  if (reinterpret_cast<uintptr_t>(scales) % es || reinterpret_cast<uintptr_t>(y) % es ||
      reinterpret_cast<uintptr_t>(bias) % es)
    return fail(VFL_ERR_INVALID_ARGUMENT, "linear_int4: scales, bias or y not aligned to their elements");
  Int4LinearParams p{x, x_stride, static_cast<const uint8_t*>(codes), scales, bias, y, y_stride, rows, n, k,
                     group_size, activation, 1, 1, 1, 1, 1};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == VFL_DTYPE_F32 ? launch_rows<float>(p, s) : launch_rows<__nv_bfloat16>(p, s);
}
