// Linear layer with 4-bit weights and group scales for the few rows of a decode step:
//     y[m, n] = act(sum_g s[n, g] sum_{k in group g} x[m, k] (c[n, k] - 8) + b[n]).
// Codes c are packed two a byte along k, the lower nibble first, rows of a torch.nn.Linear weight;
// s has the type of x.
//
// Bound: HBM, half a byte a weight; every weight meets each of the few rows of x once. The
// products run on m16n8k16 bfloat16 tensor instructions with float32 sums: a nibble n becomes
// the bfloat16 0x4300 | n = 128 + n by one logic instruction a pair, and one subtraction of 136
// leaves c - 8 exactly. bfloat16 x is used as it is; float32 x is the sum of three bfloat16
// terms, which hold its 24 bits. A group's sum is taken in float32 before its scale is applied.
//
// The 16 x k operand tile needs no re-packing: the order of k inside a product is free as long as
// both operands share it. Of each chunk of 128 k a lane holds 32 codes of two weight rows, as
// many neighbouring ones as a scale group allows (16 bytes for groups of 128 and more). A word's
// nibbles i and i + 4 make a pair, and x is staged in shared memory in that order, so that a
// lane's operands for two steps are one 16-byte read.
//
// Work split: a CTA of 8 warps takes 16 rows of the weight; the warps share out k in chunks of
// 128, and their sums meet in shared memory in a fixed order.
#include "common.cuh"

namespace vfl {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 128;    // k of a warp-wide load: 16 bytes a lane
constexpr int kMaxRows = 32;   // rows of x a launch's CTA takes; more rows are more CTAs
constexpr int kStageBytes = 96 * 1024;

struct Int4LinearParams {
  const void* x;
  int64_t x_stride;
  const uint8_t* codes;
  const void* scales;
  const void* bias;
  void* y;
  int64_t y_stride;
  int rows, n, k, group, act;
  int seg;  // k staged at a time, a multiple of kChunk
};

__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Nibbles `shift` / 4 and `shift` / 4 + 4 of w, less 8, as two bfloat16.
template <int kShift>
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
  const uint32_t biased = ((w >> kShift) & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 bias = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), bias);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 neighbouring x of a row.
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  unpack16(__ldg(reinterpret_cast<const uint4*>(p)), f, __nv_bfloat16());
}

// A lane's codes of a chunk in memory order: kWords neighbouring words at a time.
template <int kWords>
__device__ __forceinline__ void load_codes(const uint8_t* row, int k0, int tq, int k, uint32_t (&w)[4]) {
#pragma unroll
  for (int j = 0; j < 4; j += kWords) {
    const int kb = k0 + (j * 4 + tq * kWords) * 8;
    const bool in = k0 + j * 32 < k;  // k ends with a scale group
    if (kWords == 4) {
      const uint4 v = in ? ldg_nc_v4(row + kb / 2) : make_uint4(0u, 0u, 0u, 0u);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if (kWords == 2) {
      const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(row + kb / 2)) : make_uint2(0u, 0u);
      w[j] = v.x; w[j + 1] = v.y;
    } else {
      w[j] = in ? __ldg(reinterpret_cast<const unsigned int*>(row + kb / 2)) : 0u;
    }
  }
}

// 8 x as 16 bytes in the order of a word's nibble pairs: (0, 4) (1, 5) (2, 6) (3, 7).
__device__ __forceinline__ uint4 pair_order(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[4]), pack_bf16x2(f[1], f[5]), pack_bf16x2(f[2], f[6]),
                    pack_bf16x2(f[3], f[7]));
}

// NT: n8 tiles of x rows (8 * NT rows). kWords: words of a lane inside one scale group of a chunk
// (4: groups of 128 and more, 2: of 64, 1: of 32).
template <typename T, int NT, int kWords>
__global__ void __launch_bounds__(kThreads) int4_linear_kernel(const Int4LinearParams p) {
  constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
  extern __shared__ uint4 xs[];  // [term][n8 tile][unit][lane]: unit = 4 * chunk + word
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int n0 = blockIdx.x * 16;
  const int m0 = blockIdx.y * (8 * NT);
  const int rows = min(8 * NT, p.rows - m0);
  const int64_t row_bytes = p.k / 2;
  const int na = min(n0 + g, p.n - 1), nb = min(n0 + g + 8, p.n - 1);  // rows past the end repeat the last
  const uint8_t* wa = p.codes + na * row_bytes;
  const uint8_t* wb = p.codes + nb * row_bytes;
  const int groups = p.k / p.group;
  const T* sa = static_cast<const T*>(p.scales) + (int64_t)na * groups;
  const T* sb = static_cast<const T*>(p.scales) + (int64_t)nb * groups;

  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

  for (int k0 = 0; k0 < p.k; k0 += p.seg) {
    const int seg = min(p.seg, p.k - k0);
    const int units = seg / 8;                          // of 8 neighbouring k
    const int chunks = ceil_div(seg, kChunk);
    const int plane = chunks * 4 * 32;                  // 16-byte pieces of one n8 tile of one term
    if (k0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * chunks * 16; i += kThreads) {
      const int m = i / (chunks * 16), u = i - m * (chunks * 16);
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
      if (m < rows && u < units) {
        load8(static_cast<const T*>(p.x) + (m0 + m) * p.x_stride + k0 + u * 8, f);
      }
      // unit u of its chunk is word `word` of lane group `q`
      const int word = (u & 15) / (4 * kWords) * kWords + (u & (kWords - 1)), q = (u & 15) / kWords & 3;
      const int at = (m / 8) * plane + ((u / 16) * 4 + word) * 32 + (m & 7) * 4 + q;
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        if (term + 1 < kTerms) {  // the upper 8 bits, cut off: what is left is exact (an infinity leaves nothing)
          float top[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            top[e] = __uint_as_float(__float_as_uint(f[e]) & 0xffff0000u);
            f[e] = fabsf(f[e]) == INFINITY ? 0.f : f[e] - top[e];
          }
          xs[term * NT * plane + at] = pair_order(top);
        } else {
          xs[term * NT * plane + at] = pair_order(f);
        }
      }
    }
    __syncthreads();

    for (int c = warp; c < chunks; c += kWarps) {
      uint32_t a[4], b[4];
      load_codes<kWords>(wa, k0 + c * kChunk, tq, p.k, a);
      load_codes<kWords>(wb, k0 + c * kChunk, tq, p.k, b);
#pragma unroll
      for (int j0 = 0; j0 < 4; j0 += kWords) {  // the chunk's scale groups
        float part[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[t][e] = 0.f;
#pragma unroll
        for (int j = j0; j < j0 + kWords; ++j) {
          const uint32_t a0 = nibbles<0>(a[j]), a1 = nibbles<4>(a[j]), a2 = nibbles<8>(a[j]), a3 = nibbles<12>(a[j]);
          const uint32_t b0 = nibbles<0>(b[j]), b1 = nibbles<4>(b[j]), b2 = nibbles<8>(b[j]), b3 = nibbles<12>(b[j]);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
              const uint4 x = xs[(term * NT + t) * plane + (c * 4 + j) * 32 + lane];
              mma_bf16(part[t], a0, b0, a1, b1, x.x, x.y);
              mma_bf16(part[t], a2, b2, a3, b3, x.z, x.w);
            }
        }
        const int gi = min((k0 + c * kChunk + j0 * 32) / p.group, groups - 1);
        const float fa = as_float(sa[gi]), fb = as_float(sb[gi]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[t][0] = fmaf(fa, part[t][0], acc[t][0]);
          acc[t][1] = fmaf(fa, part[t][1], acc[t][1]);
          acc[t][2] = fmaf(fb, part[t][2], acc[t][2]);
          acc[t][3] = fmaf(fb, part[t][3], acc[t][3]);
        }
      }
    }
  }

  // the warps' sums, added in warp order
  __syncthreads();
  float* sums = reinterpret_cast<float*>(xs);  // [warp][x row][16]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sums[(warp * 8 * NT + t * 8 + 2 * tq + (e & 1)) * 16 + g + (e >> 1) * 8] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < rows * 16; i += kThreads) {
    const int m = i / 16, j = i & 15, n = n0 + j;
    if (n >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[(w * 8 * NT + m) * 16 + j];
    if (p.bias != nullptr) v += as_float(static_cast<const T*>(p.bias)[n]);
    if (p.act == VFL_ACT_GELU) v = gelu(v);
    put(static_cast<T*>(p.y) + (m0 + m) * p.y_stride + n, v);
  }
}

template <typename T, int NT, int kWords>
int launch(Int4LinearParams p, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
  auto kern = int4_linear_kernel<T, NT, kWords>;
  // x is staged in segments of k that fit
  const int per_chunk = kTerms * NT * 4 * 32 * 16;
  const int fit = kStageBytes / per_chunk;
  const int chunks = ceil_div(p.k, kChunk) < fit ? ceil_div(p.k, kChunk) : fit;
  p.seg = chunks * kChunk;
  const int merge = kWarps * 8 * NT * 16 * 4;
  const int smem = chunks * per_chunk > merge ? chunks * per_chunk : merge;
  int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), kStageBytes, smem_done);
  if (st) return st;
  const dim3 grid(ceil_div(p.n, 16), ceil_div(p.rows, 8 * NT));
  kern<<<grid, kThreads, smem, stream>>>(p);
  return cuda_status(cudaGetLastError(), "linear_int4 launch");
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
                     group_size, activation, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == VFL_DTYPE_F32 ? launch_rows<float>(p, s) : launch_rows<__nv_bfloat16>(p, s);
}
