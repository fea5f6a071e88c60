// The paged K/V cache held in 8 bits: append and read-back.
//
// A block's tokens of one head share a float32 scale: codes int8 [num_blocks, H, block_size, D],
// scales [num_blocks, H], value = code * scale. The append keeps a block consistent while it
// fills: with a = the largest finite magnitude of the new tokens, s' = max(s, a * (1/127)); when
// s' > s the codes the block holds are brought to the new step, rint(code * (s * (1/s'))), and
// the new ones are rint(x * (1/s')) held to [-127, 127]. Writing offset 0 starts a block anew
// (s = 0). Products in float32 with one rounding each, so that a plain restatement gives the
// same codes bit for bit. A growth rounds the older codes once more (at most half a step).
//
// Both kernels move bytes: the bound is HBM for many tokens and one dependent round trip (slot,
// then the block's scale and the token) for a few.
#include "common.cuh"

namespace vfl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Smallest scale kept: the attention divides by V scales, and 2^100 times a context's token
// count stays inside float32. Blocks whose largest magnitude is below 127 * 2^-100 hold zeros.
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100

// The value a scale has while a run of tokens of its block is being stored: a NaN payload that
// no arithmetic makes. It doubles as the block's lock, see append_int8_kernel.
constexpr uint32_t kScaleLocked = 0xffe5a5a5u;
constexpr uint64_t kLockLimitNs = 500000000ull;

struct AppendParams {
  const uint8_t* x[2];       // key, value rows
  int64_t x_stride_bytes[2];
  int8_t* cache[2];
  float* scale[2];
  const int64_t* slots;
  int64_t num_tokens, capacity;
  int num_heads, head_dim, block_size;
  int window;                // consecutive rows whose runs one warp takes
  unsigned int* err;
};

__device__ __forceinline__ int64_t block_of(int64_t slot, int block_size) {
  // slots of real pools fit 32 bits; the 64-bit division is several times longer
  return slot <= 0xffffffffll ? (int64_t)((uint32_t)slot / (uint32_t)block_size) : slot / block_size;
}

// One code: rint(x * inv) held to [-127, 127]; 0 where the product is a NaN (x a NaN, or an
// infinity in a block whose scale is zero).
__device__ __forceinline__ int quantize(float x, float inv) {
  const float y = __fmul_rn(x, inv);
  return y != y ? 0 : __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

// code * ratio, rounded, for the four codes of a word.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  int c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int code = (int)(int8_t)(w >> (8 * i));
    c[i] = __float2int_rn(__fmul_rn((float)code, ratio));
  }
  return pack4(c[0], c[1], c[2], c[3]);
}

// One warp stores the runs that begin in its window of rows, for one head of K or of V. A run is
// a stretch of consecutive rows whose slots lie in one block: all of an encoder block's tokens,
// or the one token of a decode step. Its largest magnitude is known before its first code is
// written, so a block filled by one call is rounded once.
//
// Two runs of one block in a call (rows of a block that are not neighbours) are taken one after
// the other: the warp swaps kScaleLocked into the scale before it reads the block and puts the
// new scale back after its stores. The holder never waits, so the wait ends; it is bounded all
// the same. The swap is the read of the old scale, so the usual call pays nothing for it.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_int8_kernel(const AppendParams p) {
  constexpr int kVec = Elem<T>::kVec;
  const int lane = threadIdx.x & 31;
  const int64_t unit = blockIdx.x * (int64_t)kWarps + (threadIdx.x >> 5);
  // units: (window, K or V, head), heads fastest so that neighbours read neighbouring rows
  const int per_window = 2 * p.num_heads;
  const int64_t win = unit / per_window;
  const int64_t t_begin = win * p.window;
  if (t_begin >= p.num_tokens) return;
  const int rest = static_cast<int>(unit - win * per_window);
  const int kv = rest / p.num_heads, h = rest - kv * p.num_heads;
  const int64_t t_end = min(t_begin + p.window, p.num_tokens);
  const int D = p.head_dim, bs = p.block_size;
  const int vecs = D / kVec;                       // 16-byte pieces of a row
  const int group = vecs >= 32 ? 32 : next_pow2(vecs);  // lanes on a row
  const int sub = lane / group, col = lane - sub * group, rows_par = 32 / group;

  for (int64_t t = t_begin; t < t_end;) {
    // the row before t decides whether a run begins here
    const int64_t slot = __ldg(p.slots + t);
    if (slot < 0 || slot >= p.capacity) {
      if (slot >= 0 && rest == 0 && lane == 0) report(p.err, VFL_DEVERR_SLOT);
      ++t;
      continue;
    }
    const int64_t blk = block_of(slot, bs);
    if (t == t_begin && t > 0) {
      const int64_t before = __ldg(p.slots + t - 1);
      if (before >= 0 && before < p.capacity && block_of(before, bs) == blk) {
        ++t;  // an earlier warp's run
        while (t < t_end) {
          const int64_t s = __ldg(p.slots + t);
          if (s < 0 || s >= p.capacity || block_of(s, bs) != blk) break;
          ++t;
        }
        continue;
      }
    }
    int64_t run_end = t + 1;
    bool fresh = slot == blk * bs;
    while (run_end < p.num_tokens) {
      const int64_t s = __ldg(p.slots + run_end);
      if (s < 0 || s >= p.capacity || block_of(s, bs) != blk) break;
      fresh |= s == blk * bs;
      ++run_end;
    }
    const int n = static_cast<int>(run_end - t);

    // take the block's scale
    uint32_t* word = reinterpret_cast<uint32_t*>(p.scale[kv] + blk * p.num_heads + h);
    uint32_t old_bits = 0;
    if (lane == 0) {
      old_bits = atomicExch(word, kScaleLocked);
      if (old_bits == kScaleLocked) {
        const uint64_t t0 = globaltimer_ns();
        do {
          __nanosleep(100);
          old_bits = atomicExch(word, kScaleLocked);
        } while (old_bits == kScaleLocked && globaltimer_ns() - t0 < kLockLimitNs);
      }
      __threadfence();
    }

    // largest finite magnitude of the run
    float largest = 0.f;
    bool odd = false;  // an infinity or a NaN
    const uint8_t* base = p.x[kv] + (int64_t)h * D * sizeof(T);
    for (int j = sub; j < n; j += rows_par) {
      const uint4* row = reinterpret_cast<const uint4*>(base + (t + j) * p.x_stride_bytes[kv]);
      for (int c = col; c < vecs; c += group) {
        float f[kVec];
        unpack16(__ldg(row + c), f, T());
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float a = fabsf(f[i]);
          const bool finite = a <= 3.402823466e38f;
          largest = fmaxf(largest, finite ? a : 0.f);
          odd |= !finite;
        }
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    odd = __any_sync(0xffffffffu, odd);
    old_bits = __shfl_sync(0xffffffffu, old_bits, 0);
    if (old_bits == kScaleLocked) {  // another run never let go: nothing is stored
      if (lane == 0) report(p.err, VFL_DEVERR_SLOT);
      t = run_end;
      continue;
    }
    if (odd && lane == 0) report(p.err, VFL_DEVERR_NONFINITE);
    const float stored = __uint_as_float(old_bits);
    const float old = fresh || !(stored > 0.f) ? 0.f : stored;
    float want = __fmul_rn(largest, 1.f / 127.f);
    want = want < kMinScale ? 0.f : want;
    const float now = fmaxf(old, want);
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;

    int8_t* block = p.cache[kv] + (blk * p.num_heads + h) * (int64_t)bs * D;
    if (now > old && !fresh) {  // the step grew: the codes the block holds follow
      const float ratio = __fmul_rn(old, inv);
      uint4* b16 = reinterpret_cast<uint4*>(block);
      for (int i = lane; i < bs * D / 16; i += 32) {
        uint4 w = __ldcg(b16 + i);
        w = make_uint4(rescale4(w.x, ratio), rescale4(w.y, ratio), rescale4(w.z, ratio), rescale4(w.w, ratio));
        __stcg(b16 + i, w);
      }
      __syncwarp();  // the new codes overwrite theirs after it
    }
    for (int j = sub; j < n; j += rows_par) {
      const int64_t off = __ldg(p.slots + t + j) - blk * bs;
      const uint4* row = reinterpret_cast<const uint4*>(base + (t + j) * p.x_stride_bytes[kv]);
      for (int c = col; c < vecs; c += group) {
        float f[kVec];
        unpack16(__ldg(row + c), f, T());
        uint32_t* dst = reinterpret_cast<uint32_t*>(block + off * D + c * kVec);
#pragma unroll
        for (int i = 0; i < kVec / 4; ++i)
          __stcg(dst + i, pack4(quantize(f[4 * i], inv), quantize(f[4 * i + 1], inv), quantize(f[4 * i + 2], inv),
                                quantize(f[4 * i + 3], inv)));
      }
    }
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      atomicExch(word, __float_as_uint(now));
    }
    t = run_end;
  }
}

struct GatherParams {
  const int8_t* cache[2];
  const float* scale[2];
  uint4* out[2];
  const int64_t* slots;
  int64_t num_tokens, capacity;
  int num_heads, head_dim, block_size;
  unsigned int* err;
};

// One thread per 8 codes of K and of V; rows without a slot read as zeros.
template <typename T>
__global__ void __launch_bounds__(kThreads) gather_int8_kernel(const GatherParams p) {
  constexpr int kPieces = 8 / Elem<T>::kVec;  // 16-byte stores per 8 codes
  const int row_words = p.head_dim / 8;
  const int64_t total = p.num_tokens * p.num_heads * row_words;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t th = i / row_words;
    const int c = static_cast<int>(i - th * row_words);
    const int64_t t = th / p.num_heads;
    const int h = static_cast<int>(th - t * p.num_heads);
    const int64_t slot = __ldg(p.slots + t);
    const bool ok = slot >= 0 && slot < p.capacity;
    if (slot >= p.capacity && h == 0 && c == 0) report(p.err, VFL_DEVERR_SLOT);
    int64_t src = 0, sc = 0;
    if (ok) {
      const int64_t blk = block_of(slot, p.block_size);
      sc = blk * p.num_heads + h;
      src = (sc * p.block_size + (slot - blk * p.block_size)) * p.head_dim + c * 8;
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float f[8];
      uint2 w = make_uint2(0u, 0u);
      float s = 0.f;
      if (ok) {
        w = __ldg(reinterpret_cast<const uint2*>(p.cache[kv] + src));
        s = __ldg(p.scale[kv] + sc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = (float)(int)(int8_t)(w.x >> (8 * e)) * s;
        f[4 + e] = (float)(int)(int8_t)(w.y >> (8 * e)) * s;
      }
#pragma unroll
      for (int q = 0; q < kPieces; ++q) p.out[kv][i * kPieces + q] = pack16(f + q * Elem<T>::kVec, T());
    }
  }
}

int check_cache(const char* what, int dtype, int64_t num_tokens, int num_heads, int head_dim, int block_size,
                int64_t num_blocks) {
  if (!dtype_ok(dtype)) return fail(VFL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (num_tokens < 0 || num_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "%s: bad sizes (tokens %lld, heads %d, head_dim %d, block_size %d, blocks %lld)",
                what, (long long)num_tokens, num_heads, head_dim, block_size, (long long)num_blocks);
  if (head_dim % 16 != 0)
    return fail(VFL_ERR_UNSUPPORTED, "%s: head_dim %d must be a multiple of 16", what, head_dim);
  return VFL_OK;
}

}  // namespace
}  // namespace vfl

using namespace vfl;

extern "C" {

int vfl_reshape_and_cache_int8(const void* key, const void* value, void* k_cache, void* v_cache, float* k_scale,
                               float* v_scale, const int64_t* slot_mapping, int64_t num_tokens, int num_heads,
                               int head_dim, int block_size, int64_t num_blocks, int64_t key_token_stride,
                               int64_t value_token_stride, int dtype, void* stream) {
  int st = check_cache("reshape_and_cache_int8", dtype, num_tokens, num_heads, head_dim, block_size, num_blocks);
  if (st) return st;
  if (num_tokens == 0) return VFL_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
    return fail(VFL_ERR_INVALID_ARGUMENT, "reshape_and_cache_int8: NULL pointer");
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  if (!aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (key_token_stride * es) % 16 != 0 || (value_token_stride * es) % 16 != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "reshape_and_cache_int8: tensors and token strides must be 16-byte aligned");
  if (key_token_stride < (int64_t)num_heads * head_dim || value_token_stride < (int64_t)num_heads * head_dim)
    return fail(VFL_ERR_INVALID_ARGUMENT, "reshape_and_cache_int8: token stride smaller than a token");
  AppendParams p;
  st = device_error_word(&p.err);
  if (st) return st;
  p.x[0] = static_cast<const uint8_t*>(key);
  p.x[1] = static_cast<const uint8_t*>(value);
  p.x_stride_bytes[0] = key_token_stride * es;
  p.x_stride_bytes[1] = value_token_stride * es;
  p.cache[0] = static_cast<int8_t*>(k_cache);
  p.cache[1] = static_cast<int8_t*>(v_cache);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.slots = slot_mapping;
  p.num_tokens = num_tokens;
  p.capacity = num_blocks * block_size;
  p.num_heads = num_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  // A decode step's rows are runs of one: a window of one row keeps them all in flight. Many
  // rows are blocks' worth of neighbours: windows of a block leave few warps without a run.
  p.window = num_tokens * 2 * num_heads <= (int64_t)kNumSMs * 256 ? 1 : (block_size < 64 ? block_size : 64);
  const int64_t warps = ceil_div(num_tokens, (int64_t)p.window) * 2 * num_heads;
  const int64_t ctas = ceil_div(warps, (int64_t)kWarps);
  if (ctas > INT32_MAX) return fail(VFL_ERR_UNSUPPORTED, "reshape_and_cache_int8: too many tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VFL_DTYPE_F32)
    append_int8_kernel<float><<<(unsigned)ctas, kThreads, 0, s>>>(p);
  else
    append_int8_kernel<__nv_bfloat16><<<(unsigned)ctas, kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "reshape_and_cache_int8 launch");
}

int vfl_gather_kv_int8(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                       const int64_t* slot_mapping, void* key, void* value, int64_t num_tokens, int num_heads,
                       int head_dim, int block_size, int64_t num_blocks, int dtype, void* stream) {
  int st = check_cache("gather_kv_int8", dtype, num_tokens, num_heads, head_dim, block_size, num_blocks);
  if (st) return st;
  if (num_tokens == 0) return VFL_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
    return fail(VFL_ERR_INVALID_ARGUMENT, "gather_kv_int8: NULL pointer");
  if (!aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(VFL_ERR_INVALID_ARGUMENT, "gather_kv_int8: tensors must be 16-byte aligned");
  GatherParams p;
  st = device_error_word(&p.err);
  if (st) return st;
  p.cache[0] = static_cast<const int8_t*>(k_cache);
  p.cache[1] = static_cast<const int8_t*>(v_cache);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.out[0] = static_cast<uint4*>(key);
  p.out[1] = static_cast<uint4*>(value);
  p.slots = slot_mapping;
  p.num_tokens = num_tokens;
  p.capacity = num_blocks * block_size;
  p.num_heads = num_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  const int64_t work = num_tokens * num_heads * (head_dim / 8);
  const int64_t want = ceil_div(work, (int64_t)kThreads), cap = (int64_t)kNumSMs * 32;
  const unsigned ctas = static_cast<unsigned>(want < cap ? want : cap);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VFL_DTYPE_F32)
    gather_int8_kernel<float><<<ctas, kThreads, 0, s>>>(p);
  else
    gather_int8_kernel<__nv_bfloat16><<<ctas, kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "gather_kv_int8 launch");
}

}  // extern "C"
