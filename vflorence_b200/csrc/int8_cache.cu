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
constexpr int kMaxWindow = 16;  // rows whose runs one warp stores, at most 31

// Smallest scale kept: the attention divides by V scales, and 2^100 times a context's token
// count stays inside float32. Blocks whose largest magnitude is below 127 * 2^-100 hold zeros.
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100

// The value a scale has while a run of tokens of its block is being stored: a NaN payload that
// no arithmetic makes. It doubles as the block's lock, see append_int8_kernel.
constexpr uint32_t kScaleLocked = 0xffe5a5a5u;
constexpr uint64_t kLockLimitNs = 500000000ull;

struct AppendParams {
  const uint8_t *key, *value;  // rows
  int key_stride_bytes, value_stride_bytes;
  int8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int64_t* slots;
  int64_t capacity;
  int num_tokens, num_heads, head_dim, block_size;
  int window;                // consecutive rows whose runs one warp takes
  uint32_t inverse;          // 2^32 / 16-byte pieces of a row, rounded up
  int rows_per_warp;         // 32 / pieces of a row
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

__device__ __forceinline__ void store_codes(int8_t* dst, const uint32_t (&c)[1]) {
  __stcg(reinterpret_cast<uint32_t*>(dst), c[0]);
}
__device__ __forceinline__ void store_codes(int8_t* dst, const uint32_t (&c)[2]) {
  __stcg(reinterpret_cast<uint2*>(dst), make_uint2(c[0], c[1]));
}

// The lock's two sides: what the holder before stored is seen after the first, what this warp
// stored is seen before the second.
__device__ __forceinline__ uint32_t exchange_acquire(uint32_t* at, uint32_t v) {
  uint32_t old;
  asm volatile("atom.acquire.gpu.global.exch.b32 %0, [%1], %2;" : "=r"(old) : "l"(at), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ void store_release(uint32_t* at, uint32_t v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(at), "r"(v) : "memory");
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

// Four codes where every product is within 127 and a rounding error: adding 1.5 * 2^23 rounds it
// to the whole number in the sum's low bits (to even, as rint does).
__device__ __forceinline__ uint32_t quantize4(const float* x, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.f));
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// One warp stores the runs that begin in its window of rows, for one head of K or of V. A run is
// a stretch of consecutive rows whose slots lie in one block: all of an encoder block's tokens,
// or the one token of a decode step. Its largest magnitude is known before its first code is
// written, so a block filled by one call is rounded once. A run of up to kHeld pieces a lane stays
// in registers from its maximum to its codes; a longer one is read a second time.
//
// Two runs of one block in a call (rows of a block that are not neighbours) are taken one after
// the other: the warp swaps kScaleLocked into the scale before it reads the block and puts the
// new scale back after its stores. The holder never waits, so the wait ends; it is bounded all
// the same. The swap is the read of the old scale, in flight together with the run's own loads.
//
// kEven: a row's pieces divide the warp, so a lane's pieces are a fixed step of rows apart (32 x 572
// tokens of 12 x 128 bfloat16: 49 us, by a multiplication a piece 61).
//
// kOneRow (windows of one row, as in a decode step): a lane holds one piece and eight CTAs share an
// SM, spills and all, since the chain of slot, scale and block is the time: 256 single tokens of
// 16 x 64 6.4 us, 512 of 16 x 128 10.8 us; by the other variant 8.7 and 15.1, by six CTAs 7.7 and 11.8.
//
// Measured: 64 x 585 tokens of 12 x 64 bfloat16 62 us, 172 MB at 2.8 TB/s: about 630 instructions a
// run of 16 rows at 0.54 a clock and scheduler are the bound, and the registers (64, for four CTAs an
// SM) what keeps them from more. A few tokens take 3.4 us.
template <typename T, bool kEven, bool kOneRow>
__global__ void __launch_bounds__(kThreads, kOneRow ? 8 : 4) append_int8_kernel(const AppendParams p) {
  constexpr int kVec = Elem<T>::kVec;
  constexpr int kHeld = kOneRow ? 1 : (sizeof(T) == 4 ? 8 : 4);
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x * (uint32_t)kWarps + (threadIdx.x >> 5);
  // units: (window, K or V, head), heads fastest so that neighbours read neighbouring rows
  const uint32_t win = unit / (2 * p.num_heads);
  const int t_begin = win * p.window;
  if (t_begin >= p.num_tokens) return;
  const int rest = static_cast<int>(unit - win * (2 * p.num_heads));
  const bool is_v = rest >= p.num_heads;
  const int h = is_v ? rest - p.num_heads : rest;
  const int D = p.head_dim, bs = p.block_size;
  const int vecs = D / kVec;                             // 16-byte pieces of a row
  const int stride = is_v ? p.value_stride_bytes : p.key_stride_bytes;
  const uint8_t* base = (is_v ? p.value : p.key) + (int64_t)h * D * sizeof(T);
  int8_t* cache = is_v ? p.v_cache : p.k_cache;
  float* scales = is_v ? p.v_scale : p.k_scale;

  // the blocks of the window's rows, the row before and those after: lane i has row t_begin - 1 + i
  // (-1: no slot, -2: a slot past the pool)
  auto block_at = [&](int t, bool* opens) -> int {
    const int64_t slot = t >= 0 && t < p.num_tokens ? __ldg(p.slots + t) : -1;
    *opens = false;
    if (slot < 0) return -1;
    if (slot >= p.capacity) return -2;
    const int blk = static_cast<int>(block_of(slot, bs));
    *opens = slot == (int64_t)blk * bs;  // offset 0
    return blk;
  };
  bool open_l;
  const int blk_l = block_at(t_begin - 1 + lane, &open_l);
  if (rest == 0 && lane >= 1 && lane <= p.window && blk_l == -2) report(p.err, VFL_DEVERR_SLOT);
  const int before = __shfl_up_sync(kAll, blk_l, 1);
  const uint32_t change = __ballot_sync(kAll, lane >= 1 && blk_l != before);
  const uint32_t opens = __ballot_sync(kAll, open_l);
  uint32_t starts = __ballot_sync(kAll, lane >= 1 && lane <= p.window && blk_l >= 0 && blk_l != before);

  while (starts != 0) {
    const int at = __ffs(starts) - 1;
    starts &= starts - 1;
    const int t = t_begin - 1 + at;
    const int blk = __shfl_sync(kAll, blk_l, at);
    const uint32_t after = at < 31 ? change >> (at + 1) << (at + 1) : 0u;  // where the run ends, if it ends here
    const int stop = after ? __ffs(after) - 1 : 32;
    int n = stop - at;
    bool fresh = (opens >> at & (n < 32 ? (1u << n) - 1 : kAll)) != 0;
    if (!after) {  // past the rows at hand
      for (;;) {
        bool open;
        const int b = block_at(t + n + lane, &open);
        const uint32_t other = __ballot_sync(kAll, b != blk);
        const int more = other ? __ffs(other) - 1 : 32;
        fresh |= (__ballot_sync(kAll, lane < more && open)) != 0;
        n += more;
        if (other) break;
      }
    }

    // 16-byte pieces of the run; lane by lane, neighbours in a row first
    const int pieces = n * vecs;
    const uint8_t* rows = base + t * (int64_t)stride;
    auto row_of = [&](int i) -> int {  // i / vecs: the product with the inverse is one too many at most
      const int j = __umulhi(i, p.inverse);
      return j - (j * vecs > i);
    };
    const int j0 = row_of(lane), c0 = lane - j0 * vecs;
    // row and place in it of this lane's piece i = lane + 32 q
    auto find = [&](int i, int* c) -> int {
      if (kEven) {
        *c = c0;
        return j0 + (i >> 5) * p.rows_per_warp;
      }
      const int j = row_of(i);
      *c = i - j * vecs;
      return j;
    };
    auto piece = [&](int i) -> uint4 {
      int c;
      const int j = find(i, &c);
      return __ldg(reinterpret_cast<const uint4*>(rows + j * (int64_t)stride) + c);
    };
    uint4 v[kHeld];
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
      v[q] = make_uint4(0u, 0u, 0u, 0u);
      if (q * 32 + lane < pieces) v[q] = piece(q * 32 + lane);
    }
    // take the block's scale
    uint32_t* word = reinterpret_cast<uint32_t*>(scales + (int64_t)blk * p.num_heads + h);
    uint32_t old_bits = 0;
    if (lane == 0) {
      old_bits = exchange_acquire(word, kScaleLocked);
      if (old_bits == kScaleLocked) {
        const uint64_t t0 = globaltimer_ns();
        do {
          __nanosleep(100);
          old_bits = exchange_acquire(word, kScaleLocked);
        } while (old_bits == kScaleLocked && globaltimer_ns() - t0 < kLockLimitNs);
      }
    }

    // largest finite magnitude of the run
    float largest = 0.f;
    auto fold = [&](const uint4& w) {  // a NaN stays
      float f[kVec];
      unpack16(w, f, T());
#pragma unroll
      for (int i = 0; i < kVec; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(f[i])));
    };
#pragma unroll
    for (int q = 0; q < kHeld; ++q) fold(v[q]);
#pragma unroll 4
    for (int i = kHeld * 32 + lane; i < pieces; i += 32) fold(piece(i));
    const bool odd = __any_sync(kAll, !(largest <= 3.402823466e38f));
    if (odd) {
      if (lane == 0) report(p.err, VFL_DEVERR_NONFINITE);
      largest = 0.f;
#pragma unroll 1
      for (int i = lane; i < pieces; i += 32) {
        float f[kVec];
        unpack16(piece(i), f, T());
#pragma unroll
        for (int e = 0; e < kVec; ++e) largest = fmaxf(largest, fabsf(f[e]) <= 3.402823466e38f ? fabsf(f[e]) : 0.f);
      }
    }
    // magnitudes are ordered as their bits are
    largest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(largest)));
    old_bits = __shfl_sync(kAll, old_bits, 0);
    if (old_bits == kScaleLocked) {  // another run never let go: nothing is stored
      if (lane == 0) report(p.err, VFL_DEVERR_SLOT);
      continue;
    }
    const float stored = __uint_as_float(old_bits);
    const float old = fresh || !(stored > 0.f) ? 0.f : stored;
    float want = __fmul_rn(largest, 1.f / 127.f);
    want = want < kMinScale ? 0.f : want;
    const float now = fmaxf(old, want);
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;

    int8_t* block = cache + ((int64_t)blk * p.num_heads + h) * (bs * D);
    if (now > old && !fresh) {  // the step grew: the codes the block holds follow
      const float ratio = __fmul_rn(old, inv);
      uint4* b16 = reinterpret_cast<uint4*>(block);
      const int words = bs * D / 16;
      for (int i0 = lane; i0 < words; i0 += 4 * 32) {
        uint4 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i0 + q * 32 < words) w[q] = __ldcg(b16 + i0 + q * 32);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i0 + q * 32 < words)
            __stcg(b16 + i0 + q * 32, make_uint4(rescale4(w[q].x, ratio), rescale4(w[q].y, ratio),
                                                 rescale4(w[q].z, ratio), rescale4(w[q].w, ratio)));
      }
      __syncwarp();  // the new codes overwrite theirs after it
    }
    const uint32_t* low = reinterpret_cast<const uint32_t*>(p.slots + t);  // low words of the slots
    const uint32_t block_low = static_cast<uint32_t>(blk) * static_cast<uint32_t>(bs);
    auto place = [&](int i) -> int8_t* {
      int c;
      const int j = find(i, &c);
      return block + ((__ldg(low + 2 * j) - block_low) * D + c * kVec);
    };
    auto put = [&](int i, const uint4& w) {
      float f[kVec];
      unpack16(w, f, T());
      uint32_t c[kVec / 4];
#pragma unroll
      for (int e = 0; e < kVec / 4; ++e) c[e] = quantize4(f + 4 * e, inv);
      store_codes(place(i), c);
    };
    // products past 127 by more than rounding come from infinities and from a tiny scale the cache
    // held before
    if (!odd && __fmul_rn(largest, inv) < 127.5f) {
#pragma unroll
      for (int q = 0; q < kHeld; ++q)
        if (q * 32 + lane < pieces) put(q * 32 + lane, v[q]);
#pragma unroll 4
      for (int i = kHeld * 32 + lane; i < pieces; i += 32) put(i, piece(i));
    } else {
#pragma unroll 1
      for (int i = lane; i < pieces; i += 32) {
        float f[kVec];
        unpack16(piece(i), f, T());
        uint32_t c[kVec / 4];
#pragma unroll
        for (int e = 0; e < kVec / 4; ++e)
          c[e] = pack4(quantize(f[4 * e], inv), quantize(f[4 * e + 1], inv), quantize(f[4 * e + 2], inv),
                       quantize(f[4 * e + 3], inv));
        store_codes(place(i), c);
      }
    }
    __syncwarp();
    if (lane == 0) store_release(word, __float_as_uint(now));
  }
}

// a / b, with the inverse 2^32 / b rounded up: their product is one too many at most.
struct Divisor {
  uint32_t b, inverse;
  explicit Divisor(uint32_t d = 1) : b(d), inverse(d > 1 ? UINT32_MAX / d + 1 : 0) {}
  __device__ __forceinline__ uint32_t divide(uint32_t a) const {
    if (b == 1) return a;
    const uint32_t q = __umulhi(a, inverse);
    return q - (q * b > a);
  }
};

struct GatherParams {
  const int8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  uint4 *key, *value;
  const int64_t* slots;
  int64_t capacity;
  uint32_t total;               // pieces of 8 codes of the launch's tokens, below 2^31
  Divisor token_pieces, row_pieces;
  int num_heads, head_dim, block_size;
  unsigned int* err;
};

// 8 codes times their scale as 16-byte pieces of T. A byte less its sign is the low byte of the
// float32 2^23 + code + 128, from which one subtraction leaves the code exactly.
template <typename T>
__device__ __forceinline__ void spread(const uint2& w, float scale, uint4* out) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t word = (i < 4 ? w.x : w.y) ^ 0x80808080u;
    f[i] = __fmul_rn(__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7540 + (i & 3))) - 8388736.f, scale);
  }
#pragma unroll
  for (int q = 0; q < 8 / Elem<T>::kVec; ++q) out[q] = pack16(f + q * Elem<T>::kVec, T());
}

// One thread per 8 codes of K and of V; rows without a slot read as zeros. Bound: HBM, by the
// rows written (64 x 585 tokens of 12 x 64 bfloat16: 35.5 us for 172 MB, 4.9 TB/s; two or four places
// a thread with their loads in flight together: 34 and 38).
template <typename T>
__global__ void __launch_bounds__(kThreads) gather_int8_kernel(const GatherParams p) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.total) return;
  const uint32_t t = p.token_pieces.divide(i);
  const int64_t slot = __ldg(p.slots + t);
  const uint32_t rest = i - t * p.token_pieces.b;
  const uint32_t h = p.row_pieces.divide(rest), c = rest - h * p.row_pieces.b;
  if (slot >= p.capacity && rest == 0) report(p.err, VFL_DEVERR_SLOT);
  uint2 kw = make_uint2(0u, 0u), vw = kw;
  float ks = 0.f, vs = 0.f;
  if (slot >= 0 && slot < p.capacity) {
    const int64_t blk = block_of(slot, p.block_size), row = blk * p.num_heads + h;
    const int64_t src = (row * p.block_size + (slot - blk * p.block_size)) * p.head_dim + c * 8;
    kw = __ldg(reinterpret_cast<const uint2*>(p.k_cache + src));
    vw = __ldg(reinterpret_cast<const uint2*>(p.v_cache + src));
    ks = __ldg(p.k_scale + row);
    vs = __ldg(p.v_scale + row);
  }
  constexpr int kPieces = 8 / Elem<T>::kVec;
  spread<T>(kw, ks, p.key + (int64_t)i * kPieces);
  spread<T>(vw, vs, p.value + (int64_t)i * kPieces);
}

int check_cache(const char* what, int dtype, int64_t num_tokens, int num_heads, int head_dim, int block_size,
                int64_t num_blocks) {
  if (!dtype_ok(dtype)) return fail(VFL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (num_tokens < 0 || num_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "%s: bad sizes (tokens %lld, heads %d, head_dim %d, block_size %d, blocks %lld)",
                what, (long long)num_tokens, num_heads, head_dim, block_size, (long long)num_blocks);
  if ((int64_t)block_size * head_dim > INT32_MAX)
    return fail(VFL_ERR_UNSUPPORTED, "%s: block_size %d times head_dim %d", what, block_size, head_dim);
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
  p.key = static_cast<const uint8_t*>(key);
  p.value = static_cast<const uint8_t*>(value);
  if (num_tokens > INT32_MAX / 2 || key_token_stride * es > INT32_MAX || value_token_stride * es > INT32_MAX ||
      num_blocks > INT32_MAX)
    return fail(VFL_ERR_UNSUPPORTED, "reshape_and_cache_int8: tokens, blocks or token strides past 32 bits");
  p.key_stride_bytes = static_cast<int>(key_token_stride * es);
  p.value_stride_bytes = static_cast<int>(value_token_stride * es);
  p.k_cache = static_cast<int8_t*>(k_cache);
  p.v_cache = static_cast<int8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.slots = slot_mapping;
  p.num_tokens = static_cast<int>(num_tokens);
  p.capacity = num_blocks * block_size;
  p.num_heads = num_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  const int row_pieces = static_cast<int>(head_dim * es / 16);
  p.inverse = UINT32_MAX / static_cast<uint32_t>(row_pieces) + 1;
  p.rows_per_warp = 32 / row_pieces;
  // A decode step's rows are runs of one: windows of one row keep them all in flight. Many rows
  // are blocks' worth of neighbours: windows of a block leave few warps without a run.
  const int most = block_size < kMaxWindow ? block_size : kMaxWindow;
  const int64_t fit = ceil_div(num_tokens * 2 * num_heads, (int64_t)kNumSMs * 256);
  p.window = static_cast<int>(fit < most ? fit : most);
  const int64_t warps = ceil_div(num_tokens, (int64_t)p.window) * 2 * num_heads;
  const int64_t ctas = ceil_div(warps, (int64_t)kWarps);
  if (warps > INT32_MAX) return fail(VFL_ERR_UNSUPPORTED, "reshape_and_cache_int8: too many tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool even = 32 % row_pieces == 0;
  auto pick = [&](auto type) {
    using T = decltype(type);
    if (p.window == 1) return even ? append_int8_kernel<T, true, true> : append_int8_kernel<T, false, true>;
    return even ? append_int8_kernel<T, true, false> : append_int8_kernel<T, false, false>;
  };
  auto kern = dtype == VFL_DTYPE_F32 ? pick(float()) : pick(__nv_bfloat16());
  kern<<<(unsigned)ctas, kThreads, 0, s>>>(p);
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
  p.k_cache = static_cast<const int8_t*>(k_cache);
  p.v_cache = static_cast<const int8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.capacity = num_blocks * block_size;
  const int64_t token_pieces = (int64_t)num_heads * (head_dim / 8);
  if (token_pieces > (1 << 24))
    return fail(VFL_ERR_UNSUPPORTED, "gather_kv_int8: num_heads %d times head_dim %d", num_heads, head_dim);
  p.token_pieces = Divisor(static_cast<uint32_t>(token_pieces));
  p.row_pieces = Divisor(static_cast<uint32_t>(head_dim / 8));
  p.num_heads = num_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t slab = INT32_MAX / token_pieces;  // tokens whose pieces are counted in 32 bits
  for (int64_t t = 0; t < num_tokens; t += slab) {
    const int64_t tokens = num_tokens - t < slab ? num_tokens - t : slab;
    const int64_t at = t * num_heads * head_dim * (int64_t)dtype_size(dtype);
    p.slots = slot_mapping + t;
    p.key = reinterpret_cast<uint4*>(static_cast<uint8_t*>(key) + at);
    p.value = reinterpret_cast<uint4*>(static_cast<uint8_t*>(value) + at);
    p.total = static_cast<uint32_t>(tokens * token_pieces);
    const unsigned ctas = ceil_div(p.total, (uint32_t)kThreads);
    if (dtype == VFL_DTYPE_F32)
      gather_int8_kernel<float><<<ctas, kThreads, 0, s>>>(p);
    else
      gather_int8_kernel<__nv_bfloat16><<<ctas, kThreads, 0, s>>>(p);
  }
  return cuda_status(cudaGetLastError(), "gather_kv_int8 launch");
}

}  // extern "C"
