// The paged K/V cache held in 8 bits: append and read-back.
//
// A block's tokens of one head share a float32 scale: codes int8 [num_blocks, H, block_size, D],
// scales [num_blocks, H], value = code * scale. The append keeps a block consistent while it
// fills: with a = the largest finite magnitude of the call's tokens in the block, s' = max(s, a *
// (1/127)); when s' > s the codes the block holds are brought to the new step, rint(code * (s *
// (1/s'))), and the new ones are rint(x * (1/s')) held to [-127, 127]. A call that writes offset 0
// starts the block anew (s = 0). Products in float32 with one rounding each, so that a plain
// restatement gives the same codes bit for bit. A growth rounds the older codes once more (at most
// half a step).
//
// Both kernels move bytes: the bound is HBM for many tokens and one dependent round trip (slot,
// then the block's scale and the token) for a few.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxWindow = 16;  // rows whose runs one warp stores, at most 31

// Smallest scale kept: the attention divides by V scales, and 2^100 times a context's token
// count stays inside float32. Blocks whose largest magnitude is below 127 * 2^-100 hold zeros.
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100

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
  uint32_t parts;            // CTAs that share a window's heads
  int threads;               // of each
  int block_mask;            // block_size - 1 where that is a power of two, else 0
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

constexpr float kFloatMax = 3.402823466e38f;

// The scale of a block that held tokens of step `old` and takes tokens of magnitude `largest`.
__device__ __forceinline__ float next_scale(float old, float largest) {
  const float want = __fmul_rn(largest, 1.f / 127.f);
  return fmaxf(old, want < kMinScale ? 0.f : want);
}

// Codes of `bytes` bytes of a block, brought to another step by one warp.
__device__ __forceinline__ void rescale_block(int8_t* block, int bytes, float ratio, int lane) {
  uint4* b16 = reinterpret_cast<uint4*>(block);
  const int words = bytes / 16;
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

// Low words of the slots of rows r0 + lane, r0 + 32 + lane ...
template <int kLook>
__device__ __forceinline__ void look_at(const AppendParams& p, int r0, uint32_t (&word)[kLook]) {
  const uint32_t* low = reinterpret_cast<const uint32_t*>(p.slots + r0 + (threadIdx.x & 31));
  if (r0 + 32 * kLook <= p.num_tokens) {
#pragma unroll
    for (int u = 0; u < kLook; ++u) word[u] = __ldg(low + u * 64);
  } else {
    const int left = p.num_tokens - r0 - static_cast<int>(threadIdx.x & 31);
#pragma unroll
    for (int u = 0; u < kLook; ++u) word[u] = u * 32 < left ? __ldg(low + u * 64) : 0xffffffffu;
  }
}

// Whether one of these rows may lie in the `bs` slots from slot0 on (or among slots 2^32 apart)
template <int kLook>
__device__ __forceinline__ bool may_hit(const uint32_t (&word)[kLook], int64_t slot0, int bs) {
  uint32_t least = 0xffffffffu;
#pragma unroll
  for (int u = 0; u < kLook; ++u) least = __viaddmin_u32(word[u], 0u - (uint32_t)slot0, least);
  return least < (uint32_t)bs;
}

// The run that begins at row t, and where `more_rows` says so the later rows of its block, stored by
// a warp piece by piece: blocks whose rows are not neighbours, infinities and NaNs among the tokens, and
// products past 127 by more than rounding (from a tiny scale the cache held before).
template <typename T>
__device__ __noinline__ void store_slowly(const AppendParams& p, bool is_v, int h, int blk, int t, bool more_rows) {
  constexpr int kVec = Elem<T>::kVec;
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int D = p.head_dim, bs = p.block_size, vecs = D / kVec;
  const int64_t slot0 = (int64_t)blk * bs, at_head = (int64_t)blk * p.num_heads + h;
  const uint8_t* base = (is_v ? p.value : p.key) + (int64_t)h * D * sizeof(T);
  const int stride = is_v ? p.value_stride_bytes : p.key_stride_bytes;
  int8_t* block = (is_v ? p.v_cache : p.k_cache) + at_head * (bs * D);
  float* scale_at = (is_v ? p.v_scale : p.k_scale) + at_head;
  auto each = [&](auto&& take) {
    constexpr int kLook = 16;
    unsigned long long had = 0;  // offsets met: up to 64 slots they tell when the block is complete
    bool done = false;
#pragma unroll 1
    for (int r0 = t; r0 < p.num_tokens && !done; r0 += 32 * kLook) {
      uint32_t word[kLook];
      look_at(p, r0, word);
      if (!__any_sync(kAll, may_hit(word, slot0, bs))) continue;
#pragma unroll 1
      for (int j0 = r0; j0 < min(r0 + 32 * kLook, p.num_tokens) && !done; j0 += 32) {
        const int64_t slot = j0 + lane < p.num_tokens ? __ldg(p.slots + j0 + lane) : -1;
        uint32_t rows = __ballot_sync(kAll, (uint64_t)(slot - slot0) < (uint64_t)bs);
        if (!more_rows) {
          done = rows != kAll;
          rows &= ~(rows + 1);  // those before the first of another block
        }
#pragma unroll 1
        for (; rows != 0; rows &= rows - 1) {
          const int l = __ffs(rows) - 1;
          const uint32_t offset = __shfl_sync(kAll, (uint32_t)(slot - slot0), l);
          had |= 1ull << (offset & 63);
          const uint4* row = reinterpret_cast<const uint4*>(base + (j0 + l) * (int64_t)stride);
#pragma unroll 1
          for (int c = lane; c < vecs; c += 32) take(__ldg(row + c), offset, c);
        }
        done |= bs <= 64 && __popcll(had) == bs;
      }
    }
  };
  float largest = 0.f;
  bool odd = false, zero = false;
  each([&](const uint4& w, uint32_t offset, int) {
    float f[kVec];
    unpack16(w, f, T());
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const bool finite = fabsf(f[e]) <= kFloatMax;
      largest = fmaxf(largest, finite ? fabsf(f[e]) : 0.f);
      odd |= !finite;
    }
    zero |= offset == 0;
  });
  if (odd) report(p.err, VFL_DEVERR_NONFINITE);
  largest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(largest)));
  const bool fresh = __any_sync(kAll, zero);
  const float stored = __ldcg(scale_at);
  const float old = fresh || !(stored > 0.f) ? 0.f : stored;
  const float now = next_scale(old, largest);
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  if (now > old && !fresh) rescale_block(block, bs * D, __fmul_rn(old, inv), lane);
  each([&](const uint4& w, uint32_t offset, int c) {
    float f[kVec];
    unpack16(w, f, T());
    uint32_t codes[kVec / 4];
#pragma unroll
    for (int e = 0; e < kVec / 4; ++e)
      codes[e] = pack4(quantize(f[4 * e], inv), quantize(f[4 * e + 1], inv), quantize(f[4 * e + 2], inv),
                       quantize(f[4 * e + 3], inv));
    store_codes(block + (offset * D + c * kVec), codes);
  });
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale_at = now;
}

// What a warp works on: one head of K or of V. The CTAs of a window share its heads; a last warp may
// have none (`on` is false): it takes part in what its CTA does.
struct Side {
  const uint8_t* base;  // the head's rows
  int stride;
  int8_t* cache;
  float* scales;
  int h;
  bool on, is_v;
  __device__ __forceinline__ Side(const AppendParams& p, int elem_size) {
    const int rest = static_cast<int>(blockIdx.x % p.parts * (blockDim.x >> 5) + (threadIdx.x >> 5));
    on = rest < 2 * p.num_heads;
    is_v = on && rest >= p.num_heads;
    h = !on ? 0 : (is_v ? rest - p.num_heads : rest);
    base = (is_v ? p.value : p.key) + (int64_t)h * p.head_dim * elem_size;
    stride = is_v ? p.value_stride_bytes : p.key_stride_bytes;
    cache = is_v ? p.v_cache : p.k_cache;
    scales = is_v ? p.v_scale : p.k_scale;
  }
};

// Where a run whose first slot is `slot` is told whose it is (see kRunAlone), for the CTAs of a part: in
// the code row of that slot, of the head of the CTAs' first warp.
__device__ __forceinline__ uint32_t* told_at(const AppendParams& p, int64_t slot, uint32_t part) {
  const int first = part * (p.threads >> 5);
  const int h = first < p.num_heads ? first : first - p.num_heads;
  const int64_t blk = block_of(slot, p.block_size), off = slot - blk * p.block_size;
  int8_t* cache = first < p.num_heads ? p.k_cache : p.v_cache;
  return reinterpret_cast<uint32_t*>(cache + ((blk * p.num_heads + h) * p.block_size + off) * p.head_dim);
}

// Row t's block (-1: no slot, -2: a slot past the pool), whether it is the block's first slot, and the
// slot less the row, which is the same all along a run in order.
__device__ __forceinline__ int block_at(const AppendParams& p, int t, bool* opens, uint32_t* lead) {
  const int64_t slot = t >= 0 && t < p.num_tokens ? __ldg(p.slots + t) : -1;
  *opens = false;
  *lead = (uint32_t)slot - t;
  if (slot < 0) return -1;
  if (slot >= p.capacity) return -2;
  const int blk = static_cast<int>(block_of(slot, p.block_size));
  *opens = slot == (int64_t)blk * p.block_size;
  return blk;
}

// Goes on with a run of block `blk` from its n-th row on, past the rows that a warp has at hand.
__device__ __forceinline__ void extend_run(const AppendParams& p, int t, int blk, uint32_t lead, int* n, bool* open,
                                           bool* in_order) {
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  for (;;) {
    bool open_b;
    uint32_t lead_b;
    const int b = block_at(p, t + *n + lane, &open_b, &lead_b);
    const uint32_t other = __ballot_sync(kAll, b != blk);
    const int more = other ? __ffs(other) - 1 : 32;
    *open |= __any_sync(kAll, lane < more && open_b);
    *in_order &= !__any_sync(kAll, lane < more && lead_b != lead);
    *n += more;
    if (other) return;
  }
}

// The 16-byte pieces of a run, neighbours in a row first.
template <typename T>
struct Pieces {
  const uint8_t* rows;
  int stride, vecs, count;
  uint32_t inverse;
  __device__ __forceinline__ Pieces(const AppendParams& p, const Side& side, int t, int n)
      : rows(side.base + t * (int64_t)side.stride), stride(side.stride), vecs(p.head_dim / Elem<T>::kVec),
        count(n * vecs), inverse(p.inverse) {}
  // row of piece i, and its place in it: the product with the inverse is one too many at most
  __device__ __forceinline__ int row(int i, int* c) const {
    int j = __umulhi(i, inverse);
    j -= j * vecs > i;
    *c = i - j * vecs;
    return j;
  }
  __device__ __forceinline__ uint4 load(int j, int c) const {
    return __ldg(reinterpret_cast<const uint4*>(rows + j * (int64_t)stride) + c);
  }
};

// largest = the larger of it and the magnitudes of a piece; a NaN stays
template <typename T>
__device__ __forceinline__ void fold(float& largest, const uint4& w) {
  float f[Elem<T>::kVec];
  unpack16(w, f, T());
#pragma unroll
  for (int i = 0; i < Elem<T>::kVec; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(f[i])));
}

template <typename T>
__device__ __forceinline__ void put(int8_t* to, const uint4& w, float inv) {
  constexpr int kVec = Elem<T>::kVec;
  float f[kVec];
  unpack16(w, f, T());
  uint32_t codes[kVec / 4];
#pragma unroll
  for (int e = 0; e < kVec / 4; ++e) codes[e] = quantize4(f + 4 * e, inv);
  store_codes(to, codes);
}

// A warp stores a run of consecutive rows in one block: all of an encoder block's tokens, or the one
// token of a decode step. Its largest magnitude is known before its first code is written, so a block
// filled by one call is rounded once.
//
// A block may have other rows in the call (time-major prompts; a padding row in a block's middle). Its
// first run stores them all, unless a run is the whole block in order, which leaves no slot to another
// row. So a block is written by one warp a head and needs no lock, and the order of the rows changes
// nothing. Which run is whose is found out by a kernel before (many rows) or by the CTA that stores the
// row (few).

// What a run that is not a whole block in order is told, in the first 4 bytes of code rows of its first
// slot (see told_at). A CTA has read its word before it stores, and the bytes are written anew with the
// run's codes. No code is -128: a run whose word the codes of another have overwritten is a later one.
constexpr uint32_t kRunAlone = 0x80808001u;  // the block's only run
constexpr uint32_t kRunFirst = 0x80808002u;  // the block has more
constexpr uint32_t kRunLater = 0x80808000u;  // another run stores its rows

constexpr int kRunsCluster = 8;
constexpr int kRunsThreads = 1024;
constexpr int kRunsPerCta = 2048;  // rows, and so runs at most, for which a launch has a CTA
constexpr int kTableSize = 4096;   // blocks of a CTA's table
constexpr int kListSize = 3584;    // its entries, and the runs of a CTA's list, at most

// Tells the runs. A cluster looks at all slots, each CTA at a stretch of them, and keeps the runs of a
// share of the blocks, by a hash of their numbers: each in the list of the CTA that met it, their blocks
// with their first rows in the CTAs' tables. The launch after it reads its slots and rows meanwhile.
//
// Measured: 13 to 16 us alone (37000 to 60000 rows; 50 for 512 x 585), nearly all of it beside the launch
// after it: an append of 3000 prompts of 20 tokens (12 x 64 bfloat16) takes 143 us, of 512 x 585 rows 466.
// With each storing CTA looking through the slots, as for few rows, they took 318 and 520, and 64 x 585
// rows 59 as they do here.
__global__ void __cluster_dims__(kRunsCluster, 1, 1) __launch_bounds__(kRunsThreads)
append_int8_runs_kernel(const __grid_constant__ AppendParams p) {
  griddep_launch_dependents();
  __shared__ int s_block[kTableSize], s_first[kTableSize];  // -1: no block
  __shared__ uint32_t s_more[kTableSize / 32], s_whole[kTableSize / 32];  // has several runs; one in order
  __shared__ int s_list[kListSize], s_count, s_used;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), lane = threadIdx.x & 31;
  const uint32_t share = blockIdx.x / kRunsCluster, shares = gridDim.x / kRunsCluster;
  const int bs = p.block_size;
  for (int i = threadIdx.x; i < kTableSize; i += kRunsThreads) {
    s_block[i] = -1;
    s_first[i] = INT32_MAX;
  }
  for (int i = threadIdx.x; i < kTableSize / 32; i += kRunsThreads) s_more[i] = s_whole[i] = 0;
  if (threadIdx.x == 0) s_count = s_used = 0;
  cluster.sync();

  auto slot_at = [&](int row) { return row >= 0 && row < p.num_tokens ? __ldg(p.slots + row) : -1; };
  auto inside = [&](int64_t slot, int64_t slot0) { return (uint64_t)(slot - slot0) < (uint64_t)bs; };
  auto hash_of = [](int blk) { return (uint32_t)blk * 2654435761u; };
  auto table_of = [&](int blk) { return static_cast<int>(hash_of(blk) >> 12) & (kRunsCluster - 1); };  // whose it is in
  // the entry of a block in a table: its own, or the free one where it is to be
  auto entry_of = [&](const int* blocks, int blk) {
    uint32_t i = (hash_of(blk) ^ (uint32_t)blk >> 9) % kTableSize;
    for (;; i = (i + 1) % kTableSize) {
      const int there = *const_cast<volatile const int*>(blocks + i);
      if (there == -1 || there == blk) return i;
    }
  };

  // this CTA's stretch
  const int per = ceil_div(ceil_div(p.num_tokens, kRunsCluster), 32) * 32, r_begin = rank * per;
  const int r_end = min(r_begin + per, p.num_tokens);
  constexpr int kFlight = 4;
  for (int r0 = r_begin + threadIdx.x; r0 - lane < r_end; r0 += kFlight * kRunsThreads) {
    int64_t slot[kFlight], edge[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int row = r0 + u * kRunsThreads;
      slot[u] = row < r_end ? slot_at(row) : -1;
      edge[u] = lane == 0 ? slot_at(row - 1) : -1;
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      int64_t before = __shfl_up_sync(0xffffffffu, slot[u], 1);
      if (lane == 0) before = edge[u];
      // a run goes on, most often, with the next slot of the block
      if (slot[u] < 0 || slot[u] >= p.capacity || (slot[u] == before + 1 && p.block_mask && (slot[u] & p.block_mask))) continue;
      const int blk = static_cast<int>(block_of(slot[u], bs));
      if (inside(before, (int64_t)blk * bs) || __umulhi(hash_of(blk), shares) != share) continue;
      const int at = atomicAdd(&s_count, 1);
      if (at < kListSize) s_list[at] = r0 + u * kRunsThreads;
    }
  }
  __syncthreads();

  auto whole_block = [&](int row, int64_t slot, int64_t slot0) {  // the run that begins here is, in order, and ends
    bool same = slot == slot0 && slot_at(row + bs - 1) == slot + bs - 1 && !inside(slot_at(row + bs), slot0);
    for (int i = 1; i < bs - 1 && same; ++i) same = slot_at(row + i) == slot + i;
    return same;
  };
  const int runs = min(s_count, kListSize);
  for (int j = threadIdx.x; j < runs; j += kRunsThreads) {
    const int row = s_list[j];
    const int64_t slot = slot_at(row);
    const int blk = static_cast<int>(block_of(slot, bs)), to = table_of(blk);
    const bool whole = whole_block(row, slot, (int64_t)blk * bs);
    if (whole) s_list[j] = -1;
    // entries are counted before they are made, so that a table never fills up
    if (atomicAdd(cluster.map_shared_rank(&s_used, to), 1) >= kListSize) continue;
    int* blocks = cluster.map_shared_rank(s_block, to);
    uint32_t i = entry_of(blocks, blk);
    int old = atomicCAS(blocks + i, -1, blk);
    while (old != -1 && old != blk) {  // another block took it
      i = entry_of(blocks, blk);
      old = atomicCAS(blocks + i, -1, blk);
    }
    atomicMin(cluster.map_shared_rank(s_first, to) + i, row);
    if (old == blk) atomicOr(cluster.map_shared_rank(s_more, to) + i / 32, 1u << i % 32);
    if (whole) atomicOr(cluster.map_shared_rank(s_whole, to) + i / 32, 1u << i % 32);
  }
  cluster.sync();

  auto tell = [&](int64_t slot, uint32_t what) {
    for (uint32_t part = 0; part < p.parts; ++part) __stcg(told_at(p, slot, part), what);
  };
  bool fits = true;
  for (int c = 0; c < kRunsCluster; ++c)
    fits &= *cluster.map_shared_rank(&s_count, c) <= kListSize && *cluster.map_shared_rank(&s_used, c) <= kListSize;
  if (fits) {
    for (int j = threadIdx.x; j < runs; j += kRunsThreads) {
      const int row = s_list[j];
      if (row < 0) continue;
      const int64_t slot = slot_at(row);
      const int blk = static_cast<int>(block_of(slot, bs)), in = table_of(blk);
      const uint32_t i = entry_of(cluster.map_shared_rank(s_block, in), blk);
      uint32_t what = kRunAlone;
      if (cluster.map_shared_rank(s_more, in)[i / 32] >> i % 32 & 1)
        what = cluster.map_shared_rank(s_first, in)[i] == row ? kRunFirst : kRunLater;
      if (cluster.map_shared_rank(s_whole, in)[i / 32] >> i % 32 & 1) what = kRunLater;
      tell(slot, what);
    }
  } else {  // more runs than that (their blocks' numbers meet in the hash): each looks for itself
    for (int row = r_begin + threadIdx.x; row < r_end; row += kRunsThreads) {
      const int64_t slot = slot_at(row);
      if (slot < 0 || slot >= p.capacity) continue;
      const int blk = static_cast<int>(block_of(slot, bs));
      const int64_t slot0 = (int64_t)blk * bs;
      if (__umulhi(hash_of(blk), shares) != share || inside(slot_at(row - 1), slot0) || whole_block(row, slot, slot0)) continue;
      int end = row + 1;
      while (inside(slot_at(end), slot0)) ++end;
      uint32_t what = kRunAlone;
      for (int j = 0; j < p.num_tokens && what != kRunLater; ++j)
        if ((j < row || j >= end) && inside(slot_at(j), slot0)) what = j < row ? kRunLater : kRunFirst;
      tell(slot, what);
    }
  }
  cluster.sync();  // no CTA leaves while another still reads its table
}

// The runs of many rows: a warp takes those that begin in its window of rows. A run of up to kHeld pieces
// a lane stays in registers from its maximum to its codes; a longer one is read a second time.
//
// kEven: a row's pieces divide the warp, so a lane's pieces are a fixed step of rows apart.
//
// Measured: 64 x 585 tokens of 12 x 64 bfloat16 60 us, 172 MB at 2.9 TB/s: the instructions (780 a run of
// 16 rows, 0.73 a clock and scheduler) are the bound; 80 registers, for three CTAs an SM instead of four,
// changed nothing. 2000 single rows of 16 x 64 46 us. The same 64 x 585 rows token by token of all
// requests, which take the slow way block by block: 0.76 ms.
template <typename T, bool kEven>
__global__ void __launch_bounds__(kThreads, 4) append_int8_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kVec = Elem<T>::kVec;
  constexpr int kHeld = 4;
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int t_begin = blockIdx.x / p.parts * p.window;
  const Side side(p, sizeof(T));
  const int D = p.head_dim, bs = p.block_size;

  // lane i has row t_begin - 1 + i: those of the window, the one before and those after
  bool open_l;
  uint32_t lead_l;
  const int blk_l = block_at(p, t_begin - 1 + lane, &open_l, &lead_l);
  if (side.on && side.h == 0 && !side.is_v && lane >= 1 && lane <= p.window && blk_l == -2) report(p.err, VFL_DEVERR_SLOT);
  const int before = __shfl_up_sync(kAll, blk_l, 1);
  const uint32_t change = __ballot_sync(kAll, lane >= 1 && blk_l != before);
  const uint32_t opens = __ballot_sync(kAll, open_l);
  uint32_t starts = __ballot_sync(kAll, lane >= 1 && lane <= p.window && blk_l >= 0 && blk_l != before);

  // the runs' lengths (lane i: of the run at row t_begin - 1 + i), whether they write offset 0, and
  // which of them are not a whole block in order
  int n_l = 0;
  uint32_t fresh = 0, partial = 0;
#pragma unroll 1
  for (uint32_t left = starts; left != 0; left &= left - 1) {
    const int at = __ffs(left) - 1;
    const int blk = __shfl_sync(kAll, blk_l, at);
    const uint32_t lead = __shfl_sync(kAll, lead_l, at);
    const uint32_t after = at < 31 ? change >> (at + 1) << (at + 1) : 0u;  // where the run ends, if it ends here
    int n = (after ? __ffs(after) - 1 : 32) - at;
    const uint32_t here = (n < 32 ? (1u << n) - 1 : kAll) << at;
    bool open = (opens & here) != 0;
    bool in_order = (__ballot_sync(kAll, lead_l != lead) & here) == 0;
    if (!after && !(in_order && n == bs)) extend_run(p, t_begin - 1 + at, blk, lead, &n, &open, &in_order);
    if (lane == at) n_l = n;
    fresh |= open ? 1u << at : 0u;
    partial |= in_order && n == bs ? 0u : 1u << at;
  }

  // what these runs were told
  uint32_t apart = 0;
  if (partial != 0) {
    griddep_wait();
    uint32_t told = 0;
    if (partial >> lane & 1) told = __ldcg(told_at(p, __ldg(p.slots + t_begin - 1 + lane), blockIdx.x % p.parts));
    apart = __ballot_sync(kAll, told == kRunFirst);
    starts &= ~partial | apart | __ballot_sync(kAll, told == kRunAlone);
    __syncthreads();  // every warp has read before one stores
  }
  if (!side.on) return;

  uint32_t slow = apart;  // runs left for the end
  for (starts &= ~apart; starts != 0; starts &= starts - 1) {
    const int at = __ffs(starts) - 1;
    const int t = t_begin - 1 + at;
    const int blk = __shfl_sync(kAll, blk_l, at), n = __shfl_sync(kAll, n_l, at);
    const float stored = __ldcg(side.scales + (int64_t)blk * p.num_heads + side.h);
    const Pieces<T> run(p, side, t, n);
    int c0;
    const int j0 = run.row(lane, &c0);
    // row and place in it of this lane's piece i = lane + 32 q
    auto find = [&](int i, int* c) -> int {
      if (!kEven) return run.row(i, c);
      *c = c0;
      return j0 + (i >> 5) * p.rows_per_warp;
    };
    auto piece = [&](int i) -> uint4 {
      int c;
      const int j = find(i, &c);
      return run.load(j, c);
    };
    uint4 v[kHeld];
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
      v[q] = make_uint4(0u, 0u, 0u, 0u);
      if (q * 32 + lane < run.count) v[q] = piece(q * 32 + lane);
    }
    float largest = 0.f;  // finite magnitude of the run
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
      if (q * 32 >= run.count) break;
      fold<T>(largest, v[q]);
    }
#pragma unroll 4
    for (int i = kHeld * 32 + lane; i < run.count; i += 32) fold<T>(largest, piece(i));
    const bool odd = __any_sync(kAll, !(largest <= kFloatMax));
    // magnitudes are ordered as their bits are
    largest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(largest)));
    const bool anew = fresh >> at & 1;
    const float old = anew || !(stored > 0.f) ? 0.f : stored;
    const float now = next_scale(old, largest);
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
    int8_t* block = side.cache + ((int64_t)blk * p.num_heads + side.h) * (bs * D);
    if (odd || !(__fmul_rn(largest, inv) < 127.5f)) {
      slow |= 1u << at;
      continue;
    }
    if (now > old && !anew) rescale_block(block, bs * D, __fmul_rn(old, inv), lane);  // the step grew
    const uint32_t* low = reinterpret_cast<const uint32_t*>(p.slots + t);  // low words of the slots
    auto place = [&](int i) -> int8_t* {
      int c;
      const int j = find(i, &c);
      return block + ((__ldg(low + 2 * j) - (uint32_t)blk * (uint32_t)bs) * D + c * kVec);
    };
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
      if (q * 32 >= run.count) break;
      if (q * 32 + lane < run.count) put<T>(place(q * 32 + lane), v[q], inv);
    }
#pragma unroll 4
    for (int i = kHeld * 32 + lane; i < run.count; i += 32) put<T>(place(i), piece(i), inv);
    if (lane == 0) side.scales[(int64_t)blk * p.num_heads + side.h] = now;
  }
#pragma unroll 1
  for (; slow != 0; slow &= slow - 1) {
    const int at = __ffs(slow) - 1;
    store_slowly<T>(p, side.is_v, side.h, __shfl_sync(kAll, blk_l, at), t_begin - 1 + at, apart >> at & 1);
  }
  if (blockIdx.x == gridDim.x - 1) griddep_wait();  // this launch ends after the one before it
}

// Few rows, as in a decode step: a CTA has one row, whose run is most often itself, and eight CTAs share
// an SM. The chain of slot, token and store is the time, so the slots of the other rows are read with
// the row's own. 4 tokens of 16 x 64 float32 3.0 us, 256 of bfloat16 6.2, 512 of 16 x 128 10.3.
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) append_int8_row_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kVec = Elem<T>::kVec;
  constexpr int kLook = 4;
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x / p.parts, bs = p.block_size;
  uint32_t word[kLook];
  const int warp_rows = (blockDim.x >> 5) * (32 * kLook);
  int r0 = (threadIdx.x >> 5) * (32 * kLook);
  if (r0 < p.num_tokens) look_at(p, r0, word);
  bool open_l;
  uint32_t lead_l;
  const int blk_l = block_at(p, t - 1 + lane, &open_l, &lead_l);
  const int blk = __shfl_sync(kAll, blk_l, 1);
  if (blk == -2 && blockIdx.x % p.parts == 0 && threadIdx.x == 0) report(p.err, VFL_DEVERR_SLOT);
  if (blk < 0 || blk == __shfl_sync(kAll, blk_l, 0)) return;
  const Side side(p, sizeof(T));
  const uint32_t lead = __shfl_sync(kAll, lead_l, 1);
  const uint32_t after = __ballot_sync(kAll, blk_l != blk) >> 1;
  int n = after ? __ffs(after) - 1 : 31;
  const uint32_t here = ((1u << n) - 1) << 1;
  bool anew = (__ballot_sync(kAll, open_l) & here) != 0;
  bool in_order = (__ballot_sync(kAll, lead_l != lead) & here) == 0;
  if (!after) extend_run(p, t, blk, lead, &n, &anew, &in_order);

  const Pieces<T> run(p, side, t, n);
  float* const scale_at = side.scales + (int64_t)blk * p.num_heads + side.h;
  const float stored = __ldcg(scale_at);
  int c0;
  const int j0 = run.row(lane, &c0);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (lane < run.count) v = run.load(j0, c0);

  bool apart = false;
  if (!(in_order && n == bs)) {
    const int64_t slot0 = (int64_t)blk * bs;
    bool hit = false, earlier = false;
#pragma unroll 1
    while (r0 < p.num_tokens) {
      if (__any_sync(kAll, may_hit(word, slot0, bs))) {  // the whole slots decide
#pragma unroll 1
        for (int row = r0 + lane; row < min(r0 + 32 * kLook, p.num_tokens); row += 32) {
          if ((uint64_t)(__ldg(p.slots + row) - slot0) >= (uint64_t)bs || (uint32_t)(row - t) < (uint32_t)n) continue;
          hit = true;
          earlier |= row < t;
        }
        __syncwarp();
      }
      r0 += warp_rows;
      if (r0 < p.num_tokens) look_at(p, r0, word);
    }
    apart = __syncthreads_or(hit);
    if (apart && __syncthreads_or(earlier)) return;  // the block's first run stores this one's rows
  }
  if (!side.on) return;

  float largest = 0.f;  // finite magnitude of the run
  fold<T>(largest, v);
#pragma unroll 1
  for (int i = 32 + lane; i < run.count; i += 32) {
    int c;
    const int j = run.row(i, &c);
    fold<T>(largest, run.load(j, c));
  }
  const bool odd = __any_sync(kAll, !(largest <= kFloatMax));
  largest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(largest)));
  const float old = anew || !(stored > 0.f) ? 0.f : stored;
  const float now = next_scale(old, largest);
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  if (apart || odd || !(__fmul_rn(largest, inv) < 127.5f)) {
    store_slowly<T>(p, side.is_v, side.h, blk, t, apart);
    return;
  }
  const int D = p.head_dim;
  int8_t* block = side.cache + ((int64_t)blk * p.num_heads + side.h) * (bs * D);
  if (now > old && !anew) rescale_block(block, bs * D, __fmul_rn(old, inv), lane);  // the step grew
  const uint32_t* low = reinterpret_cast<const uint32_t*>(p.slots + t);  // low words of the slots
  auto place = [&](int j, int c) -> int8_t* {
    return block + ((__ldg(low + 2 * j) - (uint32_t)blk * (uint32_t)bs) * D + c * kVec);
  };
  if (lane < run.count) put<T>(place(j0, c0), v, inv);
#pragma unroll 1
  for (int i = 32 + lane; i < run.count; i += 32) {
    int c;
    const int j = run.row(i, &c);
    put<T>(place(j, c), run.load(j, c), inv);
  }
  if (lane == 0) *scale_at = now;
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
// a thread with their loads in flight together: 34 and 38, and slower for small calls and float32).
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
  p.block_mask = (block_size & (block_size - 1)) == 0 ? block_size - 1 : 0;
  // the CTAs of a window share its heads evenly
  p.parts = ceil_div(2u * num_heads, (uint32_t)kWarps);
  const unsigned threads = 32 * ceil_div(2u * num_heads, p.parts);
  p.threads = static_cast<int>(threads);
  const int64_t ctas = ceil_div(num_tokens, (int64_t)p.window) * p.parts;
  if (num_heads > INT32_MAX / 4 || ctas > INT32_MAX) return fail(VFL_ERR_UNSUPPORTED, "reshape_and_cache_int8: too many tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool even = 32 % row_pieces == 0;
  auto pick = [&](auto type) {
    using T = decltype(type);
    if (p.window == 1) return append_int8_row_kernel<T>;
    return even ? append_int8_kernel<T, true> : append_int8_kernel<T, false>;
  };
  auto kern = dtype == VFL_DTYPE_F32 ? pick(float()) : pick(__nv_bfloat16());
  if (p.window == 1) {
    kern<<<(unsigned)ctas, threads, 0, s>>>(p);
    return cuda_status(cudaGetLastError(), "reshape_and_cache_int8 launch");
  }
  const int64_t shares = ceil_div(num_tokens, (int64_t)(kRunsPerCta * kRunsCluster));
  append_int8_runs_kernel<<<(unsigned)(shares * kRunsCluster), kRunsThreads, 0, s>>>(p);
  st = cuda_status(cudaGetLastError(), "reshape_and_cache_int8 launch of its runs");
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "reshape_and_cache_int8 launch");
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
