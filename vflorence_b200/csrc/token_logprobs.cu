// Log probabilities of given tokens, with each row's entropy and its most likely alternatives.
//
// For a row x of `vocab` scores, with m = max x and sums over the row
//     S = sum e^(x - m),   U = sum (x - m) e^(x - m):
//     log p(t) = x_t - m - ln S,   entropy = -sum p ln p = ln S - U / S,
//     alternatives: the k largest x (ties: lower index first) as log probabilities.
// S and U are float32 running sums against a running maximum. x - m is taken before it is scaled
// for the base-2 exponential: entries and m may be near float32's lowest value, where m log2 e
// overflows, or large, where its rounding would shift the whole row. An entry of -inf (a
// forbidden token) adds nothing. Bound: HBM, the row read once.
//
// One pass gives the sums and, in shared memory, the largest value of each thread's batches of four
// 16-byte vectors. A value T is then taken that at least k, and not many more, of the maxima of 128 groups
// of threads reach: a lower bound of the k-th largest entry, since the maxima are distinct entries.
// Only batches whose maximum reaches T, a few more than k, are read again, from L2; their entries
// >= T are ranked by counting. (A bound from the first batches, with entries picked up as they
// pass, reads nothing twice but collects six times as many: 58 us against 36 at 1024 x 51289,
// k = 20.) Where ties at T overflow the list (rows of mostly one value), the bound becomes the k-th
// best (value, index) pair of the threads' best entries and the collection runs again. A row is
// cut over a cluster of up to 8 CTAs when there are few rows; the pieces meet in the first CTA's
// shared memory.
//
// The pass is close to two other bounds: 1024 x 51289 bfloat16 entries are 11.5 a clock and SM at
// the copy rate, the exponentials allow 16, and at about 6 instructions an entry the issue rate 21.
// Measured there: 24 us without alternatives (4.4 TB/s), 35 with k = 20, whose selection all rows
// reach at the same time; 4 x 50265 float32: 4.6 and (k = 5) 8.1 us, where the selection's short
// steps, each run once, are most of the time.
#include <cooperative_groups.h>

#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kMaxK = 64;
constexpr int kStages = 3;          // batches of a thread in flight
constexpr int kCandidates = 1024;
constexpr int kGroups = 128;        // of threads, whose maxima bound the k-th largest entry
constexpr int kMaxCluster = 8;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2eF = 1.4426950408889634f;

__device__ __forceinline__ uint32_t ordered_bits(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// Larger value first, then lower index; -0 counts as 0. Every entry's key is distinct, none is 0
// (a NaN's would be above all others: NaNs get no key).
__device__ __forceinline__ uint64_t make_key(float v, uint32_t idx) {
  return ((uint64_t)ordered_bits(v + 0.f) << 32) | (uint32_t)~idx;
}

// Sums of a piece of a row: s = sum e^d, u = sum d e^d, d = x - m, where m is at most kSlack below
// the largest entry. d is held above kFar: the term of an entry of -inf is 0, and not -inf * 0.
constexpr float kSlack = 8.f, kFar = -1000.f;

// Batches are summed in base 2 with one multiply-add an entry, t = x log2 e - r, r = m log2 e
// rounded; what the rounding shifts all t by, at most 2^-8 for |m| below kRoom, is put right once
// a batch. Entries are held at kLow, so that t stays finite. Batches of rows past kRoom go entry
// by entry.
constexpr float kLow = -1e38f, kRoom = 65536.f;

struct Sums {
  float m, s, u;
  bool nan;  // a NaN among the entries
  __device__ __forceinline__ void reset() {
    m = -INFINITY;
    s = u = 0.f;
    nan = false;
  }
  __device__ __forceinline__ void raise(float m_new) {
    if (m_new > m) {
      if (m != -INFINITY) {
        const float d = fmaxf(m - m_new, kFar);
        const float f = exp2_approx(d * kLog2eF);
        u = fmaf(s, d, u) * f;
        s *= f;
      }
      m = m_new;
    }
  }
  __device__ __forceinline__ void add(float x) {
    nan |= x != x;
    if (x > m + kSlack) raise(x);
    if (x != -INFINITY) {
      const float d = fmaxf(x - m, kFar);
      const float f = exp2_approx(d * kLog2eF);
      s += f;
      u = fmaf(d, f, u);
    }
  }
};

// 16 bytes of a row.
template <typename T>
struct Vec;

template <>
struct Vec<float> {
  static constexpr uint32_t kFill = 0xff800000u;  // -inf
  // the largest entry, or a NaN if there is one
  __device__ __forceinline__ static float max(const uint4& v) {
    float m = __uint_as_float(v.x);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(v.y)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(v.z)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(v.w)));
    return m;
  }
  template <typename F>
  __device__ __forceinline__ static void each(const uint4& v, F&& f) {
    f(__uint_as_float(v.x), 0);
    f(__uint_as_float(v.y), 1);
    f(__uint_as_float(v.z), 2);
    f(__uint_as_float(v.w), 3);
  }
  // entries held at `low`
  __device__ __forceinline__ static uint4 held(const uint4& v, float low) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(v.x), low)), __float_as_uint(fmaxf(__uint_as_float(v.y), low)),
                      __float_as_uint(fmaxf(__uint_as_float(v.z), low)), __float_as_uint(fmaxf(__uint_as_float(v.w), low)));
  }
};

template <>
struct Vec<__nv_bfloat16> {
  static constexpr uint32_t kFill = 0xff80ff80u;
  __device__ __forceinline__ static __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  __device__ __forceinline__ static float max(const uint4& v) {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(two(v.x), two(v.y)), __hmax2_nan(two(v.z), two(v.w)));
    float a = __low2float(m);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(__high2float(m)));
    return a;
  }
  template <typename F>
  __device__ __forceinline__ static void each(const uint4& v, F&& f) {
    f(__uint_as_float(v.x << 16), 0);
    f(__uint_as_float(v.x & 0xffff0000u), 1);
    f(__uint_as_float(v.y << 16), 2);
    f(__uint_as_float(v.y & 0xffff0000u), 3);
    f(__uint_as_float(v.z << 16), 4);
    f(__uint_as_float(v.z & 0xffff0000u), 5);
    f(__uint_as_float(v.w << 16), 6);
    f(__uint_as_float(v.w & 0xffff0000u), 7);
  }
  __device__ __forceinline__ static uint32_t held(uint32_t w, __nv_bfloat162 low) {
    const __nv_bfloat162 x = __hmax2(two(w), low);
    return *reinterpret_cast<const uint32_t*>(&x);
  }
  __device__ __forceinline__ static uint4 held(const uint4& v, float low) {
    const __nv_bfloat162 l = __float2bfloat162_rn(low);
    return make_uint4(held(v.x, l), held(v.y, l), held(v.z, l), held(v.w, l));
  }
};

// The sums of a warp's lanes, against the largest of their maxima, in every lane.
__device__ __forceinline__ void merge_warp(Sums& a) {
  constexpr uint32_t kAll = 0xffffffffu;
  a.nan = __any_sync(kAll, a.nan);
  a.raise(from_ordered(__reduce_max_sync(kAll, ordered_bits(a.m))));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    a.s += __shfl_xor_sync(kAll, a.s, o);
    a.u += __shfl_xor_sync(kAll, a.u, o);
  }
}

struct LogprobParams {
  const void* x;
  int64_t row_stride;
  int64_t vocab;
  const int32_t* targets;
  int k, pieces;
  float* logprobs;
  float* entropy;
  float* values;
  int32_t* indices;
  unsigned int* err;
};

__device__ __forceinline__ float elem(const float* p) { return __ldg(p); }
__device__ __forceinline__ float elem(const __nv_bfloat16* p) {
  return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
}

// What the selection needs, in the place of the ring once the row has passed.
template <int kThreads>
struct Selection {
  static constexpr int kMaxima = (kThreads < 512 ? 16 : 8) * kThreads;
  uint64_t keys[kCandidates];
  uint64_t best[kMaxCluster][kMaxK];  // of the pieces (used in the first CTA)
  uint64_t lane_key[kThreads];
  uint16_t list[kMaxima];
};

template <int kThreads>
struct Shared {
  union {
    uint4 ring[kStages][4][kThreads];  // a thread reads what it copied itself
    Selection<kThreads> sel;
  };
  // of the threads' batches, rounded up to 16 bits; longer pieces fold batches together
  __nv_bfloat16 maxima[Selection<kThreads>::kMaxima];
  uint32_t group_max[kGroups];
  Sums part[kMaxCluster];
  Sums warp[kThreads / 32];
  int listed, found, nan;
  uint64_t bound;
};

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// A value that at least k of the groups' maxima reach, and where ties allow not many more: found by
// halving, in one warp (counting each maximum's rank by a thread of its own is no faster in one CTA
// and 5 us slower with seven on an SM).
__device__ __forceinline__ uint32_t value_bound(const uint32_t* maxima, int k, int lane) {
  uint32_t v[kGroups / 32];
#pragma unroll
  for (int i = 0; i < kGroups / 32; ++i) v[i] = maxima[i * 32 + lane];
  uint32_t lo = v[0], hi = v[0];
#pragma unroll
  for (int i = 1; i < kGroups / 32; ++i) {
    lo = min(lo, v[i]);
    hi = max(hi, v[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);  // every maximum reaches lo
  hi = __reduce_max_sync(0xffffffffu, hi);
  // invariant: at least k reach lo, fewer than k reach hi + 1
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kGroups / 32; ++i) c += __popc(__ballot_sync(0xffffffffu, v[i] >= mid));
    if (c >= k) {
      lo = mid;
      if (c <= k + k / 2 + 4) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// grid: rows x pieces, a cluster a row.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) token_logprobs_kernel(const LogprobParams p) {
  constexpr int N = Elem<T>::kVec;
  constexpr int U = 4;  // vectors of a thread's batch
  constexpr int kWarps = kThreads / 32, kMaxima = Selection<kThreads>::kMaxima;
  using V = Vec<T>;
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<kThreads>& sh = *reinterpret_cast<Shared<kThreads>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / p.pieces;
  const int piece = static_cast<int>(blockIdx.x - r * p.pieces);
  const T* row = static_cast<const T*>(p.x) + r * p.row_stride;
  const int k = p.k;

  // the row's 16-byte vectors: entries [head, head + N * nvec); ragged ends for the first and
  // last piece. A row has fewer than 2^31 entries.
  const int vocab = static_cast<int>(p.vocab);
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int head = min(mis == 0 ? 0 : N - mis, vocab);
  const int nvec = (vocab - head) / N;
  const int per = ceil_div(nvec, p.pieces);
  const int vbegin = min(piece * per, nvec), vend = min(vbegin + per, nvec);
  const T* xv = row + head;

  if (tid == 0) sh.listed = sh.found = sh.nan = 0;
  // the target's entry, in flight while the row passes: at the end the two loads cost 1 to 2 us
  int32_t target = -1;
  float target_x = NAN;
  if (tid == kThreads - 1 && piece == 0 && p.targets != nullptr) {
    target = __ldg(p.targets + r);
    if (target >= 0 && target < vocab) target_x = elem(row + target);
  }
  Sums st;
  st.reset();
  // ragged ends: fewer than 8 entries each
  int edge = -1;
  if (piece == 0 && tid < head) edge = tid;
  if (piece == p.pieces - 1 && tid >= 32 && head + nvec * N + (tid - 32) < vocab) edge = head + nvec * N + (tid - 32);
  float edge_x = -INFINITY;
  if (edge >= 0) {
    edge_x = elem(row + edge);
    st.add(edge_x);
  }
  float lane_max = -INFINITY;
  int lane_at = -1;  // the first batch that holds lane_max

  const int per_batch = kThreads * U;
  const int whole = (vend - vbegin) / per_batch, batches = ceil_div(vend - vbegin, per_batch);
  const int fold = max(1, ceil_div(batches, kMaxima / kThreads));  // batches that share an entry of maxima
  __nv_bfloat16* entry = sh.maxima + tid;
  int entry_left = fold;
  float entry_max = -INFINITY;
  float ref, off, scale;  // of st.m: (x - m) log2 e = t + off
  auto refer = [&]() {
    ref = st.m * kLog2eF;
    off = -fmaf(st.m, kLog2eF, -ref);
    scale = fabsf(st.m) < kRoom ? exp2_approx(off) : 0.f;
  };
  refer();
  // takes batch b, of which this thread has the vectors e[0 .. valid)
  auto take = [&](const uint4 (&e)[U], int b, int valid) {
    float bm = V::max(e[0]);
#pragma unroll
    for (int u = 1; u < U; ++u)
      if (u < valid) asm("max.NaN.f32 %0, %0, %1;" : "+f"(bm) : "f"(V::max(e[u])));
    if (!(bm <= st.m + kSlack)) {  // a new reference, or a NaN
      st.nan |= bm != bm;
      st.raise(bm);
      refer();
    }
    if (scale != 0.f) {
      float s = 0.f, w = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u < valid) {
          V::each(V::held(e[u], kLow), [&](float x, int) {
            const float t = fmaf(x, kLog2eF, -ref);
            const float f = exp2_approx(t);
            s += f;
            w = fmaf(t, f, w);
          });
        }
      }
      w = fmaf(off, s, w) * kLn2;
      st.s = fmaf(s, scale, st.s);
      st.u = fmaf(w, scale, st.u);
    } else if (st.m != -INFINITY) {
#pragma unroll 1
      for (int i = 0; i < valid * N; ++i)
        st.add(elem(xv + (int64_t)(vbegin + b * per_batch + i / N * kThreads + tid) * N + i % N));
    }
    if (k > 0) {
      entry_max = fmaxf(entry_max, bm);
      if (--entry_left == 0) {
        *entry = __float2bfloat16_ru(entry_max);
        entry += kThreads;
        entry_left = fold;
        entry_max = -INFINITY;
      }
      if (bm > lane_max || lane_at < 0) {
        lane_max = bm;
        lane_at = b;
      }
    }
  };
  const T* src = xv + (int64_t)(vbegin + tid) * N;
  const int left = vend - vbegin - whole * per_batch - tid;  // of the last batch, from this thread's first on
  const int last_valid = whole < batches && left > 0 ? ceil_div(left, kThreads) : 0;
  auto fetch = [&](int b, int stage) {  // a group of its own, empty past the end
    if (b < whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) copy16(&sh.ring[stage][u][tid], src + u * kThreads * N);
    } else if (b == whole) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < last_valid) copy16(&sh.ring[stage][u][tid], src + u * kThreads * N);
    }
    src += per_batch * N;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i, i);
#pragma unroll 1
  for (int b0 = 0; b0 < whole; b0 += kStages) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      if (b0 + i < whole) {
        fetch(b0 + i + kStages - 1, (i + kStages - 1) % kStages);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        uint4 e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = sh.ring[i][u][tid];
        take(e, b0 + i, U);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (last_valid > 0) {
    uint4 e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = sh.ring[whole % kStages][u][tid];
    take(e, whole, last_valid);
  }
  if (k > 0 && (entry_left < fold || last_valid == 0) && entry < sh.maxima + kMaxima)
    *entry = __float2bfloat16_ru(entry_max);
  if (k > 0) {
    uint32_t top = ordered_bits(fmaxf(lane_max, edge_x) + 0.f);
#pragma unroll
    for (int o = 1; o < kThreads / kGroups; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    sh.group_max[tid / (kThreads / kGroups)] = top;
  }
  const bool nan_here = st.nan;
  merge_warp(st);
  if (lane == 0) sh.warp[warp] = st;
  if (nan_here) sh.nan = 1;
  __syncthreads();  // the ring is free
  // the pieces' results go to the first CTA once its ring is free too
  if (p.pieces > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  // ---- the k largest of the piece
  if (k > 0) {
    int n = kCandidates + 1;  // a NaN has no place in the order: the slow way
    if (!sh.nan) {
      // first try: the bound by value; second: by (value, index)
      for (int attempt = 0; attempt < 2; ++attempt) {
        if (attempt == 0) {
          if (warp == 0) {
            const uint32_t t = value_bound(sh.group_max, k, lane);
            if (lane == 0) sh.bound = (uint64_t)t << 32;
          }
        } else {
          uint64_t mine = edge >= 0 ? make_key(edge_x, (uint32_t)edge) : 0;  // this thread's best entry
          for (int u = 0; u < U && lane_at >= 0; ++u) {
            const int v = vbegin + lane_at * per_batch + u * kThreads + tid;
            for (int q = 0; q < N && v < vend; ++q) {
              const uint64_t key = make_key(elem(xv + (int64_t)v * N + q), (uint32_t)(head + v * N + q));
              mine = key > mine ? key : mine;
            }
          }
          sh.sel.lane_key[tid] = mine;
          if (tid == 0) sh.listed = sh.found = 0;
          __syncthreads();
          int rank = 0;
          for (int j = 0; j < kThreads; ++j) rank += sh.sel.lane_key[j] > mine || (sh.sel.lane_key[j] == mine && j < tid);
          if (rank == k - 1) sh.bound = mine;
        }
        __syncthreads();
        const uint64_t bound = sh.bound;
        const float thr = from_ordered((uint32_t)(bound >> 32));
        auto collect = [&](float x, int idx) {
          const uint64_t key = make_key(x, (uint32_t)idx);
          if (key >= bound) {
            const int to = atomicAdd(&sh.found, 1);
            if (to < kCandidates) sh.sel.keys[to] = key;
          }
        };
        if (edge >= 0 && edge_x >= thr) collect(edge_x, edge);
        if (lane_max >= thr) {
          constexpr int kMine = kMaxima / kThreads;
          const int mine = ceil_div(batches, fold);
          uint32_t mask = 0;
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (i < mine && __bfloat162float(sh.maxima[i * kThreads + tid]) >= thr) mask |= 1u << i;
          int to = atomicAdd(&sh.listed, __popc(mask));
          for (; mask != 0; mask &= mask - 1) sh.sel.list[to++] = (uint16_t)((__ffs(mask) - 1) * kThreads + tid);
        }
        __syncthreads();
        // a warp reads the U * N entries of a listed batch, eight batches in flight; lanes without
        // an entry read one that is there and drop it, so that no branch parts the loads
        constexpr int kFlight = 8;
        const int visits = sh.listed * fold;
        for (int i0 = warp; i0 < visits; i0 += kWarps * kFlight) {
          float x[kFlight];
          int idx[kFlight];
#pragma unroll
          for (int i = 0; i < kFlight; ++i) {
            const int visit = min(i0 + i * kWarps, visits - 1);
            const int which = fold == 1 ? visit : visit / fold;
            const int slot = sh.sel.list[which];
            const int b = slot / kThreads * fold + (visit - which * fold);
            const int v = vbegin + b * per_batch + (slot % kThreads) + (lane / N) * kThreads;
            const bool there = i0 + i * kWarps < visits && lane < U * N && v < vend;
            const int at = head + (there ? v : vbegin) * N + lane % N;
            x[i] = elem(row + at);
            idx[i] = there ? at : -1;
          }
#pragma unroll
          for (int i = 0; i < kFlight; ++i)
            if (idx[i] >= 0 && x[i] >= thr) collect(x[i], idx[i]);
        }
        __syncthreads();
        n = sh.found;
        if (n <= kCandidates) break;
        __syncthreads();  // every thread has read `found` before it is cleared
      }
    }
    uint64_t* best = sh.sel.best[piece];
    if (n <= kCandidates) {
      for (int i = n + tid; i < k; i += kThreads) best[i] = 0;
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t mine = sh.sel.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.sel.keys[j] > mine;
        if (rank < k) best[rank] = mine;
      }
    } else {
      // more entries reach T than the list holds (a few threads own most of the large ones), or
      // a NaN: the next largest key below the last one, k times over the piece
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        if (tid == 0) sh.bound = 0;
        __syncthreads();
        uint64_t top = 0;
        const int lo = head + vbegin * N, hi = head + vend * N;
        for (int i = lo + tid; i < hi; i += kThreads) {
          const float x = elem(row + i);
          const uint64_t key = x == x ? make_key(x, (uint32_t)i) : 0;
          if (key < last && key > top) top = key;
        }
        if (edge >= 0 && edge_x == edge_x) {
          const uint64_t key = make_key(edge_x, (uint32_t)edge);
          if (key < last && key > top) top = key;
        }
        atomicMax(reinterpret_cast<unsigned long long*>(&sh.bound), (unsigned long long)top);
        __syncthreads();
        last = sh.bound;
        if (tid == 0) best[j] = last;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    Sums all;
    all.reset();
    if (lane < kWarps) all = sh.warp[lane];
    merge_warp(all);
    if (lane == 0) sh.part[piece] = all;
  }

  // ---- the pieces meet in the cluster's first CTA
  if (p.pieces > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncthreads();
    if (piece > 0) {
      Shared<kThreads>* first = cluster.map_shared_rank(&sh, 0);
      if (tid == 0) first->part[piece] = sh.part[piece];
      for (int i = tid; i < k; i += kThreads) first->sel.best[piece][i] = sh.sel.best[piece][i];
    }
    cluster.sync();
    if (piece > 0) return;
    if (warp == 0) {
      Sums all;
      all.reset();
      if (lane < p.pieces) all = sh.part[lane];
      merge_warp(all);
      if (lane == 0) sh.part[0] = all;
    }
  }
  __syncthreads();
  const Sums all = sh.part[0];
  // a row of -inf alone: nothing is possible, every log probability is -inf, entropy 0
  const bool empty = all.m == -INFINITY && !all.nan;
  const float lse = all.nan || all.m == INFINITY ? NAN : (empty ? 0.f : log2f(all.s) * kLn2);
  const float shift = empty ? 0.f : all.m;
  if (tid == kThreads - 1) {
    if (target >= vocab) report(p.err, VFL_DEVERR_SLOT);
    p.logprobs[r] = target >= 0 ? (target_x - shift) - lse : 0.f;
    p.entropy[r] = empty ? 0.f : lse - all.u / all.s;
  }
  if (k == 0) return;
  auto put = [&](uint64_t key, int rank) {
    p.values[r * k + rank] = (from_ordered((uint32_t)(key >> 32)) - shift) - lse;
    p.indices[r * k + rank] = (int32_t)~(uint32_t)key;
  };
  if (p.pieces == 1) {
    if (tid < k && sh.sel.best[0][tid] != 0) put(sh.sel.best[0][tid], tid);
  } else {
    for (int i = tid; i < p.pieces * kMaxK; i += kThreads) {
      const uint64_t mine = i % kMaxK < k ? sh.sel.best[i / kMaxK][i % kMaxK] : 0;
      if (mine == 0) continue;
      int rank = 0;
      for (int c = 0; c < p.pieces; ++c)
#pragma unroll 4
        for (int j = 0; j < k; ++j) rank += sh.sel.best[c][j] > mine;
      if (rank < k) put(mine, rank);
    }
  }
  // entries that are NaN are no alternatives: what is left of the k has none
  if (all.nan) {
    int have = 0;
    for (int c = 0; c < p.pieces; ++c)
      for (int j = 0; j < k; ++j) have += sh.sel.best[c][j] != 0;
    for (int j = have + tid; j < k; j += kThreads) {
      p.values[r * k + j] = NAN;
      p.indices[r * k + j] = -1;
    }
  }
}

// CTAs on a row: enough to give every SM one, pieces of at least 4096 entries.
int choose_pieces(int64_t rows, int64_t vocab) {
  int c = 1;
  while (c < kMaxCluster && rows * c < kNumSMs && vocab / (2 * c) >= 4096) c *= 2;
  return c;
}

template <typename T, int kThreads>
int launch(const LogprobParams& p, int64_t rows, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  auto kern = token_logprobs_kernel<T, kThreads>;
  constexpr int kSmem = sizeof(Shared<kThreads>);
  int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), kSmem, smem_done);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * p.pieces), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.pieces;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.pieces > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "token_logprobs launch");
}

// Few CTAs: 512 threads shorten each one's way through its piece. Many: 128, so that an SM holds
// six or seven rows, whose selections overlap other rows' passes.
template <typename T>
int launch_threads(const LogprobParams& p, int64_t rows, cudaStream_t s) {
  return rows * p.pieces <= 2 * kNumSMs ? launch<T, 512>(p, rows, s) : launch<T, 128>(p, rows, s);
}

}  // namespace
}  // namespace vfl

using namespace vfl;

extern "C" int vfl_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                  const int32_t* targets, int32_t k, float* logprobs, float* entropy, float* values,
                                  int32_t* indices, void* stream) {
  if (!dtype_ok(dtype)) return fail(VFL_ERR_UNSUPPORTED, "token_logprobs: dtype %d", dtype);
  if (rows < 0 || vocab <= 0 || row_stride < vocab)
    return fail(VFL_ERR_INVALID_ARGUMENT, "token_logprobs: rows %lld, vocab %lld, row_stride %lld", (long long)rows,
                (long long)vocab, (long long)row_stride);
  if (k < 0 || k > kMaxK || k > vocab)
    return fail(VFL_ERR_INVALID_ARGUMENT, "token_logprobs: k %d outside [0, min(%d, vocab)]", k, kMaxK);
  if (rows == 0) return VFL_OK;
  if (vocab > INT32_MAX - (1 << 20) || rows > INT32_MAX / kMaxCluster)
    return fail(VFL_ERR_UNSUPPORTED, "token_logprobs: %lld x %lld scores", (long long)rows, (long long)vocab);
  if (!logits || !logprobs || !entropy || (k > 0 && (!values || !indices)))
    return fail(VFL_ERR_INVALID_ARGUMENT, "token_logprobs: NULL pointer");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) != 0)
    return fail(VFL_ERR_INVALID_ARGUMENT, "token_logprobs: logits not aligned to their elements");
  LogprobParams p;
  int st = device_error_word(&p.err);
  if (st) return st;
  p.x = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.targets = targets;
  p.k = k;
  p.pieces = choose_pieces(rows, vocab);
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.values = values;
  p.indices = indices;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == VFL_DTYPE_F32 ? launch_threads<float>(p, rows, s) : launch_threads<__nv_bfloat16>(p, rows, s);
}
