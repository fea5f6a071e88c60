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
// One pass gives the sums and, in shared memory, the largest value of each lane's batch of 32
// entries. The k-th largest of the threads' own maxima is a lower bound T of the k-th largest
// entry (the maxima are distinct entries), so only batches whose maximum reaches T are read
// again: about k of them, from L2. Their entries >= T are ranked by counting. Where ties at T
// overflow the list (rows of mostly one value), T becomes the k-th best (value, index) pair and
// the collection runs again. A row is cut over a cluster of up to 8 CTAs when there are few rows; the pieces meet in the first CTA's shared
// memory.
#include <cooperative_groups.h>

#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace vfl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxK = 64;
constexpr int kMaxima = 2048;       // batch maxima kept per CTA; longer pieces fold batches together
constexpr int kCandidates = 1024;
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

constexpr float kLowest = -150.f;  // e^-150 is 0 in float32, and so is its product with -150

// Sums of a piece of a row against its maximum: s = sum e^(x - m), u = sum (x - m) e^(x - m).
struct Sums {
  float m = -INFINITY, s = 0.f, u = 0.f;
  bool nan = false;  // a NaN among the entries
  __device__ __forceinline__ void raise(float m_new) {
    if (m_new > m) {
      if (m != -INFINITY) {
        const float d = fmaxf(m - m_new, kLowest);
        const float f = exp2_approx(d * kLog2eF);
        u = fmaf(s, d, u) * f;
        s *= f;
      }
      m = m_new;
    }
  }
  __device__ __forceinline__ void merge(Sums o) {
    nan |= o.nan;
    const float top = fmaxf(m, o.m);
    raise(top);
    o.raise(top);
    s += o.s;
    u += o.u;
  }
};

__device__ __forceinline__ Sums shfl_xor(const Sums& a, int mask) {
  Sums o;
  o.m = __shfl_xor_sync(0xffffffffu, a.m, mask);
  o.s = __shfl_xor_sync(0xffffffffu, a.s, mask);
  o.u = __shfl_xor_sync(0xffffffffu, a.u, mask);
  o.nan = __shfl_xor_sync(0xffffffffu, (int)a.nan, mask) != 0;
  return o;
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

struct Shared {
  uint64_t keys[kCandidates];
  uint64_t best[kMaxCluster][kMaxK];  // of the pieces (used in the first CTA)
  Sums part[kMaxCluster];
  float maxima[kMaxima];
  uint64_t lane_key[kThreads];
  int list[kMaxima];
  Sums warp[kWarps];
  int listed, found;
  uint64_t bound;
};

// grid: rows x pieces, a cluster a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const LogprobParams p) {
  constexpr int N = Elem<T>::kVec;
  constexpr int U = 32 / N;  // vectors of a lane's batch
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / p.pieces;
  const int piece = static_cast<int>(blockIdx.x - r * p.pieces);
  const T* row = static_cast<const T*>(p.x) + r * p.row_stride;
  const int k = p.k;

  // the row's 16-byte vectors: entries [head, head + N * nvec); ragged ends for the first and
  // last piece
  const int64_t mis = (reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T);
  const int64_t head = min(mis == 0 ? (int64_t)0 : N - mis, p.vocab);
  const int64_t nvec = (p.vocab - head) / N;
  const int64_t per = ceil_div(nvec, (int64_t)p.pieces);
  const int64_t vbegin = min(piece * per, nvec), vend = min(vbegin + per, nvec);
  const T* xv = row + head;

  // ---- pass 1
  const int64_t batches = ceil_div(vend - vbegin, (int64_t)(kThreads * U));  // of every lane
  const int fold = static_cast<int>(ceil_div(batches, (int64_t)(kMaxima / kThreads)));  // batches an entry covers
  for (int i = tid; i < kMaxima; i += kThreads) sh.maxima[i] = -INFINITY;
  if (tid == 0) sh.listed = sh.found = 0;
  __syncthreads();
  // a CTA's shared memory may be written to once that CTA runs
  if (p.pieces > 1) cg::this_cluster().sync();
  Sums st;
  float lane_max = -INFINITY;
  int64_t lane_at = -1;  // the first batch that holds lane_max
  for (int64_t b = 0; b < batches; ++b) {
    float e[U][N];
    float bm = -INFINITY;
    const int64_t v0 = vbegin + b * (kThreads * U) + tid;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * kThreads;
      if (v < vend) {
        unpack16(ldg_nc_v4(xv + v * N), e[u], T());
      } else {
#pragma unroll
        for (int q = 0; q < N; ++q) e[u][q] = -INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < N; ++q) {
        bm = fmaxf(bm, e[u][q]);
        st.nan |= e[u][q] != e[u][q];
      }
    st.raise(bm);
    if (st.m != -INFINITY) {
      const float m = st.m;
      float s = 0.f, w = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < N; ++q) {
          const float d = fmaxf(e[u][q] - m, kLowest);  // NaN (inf - inf) too: such rows score NaN
          const float f = exp2_approx(d * kLog2eF);
          s += f;
          w = fmaf(d, f, w);
        }
      st.s += s;
      st.u += w;
    }
    if (k > 0) {
      float& slot = sh.maxima[(fold == 1 ? (int)b : (int)(b / fold)) * kThreads + tid];
      slot = fmaxf(slot, bm);
      if (bm > lane_max || lane_at < 0) {
        lane_max = bm;
        lane_at = b;
      }
    }
  }
  // ragged ends: fewer than 8 entries each
  int64_t edge = -1;
  if (piece == 0 && tid < head) edge = tid;
  if (piece == p.pieces - 1 && tid >= 32 && head + nvec * N + (tid - 32) < p.vocab) edge = head + nvec * N + (tid - 32);
  float edge_x = -INFINITY;
  if (edge >= 0) {
    edge_x = elem(row + edge);
    st.nan |= edge_x != edge_x;
    st.raise(edge_x);
    if (st.m != -INFINITY) {
      const float d = fmaxf(edge_x - st.m, kLowest);
      const float f = exp2_approx(d * kLog2eF);
      st.s += f;
      st.u = fmaf(d, f, st.u);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) st.merge(shfl_xor(st, o));
  if (lane == 0) sh.warp[warp] = st;

  // ---- pass 2: the k largest of the piece
  int n = 0;
  if (k > 0) {
    const int entries = static_cast<int>(ceil_div(batches, (int64_t)fold)) * kThreads;
    // first try: T by value; second: by (value, index)
    for (int attempt = 0; attempt < 2; ++attempt) {
      uint64_t mine = make_key(fmaxf(lane_max, edge_x), tid);
      if (attempt == 1) {  // the best entry of this thread's, with its index
        mine = 0;
        if (edge >= 0 && edge_x == edge_x) mine = make_key(edge_x, (uint32_t)edge);
        if (lane_at >= 0) {
          for (int u = 0; u < U; ++u) {
            const int64_t v = vbegin + lane_at * (kThreads * U) + tid + u * kThreads;
            for (int q = 0; q < N && v < vend; ++q) {
              const int64_t idx = head + v * N + q;
              const float x = elem(row + idx);
              const uint64_t key = x == x ? make_key(x, (uint32_t)idx) : 0;
              mine = key > mine ? key : mine;
            }
          }
        }
        if (tid == 0) sh.listed = sh.found = 0;
      }
      sh.lane_key[tid] = mine;
      __syncthreads();
      int rank = 0;
      for (int j = 0; j < kThreads; ++j) rank += sh.lane_key[j] > mine || (sh.lane_key[j] == mine && j < tid);
      // value alone: any index counts
      if (rank == k - 1) sh.bound = attempt == 0 ? mine & 0xffffffff00000000ull : mine;
      __syncthreads();
      const uint64_t bound = sh.bound;
      const float thr = from_ordered((uint32_t)(bound >> 32));
      for (int i = tid; i < entries; i += kThreads)
        if (bound == 0 || sh.maxima[i] >= thr) sh.list[atomicAdd(&sh.listed, 1)] = i;
      auto collect = [&](float x, int64_t idx) {
        if (x == x && make_key(x, (uint32_t)idx) >= bound) {
          const int at = atomicAdd(&sh.found, 1);
          if (at < kCandidates) sh.keys[at] = make_key(x, (uint32_t)idx);
        }
      };
      if (edge >= 0) collect(edge_x, edge);
      __syncthreads();
      // a warp reads the 32 entries of a listed batch, one a lane
      for (int i = warp; i < sh.listed; i += kWarps) {
        const int entry = sh.list[i];
        const int64_t b0 = (int64_t)(entry / kThreads) * fold;
        for (int64_t b = b0; b < min(b0 + fold, batches); ++b) {
          const int64_t v = vbegin + b * (kThreads * U) + (entry % kThreads) + (lane / N) * kThreads;
          if (v < vend) collect(elem(row + head + v * N + lane % N), head + v * N + lane % N);
        }
      }
      __syncthreads();
      n = sh.found;
      if (n <= kCandidates) break;
      __syncthreads();  // every thread has read `found` before it is cleared
    }
    uint64_t* best = sh.best[piece];
    if (n <= kCandidates) {
      for (int i = tid; i < kMaxK; i += kThreads) best[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t mine = sh.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.keys[j] > mine;
        if (rank < k) best[rank] = mine;
      }
    } else {
      // more entries reach T than the list holds (a few threads own most of the large ones, or
      // long ties): the next largest key below the last one, k times over the piece
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        if (tid == 0) sh.bound = 0;
        __syncthreads();
        uint64_t top = 0;
        const int64_t lo = head + vbegin * N, hi = head + vend * N;
        for (int64_t i = lo + tid; i < hi; i += kThreads) {
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
  if (tid == 0) {
    Sums all = sh.warp[0];
    for (int w = 1; w < kWarps; ++w) all.merge(sh.warp[w]);
    sh.part[piece] = all;
  }

  // ---- the pieces meet in the cluster's first CTA
  if (p.pieces > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    __syncthreads();
    if (piece > 0) {
      Shared* first = cluster.map_shared_rank(&sh, 0);
      if (tid == 0) first->part[piece] = sh.part[piece];
      for (int i = tid; i < k; i += kThreads) first->best[piece][i] = sh.best[piece][i];
    }
    cluster.sync();
    if (piece > 0) return;
    if (tid == 0) {
      Sums all = sh.part[0];
      for (int c = 1; c < p.pieces; ++c) all.merge(sh.part[c]);
      sh.part[0] = all;
    }
  }
  __syncthreads();
  const Sums all = sh.part[0];
  // a row of -inf alone: nothing is possible, every log probability is -inf, entropy 0
  const bool empty = all.m == -INFINITY && !all.nan;
  const float lse = all.nan || all.m == INFINITY ? NAN : (empty ? 0.f : log2f(all.s) * kLn2);
  const float shift = empty ? 0.f : all.m;
  if (tid == 0) {
    const int32_t t = p.targets == nullptr ? -1 : __ldg(p.targets + r);
    float lp = 0.f;
    if (t >= 0) {
      if (t < p.vocab) {
        lp = (elem(row + t) - shift) - lse;
      } else {
        report(p.err, VFL_DEVERR_SLOT);
        lp = NAN;
      }
    }
    p.logprobs[r] = lp;
    p.entropy[r] = empty ? 0.f : lse - all.u / all.s;
  }
  const int total = p.pieces * kMaxK;
  for (int i = tid; i < (k > 0 ? total : 0); i += kThreads) {
    const uint64_t mine = sh.best[i / kMaxK][i % kMaxK];
    if (i % kMaxK >= k) continue;
    int rank = 0;
    if (mine != 0) {
      for (int c = 0; c < p.pieces; ++c)
        for (int j = 0; j < k; ++j) rank += sh.best[c][j] > mine;
    }
    if (mine != 0 && rank < k) {
      p.values[r * k + rank] = (from_ordered((uint32_t)(mine >> 32)) - shift) - lse;
      p.indices[r * k + rank] = (int32_t)~(uint32_t)mine;
    }
  }
  // entries that are NaN are no alternatives: what is left of the k has none
  if (k > 0 && all.nan) {
    int have = 0;
    for (int c = 0; c < p.pieces; ++c)
      for (int j = 0; j < k; ++j) have += sh.best[c][j] != 0;
    for (int j = have + tid; j < k; j += kThreads) {
      p.values[r * k + j] = NAN;
      p.indices[r * k + j] = -1;
    }
  }
}

// CTAs on a row: enough to give every SM one, pieces of at least 8192 entries.
int choose_pieces(int64_t rows, int64_t vocab) {
  int c = 1;
  while (c < kMaxCluster && rows * c < kNumSMs && vocab / (2 * c) >= 4096) c *= 2;
  return c;
}

template <typename T>
int launch(const LogprobParams& p, int64_t rows, cudaStream_t stream) {
  static int smem_done[kMaxDevices] = {};
  auto kern = token_logprobs_kernel<T>;
  int st = ensure_smem_attribute(reinterpret_cast<const void*>(kern), sizeof(Shared), smem_done);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * p.pieces), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.pieces;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "token_logprobs launch");
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
  if (vocab > INT32_MAX || rows > INT32_MAX / kMaxCluster)
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
  return dtype == VFL_DTYPE_F32 ? launch<float>(p, rows, s) : launch<__nv_bfloat16>(p, rows, s);
}
