// Log probabilities of given columns of rows of logits, with each row's
// entropy and its most probable columns, and the gradient.
//
//   z_j = scale·x_j, m = max_j z_j, s1 = Σ e^(z_j − m), s2 = Σ e^(z_j − m)·(z_j − m)
//   logprob = z_t − m − log s1,  H = log s1 − s2 / s1,  lse = m + log s1
//   dx_j = scale·(g·([j = t] − p_j) − h·p_j·(log p_j + H)),  p_j = e^(z_j − lse)
//
// A row whose entries are all −∞ has log probabilities −∞, entropy 0 and
// gradient 0; a row with a NaN or a +∞ has NaN in all of them.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fg_internal.h"
#include "fg_ptx.cuh"
#include "fg_types.cuh"

namespace fg {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = FG_MAX_TOP;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Order of the alternatives as one number: the value (NaN above +∞, −0 as
// 0) in the upper half, the lower index above the higher one in the lower.
// 0 is below every entry.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  if (x != x) u = 0x7fc00000u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return uint64_t(rank_bits(x)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float rank_value(uint32_t bits) {
  return __uint_as_float((bits & 0x80000000u) ? bits & 0x7fffffffu : ~bits);
}
__device__ __forceinline__ uint32_t rank_index(uint64_t key) { return 0xffffffffu - uint32_t(key); }

// The larger of two numbers, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct LogProbsArgs {
  int64_t rows, ld;
  int width, top;
  const int32_t* targets;
  float scale;
  float* logprob;
  float* entropy;
  float* lse;
  int32_t* top_index;
  float* top_logprob;
  int* err;
};

// The sums of a part of a row about a reference, its largest entry:
// s1 = Σ e^(scale·(x − ref)), s2 = Σ e^(scale·(x − ref))·(x − ref). While
// s1 is 0, nothing above −∞ has been met and the reference says nothing.
struct RowSums {
  float ref, s1, s2;

  // the same sums about another reference; k = scale·log2 e
  __device__ __forceinline__ void move(float to, float k) {
    const float d = ref - to;
    ref = to;
    const float c = s1 == 0.f ? 0.f : ex2_approx(d * k);
    s2 = c == 0.f ? 0.f : c * fmaf(d, s1, s2);
    s1 = c == 0.f ? 0.f : c * s1;
  }
};

// One pass over each row by the blocks of a cluster (one block where there
// are rows enough for the SMs): tiles of kItems entries a thread, the next
// tile's loads under way while this one is summed, each thread's sums about
// its own running maximum (moved only when a tile has a larger one). The
// first block joins the parts through distributed shared memory.
//
// The alternatives: a block lists the entries that may be among its first
// `top`, and knows a bound that `top` of them reach, so that a tile without
// an entry above it costs a comparison and a barrier. The first bound comes
// from the first tile: of every warp the r-th largest of its lanes' maxima,
// r = ⌈top / warps⌉, and of these the least. Later ones are the `top`-th
// entry whenever the list is ranked (an entry's rank is the number of
// entries above it). A tile of which more would enter than the list holds
// (long runs of equal or rising values) gives its best `top` one at a time.
constexpr int kItems = 16;
constexpr int kListSize = 512;  // entries that may wait besides the first `top`
constexpr int kMaxSplit = 16;   // blocks of a cluster

template <int THREADS>
struct RowShared {
  uint64_t list[kListSize + kMaxTop];
  uint64_t best[kMaxTop];
  uint64_t warp_key[THREADS / 32];
  RowSums warp_sums[THREADS / 32];
  RowSums sums;
  uint32_t warp_bound[THREADS / 32];
  int count;  // entries of the list
};

// Ranks the n entries of the list; the first `top` stay, in order. Returns
// how many there are. All threads of the block.
template <int THREADS>
__device__ __forceinline__ int rank_list(RowShared<THREADS>& sh, int n, int top) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t mine = sh.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.list[j] > mine;
    if (rank < top) sh.best[rank] = mine;  // entries are distinct, so ranks are
  }
  __syncthreads();
  n = min(n, top);
  for (int i = threadIdx.x; i < n; i += THREADS) sh.list[i] = sh.best[i];
  if (threadIdx.x == 0) sh.count = n;
  __syncthreads();
  return n;
}

// sum += x, keeping in `lost` what the sum's rounding put in too much
// (Kahan's summation): a long row's many small terms count beside a large one.
__device__ __forceinline__ void add_kept(float& sum, float& lost, float x) {
  const float y = __fsub_rn(x, lost);
  const float to = __fadd_rn(sum, y);
  lost = __fsub_rn(__fsub_rn(to, sum), y);
  sum = to;
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kFull));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// The sums of all lanes together, in every lane. A lane that has met nothing
// above −∞ has the reference −∞ and sums of 0.
__device__ __forceinline__ RowSums warp_join(RowSums v, float k) {
  v.move(warp_max_nan(v.ref), k);
  v.s1 = warp_sum(v.s1);
  v.s2 = warp_sum(v.s2);
  return v;
}

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t key) {
  const uint32_t hi = __reduce_max_sync(kFull, uint32_t(key >> 32));
  const uint32_t lo = __reduce_max_sync(kFull, uint32_t(key >> 32) == hi ? uint32_t(key) : 0u);
  return uint64_t(hi) << 32 | lo;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    logprobs_kernel(LogProbsArgs a, int split, const T* __restrict__ logits) {
  constexpr int V = 16 / int(sizeof(T));  // entries of a 16-byte group
  constexpr int G = kItems / V;           // a thread's groups of a tile
  constexpr int kWarps = THREADS / 32;
  __shared__ RowShared<THREADS> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const T* x = logits + row * a.ld;
  // groups are those of memory: the first may begin before the row
  const int skip = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int tiles = int((int64_t(a.width) + skip + THREADS * kItems - 1) / (THREADS * kItems));
  const float k = a.scale * kLog2e;
  // column of a thread's entry i of a tile
  auto column = [&](int tile, int i) {
    return (tile * (THREADS * G) + (i / V) * THREADS + int(threadIdx.x)) * V - skip + i % V;
  };

  Pack<T, V> next[G];
  auto load = [&](int tile) {
    const int first = tile * (THREADS * kItems) - skip;
    if (first >= 0 && first + THREADS * kItems <= a.width) {
#pragma unroll
      for (int g = 0; g < G; ++g) next[g].load(x + column(tile, g * V));
      return;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int j = column(tile, g * V);
      if (j >= 0 && j + V <= a.width) {
        next[g].load(x + j);
      } else {  // a row's first or last group, or none of it
#pragma unroll
        for (int i = 0; i < V; ++i) next[g].v[i] = j + i >= 0 && j + i < a.width ? x[j + i] : narrow<T>(-INFINITY);
      }
    }
  };

  const int t = part == 0 && threadIdx.x == 0 ? a.targets[row] : -1;
  float xt = 0.f;
  if (t >= 0) {
    if (t < a.width)
      xt = widen(x[t]);
    else
      atomicCAS(a.err, 0, kDevBadIndex);
  }
  if (threadIdx.x == 0) sh.count = 0;
  RowSums sums{-INFINITY, 0.f, 0.f};
  float lost1 = 0.f, lost2 = 0.f;  // what rounding added to the sums too much
  int n = 0;                // entries of the list
  uint64_t bound = 0;       // `top` entries met reach this key
  float bound_value = NAN;  // and this value; NaN: no bound yet
  if (part < tiles) load(part);
  __syncthreads();
  for (int tile = part; tile < tiles; tile += split) {
    float v[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) v[i] = next[i / V].get(i % V);
    if (tile + split < tiles) load(tile + split);
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kItems; ++i) most = max_nan(most, v[i]);
    const float higher = max_nan(sums.ref, most);
    if (!(higher == sums.ref)) {
      sums.s1 -= lost1;
      sums.s2 -= lost2;
      lost1 = lost2 = 0.f;
      sums.move(higher, k);
    }
    const float ref = sums.ref == -INFINITY ? 0.f : sums.ref;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const float d = max_nan(v[i] - ref, -FLT_MAX);  // −∞ times e^−∞ = 0 would be no number
      const float e = ex2_approx(d * k);
      s1 += e;
      s2 = fmaf(e, d, s2);
    }
    add_kept(sums.s1, lost1, s1);
    add_kept(sums.s2, lost2, s2);
    if (a.top == 0) continue;

    if (tile == part) {
      const int r = (a.top + kWarps - 1) / kWarps;
      // lanes without an entry of the row come last
      uint32_t mine = column(tile, V - 1) >= 0 && column(tile, 0) < a.width ? rank_bits(most) : 0u, least = 0;
      if (r <= 32) {
        for (int i = 0; i < r; ++i) {
          least = __reduce_max_sync(kFull, mine);
          if (lane == __ffs(__ballot_sync(kFull, mine == least)) - 1) mine = 0;
        }
      }
      if (lane == 0) sh.warp_bound[warp] = least;
      __syncthreads();
      least = __reduce_min_sync(kFull, sh.warp_bound[lane < kWarps ? lane : 0]);
      bound = uint64_t(least) << 32;
      if (least) bound_value = rank_value(least);
    }
    auto key_of = [&](int i) {
      const int j = column(tile, i);
      const uint64_t key = j >= 0 && j < a.width ? rank_key(v[i], uint32_t(j)) : 0;
      return key > bound ? key : 0;
    };
    bool entered = false;
    if (!(most < bound_value)) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (v[i] < bound_value) continue;
        const uint64_t key = key_of(i);
        if (key) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kListSize + kMaxTop) sh.list[at] = key;
          entered = true;
        }
      }
    }
    if (!__syncthreads_or(entered)) continue;
    const int before = n;
    n = sh.count;
    __syncthreads();
    const bool over = n > kListSize + kMaxTop;
    if (over) {
      n = before;
      uint64_t mine = 0;
#pragma unroll
      for (int i = 0; i < kItems; ++i) mine = larger(mine, key_of(i));
      for (int r = 0; r < a.top; ++r) {
        const uint64_t w = warp_max_key(mine);
        if (lane == 0) sh.warp_key[warp] = w;
        __syncthreads();
        const uint64_t first = warp_max_key(sh.warp_key[lane < kWarps ? lane : 0]);
        if (first == 0) break;
        if (mine == first) {
          sh.list[n] = first;
          mine = 0;
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const uint64_t key = key_of(i);
            if (key < first) mine = larger(mine, key);
          }
        }
        ++n;
        __syncthreads();
      }
    }
    if (over || n > kListSize || (tile + split < tiles && n >= a.top + kListSize / 8)) {
      n = rank_list(sh, n, a.top);
      if (n == a.top) {
        bound = sh.list[n - 1];
        bound_value = rank_value(uint32_t(bound >> 32));
      }
    }
  }

  const RowSums none{-INFINITY, 0.f, 0.f};
  sums.s1 -= lost1;
  sums.s2 -= lost2;
  sums = warp_join(sums, k);
  if (kWarps > 1) {
    if (lane == 0) sh.warp_sums[warp] = sums;
    __syncthreads();
    sums = warp_join(lane < kWarps ? sh.warp_sums[lane % kWarps] : none, k);
  }
  if (a.top) n = rank_list(sh, n, a.top);
  if (split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) sh.sums = sums;
    cluster.sync();
    if (part == 0) {
      sums = warp_join(lane < split ? cluster.map_shared_rank(&sh, lane % split)->sums : none, k);
      // as many parts' lists at a time as the list has room for
      const int batch = a.top ? kListSize / a.top : split;
      for (int p0 = 1; a.top && p0 < split; p0 += batch) {
        const int parts = min(batch, split - p0);
        for (int i = threadIdx.x; i < parts * a.top; i += THREADS) {
          const RowShared<THREADS>* other = cluster.map_shared_rank(&sh, p0 + i / a.top);
          if (i % a.top < other->count) sh.list[atomicAdd(&sh.count, 1)] = other->list[i % a.top];
        }
        __syncthreads();
        n = sh.count;
        n = rank_list(sh, n, a.top);
      }
    }
    cluster.sync();  // the parts' shared memory is read until here
    if (part) return;
  }
  const bool empty = sums.s1 == 0.f;
  const float ref = empty ? 0.f : sums.ref, logs = logf(sums.s1);
  if (threadIdx.x == 0) {
    const bool skipped = t < 0 || t >= a.width;
    a.logprob[row] = skipped ? 0.f : empty ? -INFINITY : fmaf(xt - ref, a.scale, -logs);
    a.entropy[row] = empty ? 0.f : logs - a.scale * (sums.s2 / sums.s1);
    a.lse[row] = fmaf(ref, a.scale, logs);
  }
  for (int i = threadIdx.x; i < a.top; i += THREADS) {
    const uint64_t key = sh.list[i];
    a.top_index[row * a.top + i] = int32_t(rank_index(key));
    a.top_logprob[row * a.top + i] = empty ? -INFINITY : fmaf(rank_value(uint32_t(key >> 32)) - ref, a.scale, -logs);
  }
}

template <typename T, int THREADS>
int launch_logprobs(const LogProbsArgs& a, const T* logits, cudaStream_t s) {
  // blocks of a row: as many as fill the SMs (1024 threads each), at most one a tile
  const int tiles = int((int64_t(a.width) + THREADS * kItems - 1) / (THREADS * kItems));
  const int64_t room = int64_t(sm_count()) * (1024 / THREADS);
  int split = 1;
  while (split * 2 <= std::min(kMaxSplit, tiles) && a.rows * split * 2 <= room) split *= 2;
  auto kernel = logprobs_kernel<T, THREADS>;
  if (split == 1) {
    kernel<<<unsigned(a.rows), THREADS, 0, s>>>(a, 1, logits);
    FG_CUDA_TRY(cudaGetLastError());
    return FG_OK;
  }
  if (split > 8) FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.rows * split));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, split, logits));
  return FG_OK;
}

struct LogProbsGradArgs {
  int64_t rows, ld, ldd;
  int width;
  const int32_t* targets;
  float scale;
  const float* lse;
  const float* entropy;
  const float* dlogprob;
  const float* dentropy;
  int* err;
};

// Elementwise: a block takes kGradGroups 16-byte groups a thread of one row,
// all loaded before the first is used; groups are those of the logits'
// memory, stored whole where the gradient's lie alike.
constexpr int kGradThreads = 256;
constexpr int kGradGroups = 4;

template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kGradThreads) logprobs_grad_kernel(LogProbsGradArgs a, int parts, const T* logits,
                                                                    T* dlogits) {
  constexpr int V = 16 / int(sizeof(T));
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* x = logits + row * a.ld;
  T* dx = dlogits + row * a.ldd;
  const int skip = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const int64_t j0 = (int64_t(part) * (kGradThreads * kGradGroups) + threadIdx.x) * V - skip;
  Pack<T, V> in[kGradGroups];
#pragma unroll
  for (int g = 0; g < kGradGroups; ++g) {
    const int64_t j = j0 + g * kGradThreads * V;
    if (j >= 0 && j + V <= a.width) {
      in[g].load_own(x + j);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) in[g].v[i] = j + i >= 0 && j + i < a.width ? x[j + i] : narrow<T>(0.f);
    }
  }
  const int t = a.targets[row];
  if (t >= a.width && part == 0 && threadIdx.x == 0) atomicCAS(a.err, 0, kDevBadIndex);
  const bool none = t < 0 || t >= a.width;
  const float lse = a.lse[row];
  const float g0 = none ? 0.f : a.dlogprob[row];
  const bool empty = lse == -INFINITY;
  float h = 0.f, H = 0.f;
  if (ENTROPY) {
    h = a.dentropy[row];
    H = a.entropy[row];
  }
#pragma unroll
  for (int g = 0; g < kGradGroups; ++g) {
    const int64_t j = j0 + g * kGradThreads * V;
    if (j >= a.width) break;
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float lp = fmaf(in[g].get(i), a.scale, -lse);
      const float p = ex2_approx(lp * kLog2e);
      float d = g0 * ((j + i == t ? 1.f : 0.f) - p);
      if (ENTROPY && p != 0.f) d = fmaf(-h * p, lp + H, d);
      out.set(i, empty ? 0.f : d * a.scale);
    }
    if (alike && j >= 0 && j + V <= a.width) {
      out.store(dx + j);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (j + i >= 0 && j + i < a.width) dx[j + i] = out.v[i];
    }
  }
}

template <typename T>
int launch_logprobs_grad(const LogProbsGradArgs& a, const T* logits, T* dlogits, cudaStream_t s) {
  constexpr int V = 16 / int(sizeof(T)), kPart = kGradThreads * kGradGroups * V;
  const int64_t parts = (int64_t(a.width) + V - 1 + kPart - 1) / kPart;
  // rows that one launch's grid holds; more only past 2^31 blocks
  const int64_t most = INT32_MAX / parts;
  for (int64_t r = 0; r < a.rows; r += most) {
    LogProbsGradArgs b = a;
    b.rows = std::min(most, a.rows - r);
    b.targets += r;
    b.lse += r;
    b.dlogprob += r;
    const unsigned blocks = unsigned(b.rows * parts);
    if (a.dentropy) {
      b.dentropy += r;
      b.entropy += r;
      logprobs_grad_kernel<T, true><<<blocks, kGradThreads, 0, s>>>(b, int(parts), logits + r * a.ld, dlogits + r * a.ldd);
    } else {
      logprobs_grad_kernel<T, false><<<blocks, kGradThreads, 0, s>>>(b, int(parts), logits + r * a.ld, dlogits + r * a.ldd);
    }
    FG_CUDA_TRY(cudaGetLastError());
  }
  return FG_OK;
}

}  // namespace

}  // namespace fg

using namespace fg;

extern "C" {

int fg_log_probs(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                 float scale, int top, float* logprob, float* entropy, float* lse, int32_t* top_index,
                 float* top_logprob, void* stream) {
  clear_error();
  if (rows < 0 || width <= 0 || rows >= INT32_MAX || width > (1 << 30))
    return set_error(FG_EINVAL, "fg_log_probs: bad shape [%lld x %lld]", (long long)rows, (long long)width);
  if (!known_dtype(dtype)) return set_error(FG_EINVAL, "fg_log_probs: unknown element type %d", dtype);
  if (ld < width) return set_error(FG_EINVAL, "fg_log_probs: leading dimension smaller than the row");
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(FG_EINVAL, "fg_log_probs: scale must be positive and finite");
  if (top < 0 || top > kMaxTop || top > width)
    return set_error(FG_EINVAL, "fg_log_probs: %d alternatives of %lld columns (at most %d)", top, (long long)width, kMaxTop);
  if (rows == 0) return FG_OK;
  if (!logits || !targets || !logprob || !entropy || !lse || (top > 0 && (!top_index || !top_logprob)))
    return set_error(FG_EINVAL, "fg_log_probs: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LogProbsArgs a{rows, ld, int(width), top, targets, scale, logprob, entropy, lse, top_index, top_logprob, nullptr};
  FG_TRY(device_error_word(&a.err));
  return by_dtype(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    const T* x = static_cast<const T*>(logits);
    // Threads of a block: with rows enough to fill the SMs a warp alone takes
    // a row, without a barrier; fewer rows or a wide one get more.
    const int64_t fill = int64_t(sm_count()) * 1024;
    if (width <= 1024 || rows * 32 >= fill) return launch_logprobs<T, 32>(a, x, s);
    if (width <= 4096 || rows * 128 >= fill) return launch_logprobs<T, 128>(a, x, s);
    return launch_logprobs<T, 512>(a, x, s);
  });
}

int fg_log_probs_grad(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                      float scale, const float* lse, const float* entropy, const float* dlogprob,
                      const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  clear_error();
  if (rows < 0 || width <= 0 || rows >= INT32_MAX || width >= INT32_MAX)
    return set_error(FG_EINVAL, "fg_log_probs_grad: bad shape [%lld x %lld]", (long long)rows, (long long)width);
  if (!known_dtype(dtype)) return set_error(FG_EINVAL, "fg_log_probs_grad: unknown element type %d", dtype);
  if (ld < width || ldd < width) return set_error(FG_EINVAL, "fg_log_probs_grad: leading dimension smaller than the row");
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(FG_EINVAL, "fg_log_probs_grad: scale must be positive and finite");
  if (rows == 0) return FG_OK;
  if (!logits || !targets || !lse || !dlogprob || !dlogits || (dentropy && !entropy))
    return set_error(FG_EINVAL, "fg_log_probs_grad: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LogProbsGradArgs a{rows, ld, ldd, int(width), targets, scale, lse, entropy, dlogprob, dentropy, nullptr};
  FG_TRY(device_error_word(&a.err));
  return by_dtype(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    return launch_logprobs_grad(a, static_cast<const T*>(logits), static_cast<T*>(dlogits), s);
  });
}

}  // extern "C"
