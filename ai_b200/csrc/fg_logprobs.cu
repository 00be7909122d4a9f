// Log probabilities of given columns of rows of logits, with each row's
// entropy and its most probable columns, and the gradient.
//
//   z_j = scale·x_j, m = max_j z_j, s1 = Σ e^(z_j − m), s2 = Σ e^(z_j − m)·(z_j − m)
//   logprob = z_t − m − log s1,  H = log s1 − s2 / s1,  lse = m + log s1
//   dx_j = scale·(g·([j = t] − p_j) − h·p_j·(log p_j + H)),  p_j = e^(z_j − lse)
//
// In 32 bits lse loses log s1 beside a large m (a row of the type's lowest
// value, logits with an offset of 1e6), and p_j from it is wrong by the factor
// lost. The gradient therefore also takes the two apart, as the row's peak:
// its largest logit and that one's log probability, −log s1; then
// log p_j = scale·(x_j − peak) − log s1, as in the forward pass.
//
// A row whose entries are all −∞ has log probabilities −∞, entropy 0 and
// gradient 0; a row with a NaN or a +∞ has NaN in all of them.
//
// Bound by memory without alternatives: 8192 x 8192 fp32 in 43 us, 6.2 TB/s
// (bf16 34 us, 3.9 TB/s: instructions, 165 of a warp a tile of 512). The
// alternatives cost instructions: 8 of them 63 us, 64 of them 140. One row of
// 262144 bf16 with 20 of them 18.4 us a call (its kernel 14.5 when profiled,
// from cold caches). The gradient is elementwise: 8192 x 8192 fp32 in 83 us, 6.5 TB/s.
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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two float32 operations at once.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// Differences of entries times the scale. Below a scale of 1 the entries are
// halved first: their difference may lie past float's range and its product
// within it. (Above 1 such a product lies past it too.) The factors are pairs
// in the kernel's arguments, where they take no registers (made in the kernel,
// up to 12 registers spilled: 8192 x 8192 with 64 alternatives 143 -> 150 us).
struct Scaled {
  float2 half, log2;  // ½ or 1; the scale over it, times log2 e
  float scale;        // the scale over it
  explicit Scaled(float s) : scale(s < 1.f ? 2.f * s : s) {
    half.x = half.y = s < 1.f ? 0.5f : 1.f;
    log2.x = log2.y = scale * kLog2e;
  }
  __device__ __forceinline__ float difference(float x, float ref) const { return fmaf(x, half.x, -half.x * ref); }
};

struct LogProbsArgs {
  int64_t rows, ld;
  int width, top;
  const int32_t* targets;
  float scale;
  Scaled k;
  float* logprob;
  float* entropy;
  float* lse;
  float* peak;  // [2, rows] or null: the largest logit, its log probability
  int32_t* top_index;
  float* top_logprob;
  int* bad_index;
};

// The sums of a part of a row about a reference, its largest entry, with
// t = log2(e^(scale·(x − ref))): s1 = Σ 2^t, s2 = Σ 2^t·t. While s1 is 0,
// nothing above −∞ has been met and the reference says nothing.
struct RowSums {
  float ref, s1, s2;

  // the same sums about another reference
  __device__ __forceinline__ void move(float to, const Scaled& k) {
    const float t = k.difference(ref, to) * k.log2.x;
    ref = to;
    const float c = s1 == 0.f ? 0.f : ex2_approx(t);
    s2 = c == 0.f ? 0.f : c * fmaf(t, s1, s2);
    s1 = c == 0.f ? 0.f : c * s1;
  }
};

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
__device__ __forceinline__ RowSums warp_join(RowSums v, const Scaled& k) {
  v.move(warp_max_nan(v.ref), k);
  v.s1 = warp_sum(v.s1);
  v.s2 = warp_sum(v.s2);
  return v;
}

// One pass over each row by the warps of a block, or of a cluster of blocks
// where there are too few rows for the SMs. A warp takes tiles of 32·kItems
// entries, the next tile's loads under way while this one is summed; each
// thread's sums are about its own running maximum (moved only when a tile
// has a larger one). No warp waits for another until its row is read.
//
// The alternatives: every warp keeps its first `top` in order in registers,
// one or two a lane, and a bound that `top` entries of the row reach, so that
// a tile without an entry above it costs a comparison. A tile's entries above
// it go to shared memory; a few of them are put in their places one by one,
// more are sorted across the lanes, 32 at a time, and merged, and either
// gives a new bound. (Both lie outside the unrolled loop over the entries:
// inside it they missed the instruction cache, 118 issue slots an entry.) The first
// bound comes from the first tile: the top-th largest of the lanes' maxima
// (of half a lane's entries each past 32); a tile with many entries above the
// bound gives another one in the same way before any is taken. The warps of
// a block tell one another their bounds. At the end the lists are joined two
// by two, in the block and then by the cluster's first block.
constexpr int kItems = 16;
constexpr int kMany = 24;      // lanes with entries above the bound that ask for another bound first
constexpr uint32_t kAnyColumn = 0x7fffffffu;  // of a bound that is a value only: behind all columns
constexpr int kFew = 3;        // entries that are put in their places one by one
constexpr int kMaxSplit = 16;  // blocks of a cluster
constexpr int kMaxWarps = 16;  // of a block
static_assert(kMaxSplit <= kMaxWarps, "a warp for every part of a row");

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A warp's first 32·N keys in descending order: place 32·n + lane.
template <int N>
struct TopKeys {
  uint64_t key[N];

  __device__ __forceinline__ void insert(uint64_t x, int lane) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int above = __popc(__ballot_sync(kFull, key[n] > x));
      const uint64_t last = __shfl_sync(kFull, key[n], 31), up = __shfl_up_sync(kFull, key[n], 1);
      key[n] = lane < above ? key[n] : lane == above ? x : up;
      if (above < 32) x = last;  // goes to the head of the next 32
    }
  }
  // One step of a bitonic network: the lanes whose `bit` is 0 keep the larger
  // of a pair where `falling`, the others the smaller.
  static __device__ __forceinline__ uint64_t exchange(uint64_t x, int bit, bool falling, int lane) {
    const uint64_t other = __shfl_xor_sync(kFull, x, bit);
    return (other > x) == (((lane & bit) == 0) == falling) ? other : x;
  }
  static __device__ __forceinline__ uint64_t fall(uint64_t x, int lane) {
#pragma unroll
    for (int bit = 16; bit > 0; bit >>= 1) x = exchange(x, bit, true, lane);
    return x;
  }
  // Takes in another warp's list.
  __device__ __forceinline__ void join(const TopKeys& o, int lane) {
    if (N == 1) {
      key[0] = fall(larger(key[0], __shfl_sync(kFull, o.key[0], 31 - lane)), lane);
    } else {
      const uint64_t a = larger(key[0], __shfl_sync(kFull, o.key[N - 1], 31 - lane));
      const uint64_t b = larger(key[N - 1], __shfl_sync(kFull, o.key[0], 31 - lane));
      key[0] = fall(larger(a, b), lane);
      key[N - 1] = fall(a < b ? a : b, lane);
    }
  }
  __device__ __forceinline__ void load(const uint64_t* p, int lane) {
#pragma unroll
    for (int n = 0; n < N; ++n) key[n] = p[32 * n + lane];
  }
  __device__ __forceinline__ void store(uint64_t* p, int lane) const {
#pragma unroll
    for (int n = 0; n < N; ++n) p[32 * n + lane] = key[n];
  }
  // Takes in the keys of the first n lanes; the others' are 0.
  __device__ __forceinline__ void merge(uint64_t x, int n, int lane) {
    // rising over the lanes, so that the larger of each lane's two are the
    // first 32 of both, in an order that `fall` makes descending; few keys are
    // sorted among few lanes and moved behind the zeros
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
      for (int bit = size / 2; bit > 0; bit >>= 1) x = exchange(x, bit, (lane & size) != 0, lane);
      if (size >= 8 && size < 32 && n <= size) {
        x = __shfl_sync(kFull, x, (lane + size) & 31);
        break;
      }
    }
    key[N - 1] = fall(larger(key[N - 1], x), lane);
    if (N == 2) {
      const uint64_t rising = __shfl_sync(kFull, key[N - 1], 31 - lane);
      key[N - 1] = fall(key[0] < rising ? key[0] : rising, lane);
      key[0] = fall(larger(key[0], rising), lane);
    }
  }
  __device__ __forceinline__ uint64_t at(int place) const {
    uint64_t r = __shfl_sync(kFull, key[0], place & 31);
#pragma unroll
    for (int n = 1; n < N; ++n) {
      const uint64_t k = __shfl_sync(kFull, key[n], place & 31);
      if (place >= 32 * n) r = k;
    }
    return r;
  }
};

template <int WARPS>
struct RowShared {
  union {
    uint2 found[WARPS][32 * kItems];  // a tile's entries that may be above the bound: value and column
    uint64_t list[WARPS][kMaxTop];    // at the end
  };
  unsigned long long bound;
  RowSums warp_sums[WARPS];
  RowSums sums;
};
// Joins the lists of `count` warps (a power of two) two by two into warp 0's.
template <int WARPS, int N>
__device__ __forceinline__ void join_lists(RowShared<WARPS>& sh, TopKeys<N>& list, int count, int warp, int lane) {
  for (int half = count / 2; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half) list.store(sh.list[warp], lane);
    __syncthreads();
    if (warp < half) {
      TopKeys<N> other;
      other.load(sh.list[warp + half], lane);
      list.join(other, lane);
    }
  }
}

// N: registers a lane for the alternatives, 0 where none are asked for.
template <typename T, int WARPS, int N>
__global__ void __launch_bounds__(WARPS * 32, 32 / WARPS)
    logprobs_kernel(LogProbsArgs a, int split, const T* __restrict__ logits) {
  constexpr int V = 16 / int(sizeof(T));  // entries of a 16-byte group
  constexpr int G = kItems / V;           // a lane's groups of a tile
  constexpr int kTile = 32 * kItems;
  extern __shared__ __align__(16) unsigned char row_memory[];
  RowShared<WARPS>& sh = *reinterpret_cast<RowShared<WARPS>*>(row_memory);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const T* x = logits + row * a.ld;
  // groups are those of memory: the first may begin before the row
  const int skip = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int tiles = (a.width + skip + kTile - 1) / kTile;
  const int step = WARPS * split;
  const Scaled& k = a.k;
  // column of a lane's entry i of a tile
  auto column = [&](int tile, int i) { return tile * kTile + (i / V) * (32 * V) + lane * V - skip + i % V; };

  Pack<T, V> next[G];
  auto load = [&](int tile) {
    const int first = tile * kTile - skip;
    if (first >= 0 && first + kTile <= a.width) {
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

  int tile = part * WARPS + warp;
  if (tile < tiles) load(tile);
  const int t = part == 0 && threadIdx.x == 0 ? a.targets[row] : -1;
  float xt = 0.f;
  if (t >= 0) {
    if (t < a.width)
      xt = widen(x[t]);
    else
      *a.bad_index = 1;
  }
  RowSums sums{-INFINITY, 0.f, 0.f};
  float lost1 = 0.f, lost2 = 0.f;  // what rounding added to the sums too much
  TopKeys<N ? N : 1> list;
#pragma unroll
  for (int n = 0; n < (N ? N : 1); ++n) list.key[n] = 0;
  uint64_t bound = 0;  // an entry has to be above this key; 0: no bound yet
  // the least value above the bound: the bound's own for columns before its
  // own, the next one for columns behind it
  float least_before = NAN, least_behind = NAN;
  uint32_t bound_column = 0;
  auto raise = [&](uint64_t to) {
    bound = to;
    bound_column = rank_index(to);
    least_before = rank_value(uint32_t(to >> 32));
    least_behind = rank_value(uint32_t(to >> 32) + 1);
  };
  if (N && WARPS > 1) {
    if (threadIdx.x == 0) sh.bound = 0;
    __syncthreads();
  }
  for (; tile < tiles; tile += step) {
    float v[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) v[i] = next[i / V].get(i % V);
    if (tile + step < tiles) load(tile + step);
    float quarter[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) quarter[q] = max3_nan(max_nan(v[4 * q], v[4 * q + 1]), v[4 * q + 2], v[4 * q + 3]);
    const float half0 = max_nan(quarter[0], quarter[1]), half1 = max_nan(quarter[2], quarter[3]);
    const float most = max_nan(half0, half1);
    const float higher = max_nan(sums.ref, most);
    if (!(higher == sums.ref)) {
      sums.s1 -= lost1;
      sums.s2 -= lost2;
      lost1 = lost2 = 0.f;
      sums.move(higher, k);
    }
    const float ref = sums.ref == -INFINITY ? 0.f : sums.ref;
    float2 s1 = make_float2(0.f, 0.f), s2 = s1;
    const float2 minus = make_float2(-k.half.x * ref, -k.half.x * ref);
#pragma unroll
    for (int i = 0; i < kItems; i += 2) {
      float2 t = mul2(fma2(make_float2(v[i], v[i + 1]), k.half, minus), k.log2);
      t = make_float2(max_nan(t.x, -FLT_MAX), max_nan(t.y, -FLT_MAX));  // −∞ times 2^−∞ = 0 would be no number
      const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
      s1 = add2(s1, e);
      s2 = fma2(e, t, s2);
    }
    add_kept(sums.s1, lost1, s1.x + s1.y);
    add_kept(sums.s2, lost2, s2.x + s2.y);
    if (N == 0) continue;

    float least = least_behind;
    if (WARPS > 1) {
      const uint64_t told = *static_cast<volatile unsigned long long*>(&sh.bound);
      if (told > bound) raise(told);
      least = column(tile, 0) - lane * V > int(bound_column) ? least_behind : least_before;
    }
    const unsigned lanes = __ballot_sync(kFull, !(most < least));
    if (lanes == 0) continue;
    if (bound == 0 || __popc(lanes) > kMany) {
      // lanes without an entry of the row give no bound
      const bool none0 = column(tile, kItems / 2 - 1) < 0 || column(tile, 0) >= a.width;
      const bool none1 = column(tile, kItems - 1) < 0 || column(tile, kItems / 2) >= a.width;
      uint32_t reached = 0;
      if (N == 1) {
        // the maxima in order over the lanes
        uint32_t mine = none0 && none1 ? 0u : rank_bits(none1 ? half0 : none0 ? half1 : most);
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
          for (int bit = size / 2; bit > 0; bit >>= 1) {
            const uint32_t other = __shfl_xor_sync(kFull, mine, bit);
            mine = ((lane & bit) == 0) == ((lane & size) == 0) ? max(mine, other) : min(mine, other);
          }
        reached = __shfl_sync(kFull, mine, a.top - 1);
      } else {
        reached = __reduce_min_sync(kFull, min(none0 ? 0u : rank_bits(half0), none1 ? 0u : rank_bits(half1)));
      }
      if (reached && uint64_t(reached) << 32 > bound) {
        raise(uint64_t(reached) << 32 | (0xffffffffu - kAnyColumn));
        if (WARPS > 1 && lane == 0) atomicMax(&sh.bound, bound);
        least = least_before;
      }
    }
    uint2* found = sh.found[warp];
    int n = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!__any_sync(kFull, !(quarter[q] < least))) continue;
#pragma unroll
      for (int i = 4 * q; i < 4 * q + 4; ++i) {
        const bool maybe = !(v[i] < least);
        const unsigned who = __ballot_sync(kFull, maybe);
        if (!who) continue;
        if (maybe) found[n + __popc(who & ((1u << lane) - 1))] = make_uint2(__float_as_uint(v[i]), column(tile, i));
        n += __popc(who);
      }
    }
    if (n == 0) continue;
    __syncwarp();
    auto key_of = [&](int i) {
      const uint2 f = found[i];
      return int(f.y) >= 0 && int(f.y) < a.width ? rank_key(__uint_as_float(f.x), f.y) : uint64_t(0);
    };
    if (n <= kFew) {
#pragma unroll 1
      for (int i = 0; i < n; ++i) list.insert(key_of(i), lane);
    } else {
#pragma unroll 1
      for (int i = 0; i < n; i += 32) list.merge(i + lane < n ? key_of(i + lane) : 0, n - i, lane);
    }
    __syncwarp();
    const uint64_t last = list.at(a.top - 1);
    if (last > bound) {
      raise(last);
      if (WARPS > 1 && lane == 0) atomicMax(&sh.bound, bound);
    }
  }

  const RowSums none{-INFINITY, 0.f, 0.f};
  sums.s1 -= lost1;
  sums.s2 -= lost2;
  sums = warp_join(sums, k);
  if (WARPS > 1) {
    if (lane == 0) sh.warp_sums[warp] = sums;
    __syncthreads();
    sums = warp_join(lane < WARPS ? sh.warp_sums[lane % WARPS] : none, k);
    if (N) join_lists<WARPS, N ? N : 1>(sh, list, WARPS, warp, lane);
  }
  if (split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) sh.sums = sums;
    if (N && warp == 0) list.store(sh.list[0], lane);
    cluster.sync();
    if (part == 0) sums = warp_join(lane < split ? cluster.map_shared_rank(&sh, lane % split)->sums : none, k);
    if (N && part == 0 && warp < split) list.load(cluster.map_shared_rank(&sh, warp)->list[0], lane);
    cluster.sync();  // the parts' shared memory is read until here
    if (part) return;
    if (N) join_lists<WARPS, N ? N : 1>(sh, list, split, warp, lane);
  }
  const bool empty = sums.s1 == 0.f;
  const float ref = empty ? 0.f : sums.ref, logs = logf(sums.s1);
  auto log_prob = [&](float x) { return empty ? -INFINITY : fmaf(k.difference(x, ref), k.scale, -logs); };
  if (threadIdx.x == 0) {
    const bool skipped = t < 0 || t >= a.width;
    a.logprob[row] = skipped ? 0.f : log_prob(xt);
    a.entropy[row] = empty ? 0.f : logs - kLn2 * (sums.s2 / sums.s1);
    a.lse[row] = fmaf(ref, a.scale, logs);
    if (a.peak) {
      a.peak[row] = sums.ref;
      a.peak[a.rows + row] = empty ? -INFINITY : -logs;
    }
  }
  if (N == 0) return;
#pragma unroll
  for (int n = 0; n < (N ? N : 1); ++n) {
    const int i = n * 32 + lane;
    if (warp > 0 || i >= a.top) return;
    const uint64_t key = list.key[n];
    a.top_index[row * a.top + i] = int32_t(rank_index(key));
    a.top_logprob[row * a.top + i] = log_prob(rank_value(uint32_t(key >> 32)));
  }
}

template <typename T, int WARPS, int N>
int launch_logprobs(const LogProbsArgs& a, const T* logits, cudaStream_t s) {
  auto kernel = logprobs_kernel<T, WARPS, N>;
  // blocks of a row: as many as fill the SMs (32 warps each), at most one for
  // every WARPS tiles
  const int64_t tiles = (int64_t(a.width) + WARPS * 32 * kItems - 1) / (WARPS * 32 * kItems);
  const int64_t room = int64_t(sm_count()) * (32 / WARPS);
  int split = 1;
  while (WARPS == kMaxWarps && split * 2 <= std::min<int64_t>(kMaxSplit, tiles) && a.rows * split * 2 <= room) split *= 2;
  static OncePerDevice ready;
  if (ready.first()) {
    FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(RowShared<WARPS>))));
    FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready.done();
  }
  if (split == 1) {
    kernel<<<unsigned(a.rows), WARPS * 32, sizeof(RowShared<WARPS>), s>>>(a, 1, logits);
    FG_CUDA_TRY(cudaGetLastError());
    return FG_OK;
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.rows * split));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = sizeof(RowShared<WARPS>);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, split, logits));
  return FG_OK;
}

template <typename T, int WARPS>
int launch_logprobs(const LogProbsArgs& a, const T* logits, cudaStream_t s) {
  if (a.top == 0) return launch_logprobs<T, WARPS, 0>(a, logits, s);
  return a.top <= 32 ? launch_logprobs<T, WARPS, 1>(a, logits, s) : launch_logprobs<T, WARPS, 2>(a, logits, s);
}

struct LogProbsGradArgs {
  int64_t rows, ld, ldd;
  int width;
  const int32_t* targets;
  float scale;
  Scaled k;
  const float* lse;  // or the peak and its log probability
  const float* peak;
  const float* peak_logprob;
  const float* entropy;
  const float* dlogprob;
  const float* dentropy;
  int* bad_index;
};

// Elementwise: a warp takes kGradGroups 16-byte groups a lane of one row, all
// loaded before the first is used; groups are those of the logits' memory,
// stored whole where the gradient's lie alike. PEAK: log p from the row's peak,
// else from lse (8192 x 8192, peak and lse: fp32 85 and 83 us, bf16 61 and 60).
constexpr int kGradWarps = 8;
constexpr int kGradGroups = 4;

template <typename T, bool ENTROPY, bool PEAK>
__global__ void __launch_bounds__(kGradWarps * 32) logprobs_grad_kernel(LogProbsGradArgs a, int parts, const T* logits,
                                                                       T* dlogits) {
  constexpr int V = 16 / int(sizeof(T));
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(blockIdx.x) * kGradWarps + (threadIdx.x >> 5);
  const int64_t row = unit / parts;
  const int part = int(unit % parts);
  if (row >= a.rows) return;
  const T* x = logits + row * a.ld;
  T* dx = dlogits + row * a.ldd;
  const int skip = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const int64_t j0 = (int64_t(part) * (32 * kGradGroups) + lane) * V - skip;
  Pack<T, V> in[kGradGroups];
#pragma unroll
  for (int g = 0; g < kGradGroups; ++g) {
    const int64_t j = j0 + g * 32 * V;
    if (j >= 0 && j + V <= a.width) {
      in[g].load_own(x + j);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) in[g].v[i] = j + i >= 0 && j + i < a.width ? x[j + i] : narrow<T>(0.f);
    }
  }
  const int t = a.targets[row];
  if (t >= a.width && part == 0 && lane == 0) *a.bad_index = 1;
  const bool none = t < 0 || t >= a.width;
  const float ref = PEAK ? a.peak[row] : a.lse[row];
  const float peak_logprob = PEAK ? a.peak_logprob[row] : 0.f;
  const Scaled& k = a.k;
  const float g0 = none ? 0.f : a.dlogprob[row];
  const bool empty = ref == -INFINITY;
  float h = 0.f, H = 0.f;
  if (ENTROPY) {
    h = a.dentropy[row];
    H = a.entropy[row];
  }
#pragma unroll
  for (int g = 0; g < kGradGroups; ++g) {
    const int64_t j = j0 + g * 32 * V;
    if (j >= a.width) break;
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // the product with lse rounded as it is in lse, so that the largest entry
      // of a row that has all the probability has exactly 1
      const float lp = PEAK ? fmaf(k.difference(in[g].get(i), ref), k.scale, peak_logprob)
                            : __fsub_rn(__fmul_rn(in[g].get(i), a.scale), ref);
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
  constexpr int V = 16 / int(sizeof(T)), kPart = 32 * kGradGroups * V;
  // a row that begins inside a 16-byte group reaches into one more
  const bool aligned = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && a.ld % V == 0;
  const int64_t parts = (int64_t(a.width) + (aligned ? 0 : V - 1) + kPart - 1) / kPart;
  // rows that one launch's grid holds; more only past 2^31 blocks
  const int64_t most = int64_t(INT32_MAX) * kGradWarps / parts;
  for (int64_t r = 0; r < a.rows; r += most) {
    LogProbsGradArgs b = a;
    b.rows = std::min(most, a.rows - r);
    b.targets += r;
    if (a.peak) {
      b.peak += r;
      b.peak_logprob += r;
    } else {
      b.lse += r;
    }
    b.dlogprob += r;
    if (a.dentropy) {
      b.dentropy += r;
      b.entropy += r;
    }
    auto kernel = a.dentropy ? (a.peak ? logprobs_grad_kernel<T, true, true> : logprobs_grad_kernel<T, true, false>)
                             : (a.peak ? logprobs_grad_kernel<T, false, true> : logprobs_grad_kernel<T, false, false>);
    const unsigned blocks = unsigned((b.rows * parts + kGradWarps - 1) / kGradWarps);
    kernel<<<blocks, kGradWarps * 32, 0, s>>>(b, int(parts), logits + r * a.ld, dlogits + r * a.ldd);
    FG_CUDA_TRY(cudaGetLastError());
  }
  return FG_OK;
}

int log_probs(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
              float scale, int top, float* logprob, float* entropy, float* lse, float* peak, int32_t* top_index,
              float* top_logprob, void* stream) {
  clear_error();
  if (rows < 0 || width <= 0 || rows >= INT32_MAX || width > (1 << 30))
    return set_error(FG_EINVAL, "fg_log_probs: bad shape [%lld x %lld]", (long long)rows, (long long)width);
  if (!known_dtype(dtype)) return set_error(FG_EINVAL, "fg_log_probs: unknown element type %d", dtype);
  if (ld < width) return set_error(FG_EINVAL, "fg_log_probs: leading dimension smaller than the row");
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(FG_EINVAL, "fg_log_probs: scale must be positive and finite");
  if (std::isinf(scale * kLog2e)) return set_error(FG_EINVAL, "fg_log_probs: scale %g is too large", double(scale));
  if (top < 0 || top > kMaxTop || top > width)
    return set_error(FG_EINVAL, "fg_log_probs: %d alternatives of %lld columns (at most %d)", top, (long long)width, kMaxTop);
  if (rows == 0) return FG_OK;
  if (!logits || !targets || !logprob || !entropy || !lse || (top > 0 && (!top_index || !top_logprob)))
    return set_error(FG_EINVAL, "fg_log_probs: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LogProbsArgs a{rows, ld, int(width), top, targets, scale, Scaled(scale), logprob, entropy, lse, peak, top_index, top_logprob, nullptr};
  FG_TRY(device_index_word(&a.bad_index));
  return by_dtype(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    const T* x = static_cast<const T*>(logits);
    // Warps of a row: a warp that takes more of a row pays its first tile's
    // alternatives less often, so no more than the SMs' 32 each (up to 0.7 of
    // them), and no more than the row has tiles; past 16, blocks of a cluster.
    // (2048 x 32768 fp32, 8 alternatives: 2 warps 64 us, 8 warps 81, 16 warps 104.)
    const int64_t enough = int64_t(sm_count()) * 32 * 7 / 10;
    int warps = 1;
    while (warps < kMaxWarps && rows * warps < enough && width > warps * 32 * kItems) warps *= 2;
    switch (warps) {
      case 1: return launch_logprobs<T, 1>(a, x, s);
      case 2: return launch_logprobs<T, 2>(a, x, s);
      case 4: return launch_logprobs<T, 4>(a, x, s);
      case 8: return launch_logprobs<T, 8>(a, x, s);
      default: return launch_logprobs<T, kMaxWarps>(a, x, s);
    }
  });
}

// From lse, or from peak where lse is null.
int log_probs_grad(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                   float scale, const float* lse, const float* peak, const float* entropy, const float* dlogprob,
                   const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  clear_error();
  if (rows < 0 || width <= 0 || rows >= INT32_MAX || width >= INT32_MAX)
    return set_error(FG_EINVAL, "fg_log_probs_grad: bad shape [%lld x %lld]", (long long)rows, (long long)width);
  if (!known_dtype(dtype)) return set_error(FG_EINVAL, "fg_log_probs_grad: unknown element type %d", dtype);
  if (ld < width || ldd < width) return set_error(FG_EINVAL, "fg_log_probs_grad: leading dimension smaller than the row");
  if (!(scale > 0.f) || std::isinf(scale)) return set_error(FG_EINVAL, "fg_log_probs_grad: scale must be positive and finite");
  if (rows == 0) return FG_OK;
  if (!logits || !targets || (!lse && !peak) || !dlogprob || !dlogits || (dentropy && !entropy))
    return set_error(FG_EINVAL, "fg_log_probs_grad: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LogProbsGradArgs a{rows, ld, ldd, int(width), targets, scale, Scaled(scale), lse, peak, peak ? peak + rows : nullptr,
                     entropy, dlogprob, dentropy, nullptr};
  FG_TRY(device_index_word(&a.bad_index));
  return by_dtype(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    return launch_logprobs_grad(a, static_cast<const T*>(logits), static_cast<T*>(dlogits), s);
  });
}

}  // namespace

}  // namespace fg

using namespace fg;

extern "C" {

int fg_log_probs(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                 float scale, int top, float* logprob, float* entropy, float* lse, int32_t* top_index,
                 float* top_logprob, void* stream) {
  return log_probs(logits, dtype, rows, width, ld, targets, scale, top, logprob, entropy, lse, nullptr, top_index,
                   top_logprob, stream);
}

int fg_log_probs_peak(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                      float scale, int top, float* logprob, float* entropy, float* lse, float* peak,
                      int32_t* top_index, float* top_logprob, void* stream) {
  return log_probs(logits, dtype, rows, width, ld, targets, scale, top, logprob, entropy, lse, peak, top_index,
                   top_logprob, stream);
}

int fg_log_probs_grad(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                      float scale, const float* lse, const float* entropy, const float* dlogprob,
                      const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  return log_probs_grad(logits, dtype, rows, width, ld, targets, scale, lse, nullptr, entropy, dlogprob, dentropy,
                        dlogits, ldd, stream);
}

int fg_log_probs_grad_peak(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld,
                           const int32_t* targets, float scale, const float* peak, const float* entropy,
                           const float* dlogprob, const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  return log_probs_grad(logits, dtype, rows, width, ld, targets, scale, nullptr, peak, entropy, dlogprob, dentropy,
                        dlogits, ldd, stream);
}

}  // extern "C"
