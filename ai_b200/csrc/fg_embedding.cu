// The embedding table's operators: rows gathered by token id and scaled,
// and the table's gradient, the sum of the gradients of the tokens that met
// each row.
//
//   lookup:   y[t] = scale · W[id_t]
//   gradient: G[v] = scale · Σ_{t : id_t = v} dy[t]
//
// Few tokens' gradient (up to 2048, of not too many columns) is one launch whose
// blocks group the tokens in a hash table each. Others are sorted by id, stably, so a row's tokens stay in
// their order (within one cluster up to 262144, through memory beyond), and
// cut into chunks of equal length however often a token occurs; the runs of
// one id are summed in registers, and those longer than a chunk joined in a
// second kernel. Sums are in 32 bits in an order that depends on the ids
// alone, so a repeated call gives the same bits; a sum is rounded once, when
// its row is written.
//
// Bound by memory for many tokens: 131072 of 768 fp32 into a table of 262144
// rows, 228 us for 1208 MB (5.3 TB/s): zeros beside the sort 107, sums 93, long
// runs 12, the rest marks and launches. 1024 of 768 bf16 into 2048 rows: 14.4 us
// a call, the latency of one kernel.
#include <cooperative_groups.h>

#include <algorithm>

#include "fg_kernels.cuh"
#include "fg_launch.cuh"
#include "fg_ptx.cuh"
#include "fg_types.cuh"

namespace fg {

namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;

bool multiple_of(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0; }

// Whether rows of type code dt at p with leading dimension ld hold whole
// groups of n values, each at a multiple of its size (16 bytes at most).
bool grouped(const void* p, int dt, int64_t dim, int64_t ld, int n) {
  const int64_t bytes = std::min<int64_t>(16, n * dtype_size(dt));
  return dim % n == 0 && multiple_of(p, bytes) && ld * dtype_size(dt) % bytes == 0;
}

// ---------------------------------------------------------------- lookup
// One warp per token; a lane takes groups of VEC columns 32 groups apart,
// kLookupUnroll of them in flight. Bound by memory: a row read (from L2 when
// it is met again) and one written per token. 131072 tokens of 768 fp32: 88 us,
// 4.6 TB/s written alone; 24 tokens: 10.4 us a call, the launch.
constexpr int kLookupWarps = 8;
constexpr int kLookupUnroll = 4;

template <typename TW, typename TY, int VEC>
__global__ void __launch_bounds__(kLookupWarps * 32) lookup_kernel(const TW* __restrict__ table, int64_t vocab, int dim,
                                                                  int64_t ldt, const int32_t* __restrict__ ids,
                                                                  int64_t n, float scale, int padding,
                                                                  TY* __restrict__ out, int64_t ldo, int* bad_index) {
  const int64_t t = int64_t(blockIdx.x) * kLookupWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= n) return;
  const int id = ids[t];
  const bool pad = id == padding;
  const bool bad = !pad && (id < 0 || id >= vocab);
  if (bad && lane == 0) *bad_index = 1;
  TY* y = out + t * ldo;
  const int groups = dim / VEC;
  if (pad || bad) {
    Pack<TY, VEC> z;
#pragma unroll
    for (int i = 0; i < VEC; ++i) z.set(i, 0.f);
    for (int c = lane; c < groups; c += 32) z.store(y + int64_t(c) * VEC);
    return;
  }
  const TW* w = table + int64_t(id) * ldt;
  for (int c0 = lane; c0 < groups; c0 += 32 * kLookupUnroll) {
    Pack<TW, VEC> in[kLookupUnroll];
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u)
      if (c0 + 32 * u < groups) in[u].load(w + int64_t(c0 + 32 * u) * VEC);
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u) {
      if (c0 + 32 * u >= groups) break;
      Pack<TY, VEC> r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) r.set(i, in[u].get(i) * scale);
      r.store(y + int64_t(c0 + 32 * u) * VEC);
    }
  }
}

// ------------------------------------------------------------------ sort
// Stable sort of (key, position) by the key's bits, DIGIT bits at a time
// from the lowest: per pass the digits of each tile of tokens are counted,
// the counts scanned digit by digit over the tiles, and every token moved to
// its digit's place. A key is the token's id, or `vocab` (after every row)
// for a token without a row: padding, and an id out of range.
constexpr int kSortThreads = 256;
constexpr int kSortItems = 16;  // a thread's tokens of a tile
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigit = 10;

__device__ __forceinline__ uint32_t token_key(int id, int64_t vocab, int padding, int* bad_index) {
  if (id == padding) return uint32_t(vocab);
  if (id < 0 || id >= vocab) {
    *bad_index = 1;
    return uint32_t(vocab);
  }
  return uint32_t(id);
}

// keys of the first pass from the ids (keys == nullptr), else from memory
__device__ __forceinline__ uint32_t sort_key(const int32_t* ids, const uint32_t* keys, int64_t i, int64_t vocab,
                                             int padding, int* bad_index) {
  return keys ? keys[i] : token_key(ids[i], vocab, padding, bad_index);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const int32_t* __restrict__ ids,
                                                                 const uint32_t* __restrict__ keys, int64_t n,
                                                                 int64_t vocab, int padding, int shift, int digit_bits,
                                                                 uint32_t* __restrict__ counts, int* bad_index) {
  __shared__ uint32_t hist[1 << kMaxDigit];
  const int radix = 1 << digit_bits;
  for (int d = threadIdx.x; d < radix; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * kSortTile;
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + k * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(sort_key(ids, keys, i, vocab, padding, bad_index) >> shift) & (radix - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) counts[int64_t(d) * gridDim.x + blockIdx.x] = hist[d];
}

// Exclusive scan of m counts by one block, in place; the total to *total.
constexpr int kScanThreads = 1024;
__global__ void __launch_bounds__(kScanThreads) scan_kernel(uint32_t* __restrict__ x, int64_t m, int32_t* total) {
  __shared__ uint32_t sums[32];
  __shared__ uint32_t carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int64_t base = 0; base < m; base += kScanThreads) {
    const int64_t i = base + threadIdx.x;
    const uint32_t v = i < m ? x[i] : 0;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
      uint32_t w = sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(kFull, w, o);
        if (lane >= o) w += u;
      }
      sums[lane] = w;
    }
    __syncthreads();
    const uint32_t before = carry + (warp ? sums[warp - 1] : 0);
    if (i < m) x[i] = before + s - v;
    __syncthreads();
    if (threadIdx.x == kScanThreads - 1) carry = before + s;
    __syncthreads();
  }
  if (total && threadIdx.x == 0) *total = int32_t(carry);
}

__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const int32_t* __restrict__ ids,
                                                                const uint32_t* __restrict__ keys,
                                                                const uint32_t* __restrict__ pos, int64_t n,
                                                                int64_t vocab, int padding, int shift, int digit_bits,
                                                                const uint32_t* __restrict__ counts,
                                                                uint32_t* __restrict__ keys_out,
                                                                uint32_t* __restrict__ pos_out, int* bad_index) {
  constexpr int kWarps = kSortThreads / 32;
  __shared__ uint32_t next[kWarps][1 << kMaxDigit];  // a warp's next place for each digit
  const int radix = 1 << digit_bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < radix; d += kSortThreads)
#pragma unroll
    for (int w = 0; w < kWarps; ++w) next[w][d] = 0;
  __syncthreads();
  // a warp's tokens are consecutive: 32 in each of its rounds
  const int64_t base = int64_t(blockIdx.x) * kSortTile + int64_t(warp) * 32 * kSortItems + lane;
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + 32 * k;
    key[k] = i < n ? sort_key(ids, keys, i, vocab, padding, bad_index) : 0;
    const unsigned live = __ballot_sync(kFull, i < n);
    rank[k] = 0;
    if (i < n) {
      const uint32_t d = (key[k] >> shift) & (radix - 1);
      const unsigned same = __match_any_sync(live, d);
      const uint32_t before = __popc(same & ((1u << lane) - 1));
      rank[k] = next[warp][d] + before;
      __syncwarp(live);
      if (before == 0) next[warp][d] += __popc(same);
    }
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) {
    uint32_t at = counts[int64_t(d) * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = next[w][d];
      next[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + 32 * k;
    if (i >= n) break;
    const uint32_t to = next[warp][(key[k] >> shift) & (radix - 1)] + rank[k];
    keys_out[to] = key[k];
    pos_out[to] = pos ? pos[i] : uint32_t(i);
  }
}

// ------------------------------------------------------ the rows met
using Mark = uint32_t;

// Number of rows whose first sorted token lies in each tile.
__global__ void __launch_bounds__(kSortThreads) heads_count_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                                  int64_t vocab, uint32_t* __restrict__ counts) {
  int mine = 0;
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = int64_t(blockIdx.x) * kSortTile + k * kSortThreads + threadIdx.x;
    const bool head = i < n && keys[i] < vocab && (i == 0 || keys[i - 1] != keys[i]);
    mine += __syncthreads_count(head);
  }
  if (threadIdx.x == 0) counts[blockIdx.x] = mine;
}

// place[i] = the number of rows met before sorted token i's, row_ids its id.
__global__ void __launch_bounds__(kSortThreads) heads_place_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                                  int64_t vocab, const uint32_t* __restrict__ counts,
                                                                  uint32_t* __restrict__ place,
                                                                  int32_t* __restrict__ row_ids) {
  __shared__ int sums[kSortThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t before = counts[blockIdx.x];
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = int64_t(blockIdx.x) * kSortTile + k * kSortThreads + threadIdx.x;
    const bool live = i < n && keys[i] < vocab;
    const bool head = live && (i == 0 || keys[i - 1] != keys[i]);
    const unsigned mask = __ballot_sync(kFull, head);
    if (lane == 0) sums[warp] = __popc(mask);
    __syncthreads();
    uint32_t mine = before;
    for (int w = 0; w < kSortThreads / 32; ++w) {
      if (w < warp) mine += sums[w];
      before += sums[w];
    }
    __syncthreads();
    mine += __popc(mask & (kFull >> (31 - lane)));  // heads up to and with this token
    if (live) place[i] = mine - 1;
    if (head) row_ids[mine - 1] = int32_t(keys[i]);
  }
}

// Marks every row that a token met. Stores to one 32-byte sector queue in L2,
// so that a row's mark is a word (131072 tokens, a quarter of them in the first
// 32 rows: 19 us with a byte a row), and an id's tokens first meet in a table
// in the block's shared memory, where all but one usually stay.
constexpr int kMarkThreads = 1024;
constexpr int kMarkBlocks = 32;
constexpr int kMarkTable = 8192;
__global__ void __launch_bounds__(kMarkThreads) met_kernel(const int32_t* __restrict__ ids, int64_t n, int64_t vocab,
                                                          int padding, Mark* met) {
  __shared__ int table[kMarkTable];
  for (int i = threadIdx.x; i < kMarkTable; i += kMarkThreads) table[i] = -1;
  __syncthreads();
#pragma unroll 4
  for (int64_t i = int64_t(blockIdx.x) * kMarkThreads + threadIdx.x; i < n; i += kMarkThreads * kMarkBlocks) {
    const int id = ids[i];
    if (id == padding || id < 0 || id >= vocab) continue;
    if (atomicExch(&table[id % kMarkTable], id) != id) met[id] = 1;
  }
}

__global__ void rest_ids_kernel(int32_t* row_ids, int64_t n, const int32_t* count) {
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < n && i >= *count) row_ids[i] = -1;
}

// -------------------------------------------------- sort within a cluster
// The same sort in one launch: the tokens lie in the registers of a cluster
// of up to 16 blocks, ITEMS a thread, and the blocks wait for one another at
// the cluster's barrier only. Per pass of kMaxDigit bits every warp ranks its
// tokens among those of their digit, 32 at a time; a block orders its tokens
// by digit in shared memory, so that neighbouring lanes write neighbouring
// places; and with all blocks' digit totals every token goes to its place.
// Totals and tokens are exchanged through L2. Measured on 131072 tokens of
// 19 bits: distributed shared memory moved 5 to 7 bytes a cycle and SM, 14200
// cycles a pass for the tokens and 9600 for the totals; lanes of one digit
// found by match_any took 2300 cycles a round (a step for every distinct
// digit), by a vote a bit 850. A pass is now 24000 cycles of 131072 tokens
// (votes 7000, L2 reads at 12 bytes a cycle and SM, which is what the cluster's
// one GPC gets, 11000), 11000 of 8192; all of it 32 and 11 us.
constexpr int kGroupThreads = 1024;
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int kRadix = 1 << kMaxDigit;
constexpr int kWords = kRadix / 2;                    // two 16-bit counters each
constexpr int kHalf = kGroupThreads / kWords;         // threads that share a word's sum over the warps
constexpr int kHalfWarps = kGroupWarps / kHalf;
constexpr int kMaxBlocks = 16;
static_assert(kRadix == kGroupThreads, "a thread for every digit");
constexpr int kMaxGroupItems = 16;

struct GroupArgs {
  const int32_t* ids;
  int n;
  int64_t vocab;
  int padding, passes;
  uint32_t* totals;  // [kMaxBlocks, kWords], two 16-bit totals each, and kMaxBlocks more
  uint32_t* key[2];  // passes write them in turn, the last one key[0] and pos[0]
  uint32_t* pos[2];
  Mark* met;         // a mark for every row, 1 where a token met it; null: not asked for
  uint32_t* place;   // with row_ids and count: the rows met; null: not asked for
  int32_t* row_ids;
  int32_t* count;
  uint32_t* long_runs;  // a count that starts at 0
  int* bad_index;
};

template <int ITEMS>
struct GroupShared {
  union {
    uint32_t counter[kGroupWarps][kWords];  // of every warp's tokens
    uint2 local[kGroupThreads * ITEMS];     // then the block's tokens ordered by digit
  };
  uint32_t offset[kHalf][kWords];
  uint32_t base[kRadix], start[kRadix];
  uint32_t warp_sum[kGroupWarps];
  uint32_t heads[kGroupWarps * ITEMS];
};

// Exclusive sum over the block's threads of v; the total in *all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sum, uint32_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(kFull, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  uint32_t w = warp_sum[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(kFull, w, o);
    if (lane >= o) w += u;
  }
  *all = __shfl_sync(kFull, w, 31);
  const uint32_t before = __shfl_sync(kFull, w, (warp + 31) & 31);
  __syncthreads();
  return s - v + (warp ? before : 0);
}

template <int ITEMS>
__global__ void __launch_bounds__(kGroupThreads, 1) group_kernel(GroupArgs a) {
  constexpr int kPart = kGroupThreads * ITEMS;  // a block's tokens
  extern __shared__ __align__(16) unsigned char smem[];
  GroupShared<ITEMS>& sh = *reinterpret_cast<GroupShared<ITEMS>*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = gridDim.x, block = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  let_next_start();
  if (block == 0 && tid == 0) *a.long_runs = 0;
  if (a.met)  // the barriers of the passes come before the first mark
    for (int64_t i = block * kGroupThreads + tid; i < (a.vocab + 3) / 4; i += blocks * kGroupThreads)
      __stcg(reinterpret_cast<uint4*>(a.met) + i, make_uint4(0, 0, 0, 0));
  uint2 mine[ITEMS];  // (key, position) of consecutive tokens of a warp, 32 a round
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = block * kPart + (warp * ITEMS + k) * 32 + lane;
    mine[k] = make_uint2(i < a.n ? uint32_t(a.ids[i]) : 0u, i);
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)  // places past the last token sort behind every key
    mine[k].x = int(mine[k].y) < a.n ? token_key(int(mine[k].x), a.vocab, a.padding, a.bad_index) : 0xffffffffu;
  for (int p = 0; p < a.passes; ++p) {
    const int shift = p * kMaxDigit;
    uint32_t* key_to = a.key[(a.passes - 1 - p) & 1];
    uint32_t* pos_to = a.pos[(a.passes - 1 - p) & 1];
    if (p > 0) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int i = block * kPart + (warp * ITEMS + k) * 32 + lane;
        mine[k] = i < a.n ? make_uint2(__ldcg(a.key[(a.passes - p) & 1] + i), __ldcg(a.pos[(a.passes - p) & 1] + i))
                          : make_uint2(0xffffffffu, i);
      }
    }
    uint4* zero = reinterpret_cast<uint4*>(&sh.counter[0][0]);
#pragma unroll
    for (int i = 0; i < kGroupWarps * kWords / 4; i += kGroupThreads) zero[i + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint16_t* count = reinterpret_cast<uint16_t*>(sh.counter[warp]);
    // the lanes of each token's digit, for all rounds before the first is counted
    uint32_t rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const uint32_t d = mine[k].x >> shift;
      uint32_t differ = 0;
#pragma unroll
      for (int b = 0; b < kMaxDigit; ++b) {
        const bool set = d >> b & 1;
        differ |= __ballot_sync(kFull, set) ^ (set ? kFull : 0u);
      }
      rank[k] = ~differ;
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const uint32_t d = (mine[k].x >> shift) & (kRadix - 1), same = rank[k];
      const uint32_t before = __popc(same & ((1u << lane) - 1)), seen = count[d];
      rank[k] = seen + before;
      __syncwarp();
      if (before == 0) count[d] = uint16_t(seen + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    {
      const int word = tid % kWords, half = tid / kWords;
      uint32_t c[kHalfWarps], run = 0;  // both counters at once: a block has fewer than 2^16 tokens
#pragma unroll
      for (int w = 0; w < kHalfWarps; ++w) c[w] = sh.counter[half * kHalfWarps + w][word];
#pragma unroll
      for (int w = 0; w < kHalfWarps; ++w) {
        sh.counter[half * kHalfWarps + w][word] = run;
        run += c[w];
      }
      sh.offset[half][word] = run;
    }
    __syncthreads();
    // a word's two digits: their totals, and where they start in the block's order
    uint32_t pair = 0, start = 0;
    if (tid < kWords) {
#pragma unroll
      for (int h = 0; h < kHalf; ++h) {
        const uint32_t c = sh.offset[h][tid];
        sh.offset[h][tid] = pair;
        pair += c;
      }
      __stcg(a.totals + block * kWords + tid, pair);
    }
    uint32_t sum;
    start = block_scan((pair & 0xffffu) + (pair >> 16), sh.warp_sum, &sum);
    if (tid < kWords) {
      sh.start[2 * tid] = start;
      sh.start[2 * tid + 1] = start + (pair & 0xffffu);
    }
    __syncthreads();
    const uint16_t* offset = reinterpret_cast<const uint16_t*>(sh.offset[warp / kHalfWarps]);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const uint32_t d = (mine[k].x >> shift) & (kRadix - 1);
      rank[k] += sh.start[d] + offset[d] + count[d];
    }
    __syncthreads();  // the counters are read: their memory takes the tokens
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) sh.local[rank[k]] = mine[k];
    cluster.sync();
    uint32_t of[kMaxBlocks], low = 0, high = 0, low_before = 0, high_before = 0;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; ++b) of[b] = b < blocks && tid < kWords ? __ldcg(a.totals + b * kWords + tid) : 0;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; ++b) {
      low += of[b] & 0xffffu;
      high += of[b] >> 16;
      low_before += b < block ? of[b] & 0xffffu : 0;
      high_before += b < block ? of[b] >> 16 : 0;
    }
    const uint32_t first = block_scan(low + high, sh.warp_sum, &sum);
    if (tid < kWords) {
      sh.base[2 * tid] = first + low_before - start;
      sh.base[2 * tid + 1] = first + low + high_before - (start + (pair & 0xffffu));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int at = k * kGroupThreads + tid;
      const uint2 it = sh.local[at];
      const uint32_t to = sh.base[(it.x >> shift) & (kRadix - 1)] + at;
      if (to < uint32_t(a.n)) {
        __stcg(key_to + to, it.x);
        __stcg(pos_to + to, it.y);
      }
    }
    if (p + 1 == a.passes && !a.met && !a.place) return;
    cluster.sync();
  }
  // where the rows begin
  unsigned heads[ITEMS];
  uint32_t key[ITEMS], left[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = block * kPart + k * kGroupThreads + tid;
    key[k] = i < a.n ? __ldcg(a.key[0] + i) : 0xffffffffu;
    left[k] = lane == 0 && i > 0 && i < a.n ? __ldcg(a.key[0] + i - 1) : 0xffffffffu;
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t lower = __shfl_up_sync(kFull, key[k], 1), prev = lane == 0 ? left[k] : lower;
    heads[k] = __ballot_sync(kFull, key[k] < a.vocab && prev != key[k]);
    if (lane == 0) sh.heads[k * kGroupWarps + warp] = __popc(heads[k]);
    if (a.met && heads[k] >> lane & 1) a.met[key[k]] = 1;
  }
  if (!a.place) return;
  __syncthreads();
  // heads before each warp's round, in the block
  const bool counts = tid < kGroupWarps * ITEMS;
  uint32_t block_heads;
  const uint32_t heads_before = block_scan(counts ? sh.heads[tid % (kGroupWarps * ITEMS)] : 0, sh.warp_sum, &block_heads);
  if (counts) sh.heads[tid] = heads_before;
  if (tid == 0) __stcg(a.totals + kMaxBlocks * kWords + block, block_heads);
  cluster.sync();
  // a lane for every block's count
  const uint32_t of_block = lane < blocks ? __ldcg(a.totals + kMaxBlocks * kWords + lane) : 0;
  const uint32_t total = __reduce_add_sync(kFull, of_block), before = __reduce_add_sync(kFull, lane < block ? of_block : 0);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = block * kPart + k * kGroupThreads + tid;
    if (i >= a.n) continue;
    const uint32_t upto = before + sh.heads[k * kGroupWarps + warp] + __popc(heads[k] & (kFull >> (31 - lane)));
    if (key[k] < a.vocab) a.place[i] = upto - 1;
    if (heads[k] >> lane & 1) a.row_ids[upto - 1] = int32_t(key[k]);
    if (uint32_t(i) >= total) a.row_ids[i] = -1;
  }
  if (block == 0 && tid == 0) *a.count = int32_t(total);
}

template <int ITEMS>
int launch_group(const GroupArgs& a, int blocks, cudaStream_t s) {
  auto kernel = group_kernel<ITEMS>;
  static OncePerDevice ready;
  if (ready.first()) {
    FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(GroupShared<ITEMS>))));
    FG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready.done();
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(blocks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kGroupThreads);
  cfg.dynamicSmemBytes = sizeof(GroupShared<ITEMS>);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return FG_OK;
}

// Most tokens that a cluster sorts.
constexpr int64_t kMaxGroup = int64_t(kMaxBlocks) * kGroupThreads * kMaxGroupItems;

int group_tokens(const GroupArgs& a, cudaStream_t s) {
  // as many blocks as the tokens fill, then more tokens a thread
  int blocks = 1, items = 1;
  while (blocks < kMaxBlocks && blocks * kGroupThreads < a.n) blocks *= 2;
  while (int64_t(blocks) * kGroupThreads * items < a.n) items *= 2;
  switch (items) {
    case 1: return launch_group<1>(a, blocks, s);
    case 2: return launch_group<2>(a, blocks, s);
    case 4: return launch_group<4>(a, blocks, s);
    case 8: return launch_group<8>(a, blocks, s);
    default: return launch_group<16>(a, blocks, s);
  }
}

// The first sorted token whose key is at least k, looked for by a warp: each
// step probes 32 places.
__device__ __forceinline__ int64_t first_token(const uint32_t* keys, int64_t n, int64_t k, int lane) {
  int64_t lo = 0, hi = n;  // it lies in [lo, hi]
  while (hi > lo) {
    const int64_t step = (hi - lo + 31) / 32, p = lo + lane * step;
    const int c = __popc(__ballot_sync(kFull, p < hi && keys[p] < k));
    if (c == 0) {
      hi = lo;
    } else {
      const int64_t last = lo + (c - 1) * step;
      hi = last + step < hi ? last + step : hi;
      lo = last + 1;
    }
  }
  return lo;
}

// ------------------------------------------------------------------ sums
constexpr int kMaxChunk = 32;  // tokens: a lane for each
constexpr int kMinChunk = 4;
constexpr int kRing = 4;       // rows in flight where tokens are summed
constexpr int kAhead = 8;      // partial sums in flight where they are joined
constexpr int kSumWarps = 8;
constexpr int kNarrowParts = 4;  // groups of 32 columns a warp where values are loaded one by one
// Bytes of a dense gradient from which its zeros are written beside the sort.
constexpr int64_t kZerosFirst = int64_t(32) << 20;

// A warp sums one chunk of sorted tokens over 32·VEC columns, with kRing
// rows in flight (4, 6 and 8 of them, with the warps that their registers
// leave room for, measured alike). A run of one id no longer than a chunk
// belongs to the chunk in which it begins, wherever it ends. A longer run is
// cut where the chunks are: the part in the chunk in which it begins
// goes to tail[chunk], the others to head[chunk], and join_kernel adds them.
// (Runs of any length cut at the chunks' ends: four times as many to join,
// 23 us of 131072 frequent tokens' 240.)
struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  const uint32_t* place;  // row of the output for each sorted token; null: its key
  int64_t n, vocab;
  int chunk;  // tokens of one, a power of two
  int dim, slices;
  int64_t ldy, ldg;
  float scale;
  int accumulate;
  float* head;
  float* tail;  // [chunks, dim] each
  uint32_t* long_runs;  // their number, then the chunks in which they begin, in any order
  // blocks that zero the rows without tokens, spread among those that sum
  int64_t rows;
  const int32_t* count;  // rows met, of the compact gradient; null: the dense one
  const Mark* met;       // a mark for every row of the dense one, 1: has tokens; null: no tokens
  int sum_blocks, zero_blocks;
};

template <typename TG, int VEC>
__device__ __forceinline__ void write_row(TG* g, const float (&acc)[VEC], float scale, int accumulate) {
  Pack<TG, VEC> r;
  if (accumulate) {
    r.load_own(g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.set(i, __fadd_rn(r.get(i), __fmul_rn(acc[i], scale)));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.set(i, acc[i] * scale);
  }
  r.store(g);
}

// Zeros in n consecutive values from anywhere, by a warp: whole 16 bytes but
// for the ends.
template <typename T>
__device__ __forceinline__ void zero_values(T* p, int64_t n, int lane) {
  constexpr int V = 16 / int(sizeof(T));
  const int64_t before = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T);
  const int64_t head = n < before ? n : before, groups = (n - head) / V, tail = head + groups * V;
  for (int64_t g = lane; g < groups; g += 32) __stcs(reinterpret_cast<uint4*>(p + head) + g, make_uint4(0, 0, 0, 0));
  if (lane < head) p[lane] = narrow<T>(0.f);
  if (tail + lane < n) p[tail + lane] = narrow<T>(0.f);
}

// Zeros in those of 32 rows whose bit of `keep` is 0, by a warp: the columns
// of its slice (col) where values are stored in fours; else whole rows, those
// that follow one another in one go (20000 tokens into 262144 x 129 bf16
// took 64 us one value a lane, 45 this way; 5000 into 60000 x 301 fp32 43 and
// 37).
template <typename TG, int VEC>
__device__ __forceinline__ void zero_kept(TG* rows, unsigned keep, int col, int dim, int64_t ldg, int lane) {
  if (VEC == 1) {
    for (int r = 0; r < 32;) {
      const unsigned left = ~keep >> r;
      if (left == 0) return;
      r += __ffs(left) - 1;
      const int more = __ffs(~(~keep >> r)) - 1, run = ldg != dim ? 1 : more < 0 ? 32 - r : more;
      zero_values(rows + r * ldg, int64_t(run) * dim, lane);
      r += run;
    }
    return;
  }
  if (col >= dim) return;
  Pack<TG, VEC> z;
#pragma unroll
  for (int i = 0; i < VEC; ++i) z.set(i, 0.f);
  TG* g = rows + col;
#pragma unroll 8
  for (int r = 0; r < 32; ++r)
    if (!(keep >> r & 1)) z.store_past(g + r * ldg);
}

// Zeros in the rows of the dense gradient that no token met (there may be
// no tokens at all), or past the last row of the compact one: a warp takes
// 32·VEC columns of 32 rows, or the rows whole.
template <typename TG, int VEC>
__device__ __forceinline__ void zero_rows(const SumArgs& a, int64_t unit, TG* grad, int lane) {
  const int slices = VEC == 1 ? 1 : a.slices;
  const int64_t r0 = unit / slices * 32;
  const int col = (int(unit % slices) * 32 + lane) * VEC;
  if (r0 >= a.rows) return;
  const int64_t count = a.count ? int64_t(*a.count) - r0 : 0;
  unsigned keep = count >= 32 ? kFull : count > 0 ? (1u << count) - 1 : 0;
  if (!a.count && a.met) keep = __ballot_sync(kFull, r0 + lane < a.rows && a.met[r0 + lane]);
  if (a.rows - r0 < 32) keep |= kFull << (a.rows - r0);
  zero_kept<TG, VEC>(grad + r0 * a.ldg, keep, col, a.dim, a.ldg, lane);
}

// The zeros alone, while the tokens are sorted: needs the marks of the rows
// met, not the sort that runs before it in the stream. Its blocks wait for the
// sort at their end, so that what comes after it comes after both.
template <typename TG, int VEC>
__global__ void __launch_bounds__(kSumWarps * 32) zero_kernel(SumArgs a, TG* grad) {
  zero_rows<TG, VEC>(a, int64_t(blockIdx.x) * kSumWarps + (threadIdx.x >> 5), grad, threadIdx.x & 31);
  wait_for_previous();
}

// SUB: groups of 32·VEC columns that a warp takes together (four where values
// cannot be loaded in fours: 65572 tokens x 529 fp16 96 us with one, 65 with four).
template <typename TY, typename TG, int VEC, int SUB>
__global__ void __launch_bounds__(kSumWarps * 32, 4) sum_kernel(SumArgs a, const TY* __restrict__ dy, TG* grad) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_previous();
  const int64_t zeros = int64_t(blockIdx.x) * a.zero_blocks / (a.sum_blocks + a.zero_blocks);  // before this block
  if (int64_t(blockIdx.x + 1) * a.zero_blocks / (a.sum_blocks + a.zero_blocks) > zeros) {
    zero_rows<TG, VEC>(a, zeros * kSumWarps + warp, grad, lane);
    return;
  }
  const int64_t unit = (blockIdx.x - zeros) * kSumWarps + warp;
  const int parts = (a.slices + SUB - 1) / SUB;
  const int64_t chunk = unit / parts;
  const int col = (int(unit % parts) * SUB * 32 + lane) * VEC;
  const int size = a.chunk;
  const int64_t i0 = chunk * size;
  if (i0 >= a.n) return;
  const uint32_t key = lane < size && i0 + lane < a.n ? a.keys[i0 + lane] : 0xffffffffu;
  const uint32_t left = i0 + lane >= 32 ? a.keys[i0 + lane - 32] : 0xffffffffu;
  const uint32_t right = i0 + size + lane < a.n ? a.keys[i0 + size + lane] : 0xffffffffu;
  const int count = __popc(__ballot_sync(kFull, key < a.vocab));  // tokens without a row come last
  if (count == 0) return;
  const uint32_t first_key = __shfl_sync(kFull, key, 0), last_key = __shfl_sync(kFull, key, count - 1);
  // tokens of the first run before this chunk and in it, of the last one in it and behind it
  const int before = __clz(~__ballot_sync(kFull, left == first_key));
  const int first = __popc(__ballot_sync(kFull, key == first_key)), last = __popc(__ballot_sync(kFull, key == last_key));
  const unsigned same = __ballot_sync(kFull, right == last_key);
  const int behind = count < size ? 0 : same == kFull ? 32 : __ffs(~same) - 1;
  const bool came = before > 0;
  const bool long_first = before + first + (first == size ? behind : 0) > size;
  const bool goes = behind > 0 && !(came && first == size);  // the last run began here
  const bool long_last = goes && last + behind > size;
  const int begin = came && !long_first ? first : 0;
  const int end = count + (goes && !long_last ? behind : 0);
  if (begin >= end) return;
  const uint32_t pos = lane < count ? a.pos[i0 + lane] : 0;
  const uint32_t pos_behind = lane < end - count ? a.pos[i0 + count + lane] : 0;
  const uint32_t row = lane < count ? (a.place ? a.place[i0 + lane] : key) : 0;
  const uint32_t next = __shfl_down_sync(kFull, key, 1);
  // the last tokens of the runs, and of the parts of long ones
  uint64_t ends = __ballot_sync(kFull, lane < count - 1 && next != key);
  ends |= uint64_t(1) << (end - 1);
  const int head = came && long_first ? first - 1 : -1, tail = long_last ? end - 1 : -1;
  if (long_last && unit % parts == 0 && lane == 0) a.long_runs[1 + atomicAdd(a.long_runs, 1u)] = uint32_t(chunk);
  bool in[SUB];
#pragma unroll
  for (int q = 0; q < SUB; ++q) in[q] = col + q * 32 * VEC < a.dim;
  const TY* y = dy + col;
  Pack<TY, VEC> v[kRing][SUB];
  auto load = [&](int u, int t) {
    const uint32_t here = __shfl_sync(kFull, pos, t & 31), there = __shfl_sync(kFull, pos_behind, (t - count) & 31);
    const TY* from = y + int64_t(t < count ? here : there) * a.ldy;
#pragma unroll
    for (int q = 0; q < SUB; ++q)
      if (t < end && in[q]) v[u][q].load(from + q * 32 * VEC);
  };
#pragma unroll
  for (int u = 0; u < kRing; ++u) load(u, begin + u);
  float acc[SUB][VEC];
#pragma unroll
  for (int q = 0; q < SUB; ++q)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[q][i] = 0.f;
  for (int t0 = begin; t0 < end; t0 += kRing) {
#pragma unroll
    for (int u = 0; u < kRing; ++u) {
      const int t = t0 + u;
      if (t >= end) break;
#pragma unroll
      for (int q = 0; q < SUB; ++q)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[q][i] += v[u][q].get(i);
      load(u, t + kRing);
      if (!(ends >> t & 1)) continue;
      const uint32_t to = __shfl_sync(kFull, row, min(t, count - 1));
      const bool part = t == head || t == tail;
      float* ws = (t == head ? a.head : a.tail) + chunk * a.dim + col;
      TG* g = grad + int64_t(to) * a.ldg + col;
#pragma unroll
      for (int q = 0; q < SUB; ++q) {
        if (in[q]) {
          if (part) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) ws[q * 32 * VEC + i] = acc[q][i];
          } else {
            write_row<TG, VEC>(g + q * 32 * VEC, acc[q], a.scale, a.accumulate);
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[q][i] = 0.f;
      }
    }
  }
}

// The long runs: the part in the chunk in which one begins, and the heads of
// the chunks after it, in their order, are its row. A warp joins a run of a
// few chunks; one of many (a frequent token) is shared by the block's warps,
// which take equal consecutive parts of it. A block's warps have different
// runs and the same columns, so the columns of a run meet in different blocks.
constexpr int kLongRun = 16;  // chunks after the first

template <typename TG, int VEC>
__global__ void __launch_bounds__(kSumWarps * 32) join_kernel(SumArgs a, TG* grad) {
  __shared__ int long_run[kSumWarps];
  __shared__ int64_t long_chunk[kSumWarps];
  __shared__ float part[kSumWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_previous();
  const int size = a.chunk, runs = int(a.long_runs[0]);
  const int groups = (runs + kSumWarps - 1) / kSumWarps;  // of a slice
  int col = 0;
  bool in = false;
  // sum of heads [c, c + count) in order, kAhead in flight
  auto add_heads = [&](float (&acc)[VEC], int64_t c, int count) {
    if (!in) return;
    for (int i = 0; i < count; i += kAhead) {
      Pack<float, VEC> h[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u < count) h[u].load_own(a.head + (c + i + u) * a.dim + col);  // written while this kernel waited
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u < count)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += h[u].get(j);
    }
  };
  auto finish = [&](const float (&acc)[VEC], int64_t chunk) {
    const int64_t last = (chunk + 1) * size - 1;
    const int64_t row = a.place ? a.place[last] : a.keys[last];
    if (in) write_row<TG, VEC>(grad + row * a.ldg + col, acc, a.scale, a.accumulate);
  };

  for (int g = blockIdx.x; g < groups * a.slices; g += gridDim.x) {
    const int at = warp * groups + g % groups;  // neighbours in the list, often the longest, apart
    col = (g / groups * 32 + lane) * VEC;
    in = col < a.dim;
    const int64_t chunk = at < runs ? a.long_runs[1 + at] : 0, end = (chunk + 1) * size;
    int run = 0;  // chunks after this one that the run covers
    if (at < runs) {
      const uint32_t key = a.keys[end - 1];
      // the starts of the next 32 chunks, then of 32 groups of 32, or all
      const int64_t start = end + int64_t(lane) * size, far = start + int64_t(lane) * 31 * size;
      const unsigned same = __ballot_sync(kFull, start < a.n && a.keys[start] == key);
      run = __ffs(~same) - 1;
      if (same == kFull) {
        const unsigned fars = __ballot_sync(kFull, far < a.n && a.keys[far] == key);
        if (fars == kFull) {
          run = int((first_token(a.keys + end, a.n - end, int64_t(key) + 1, lane) + size - 1) / size);
        } else {
          const int before = (__ffs(~fars) - 2) * 32;
          const int64_t fine = start + int64_t(before) * size;
          run = before + __popc(__ballot_sync(kFull, fine < a.n && a.keys[fine] == key));
        }
      }
    }
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (run > 0 && run <= kLongRun) {
      if (in)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = a.tail[chunk * a.dim + col + j];
      add_heads(acc, chunk + 1, run);
      finish(acc, chunk);
    }
    if (lane == 0) {
      long_run[warp] = run > kLongRun ? run : 0;
      long_chunk[warp] = chunk;
    }
    __syncthreads();
    for (int w = 0; w < kSumWarps; ++w) {
      const int count = long_run[w];
      if (count == 0) continue;
      const int share = (count + kSumWarps - 1) / kSumWarps, first = warp * share;
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      add_heads(acc, long_chunk[w] + 1 + first, max(0, min(share, count - first)));
#pragma unroll
      for (int j = 0; j < VEC; ++j) part[warp][lane * VEC + j] = acc[j];
      __syncthreads();
      if (warp == w) {
        if (in)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = a.tail[chunk * a.dim + col + j];
        for (int p = 0; p < kSumWarps; ++p)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += part[p][lane * VEC + j];
        finish(acc, chunk);
      }
      __syncthreads();
    }
    __syncthreads();  // long_run is read until here
  }
}

// ------------------------------------------------ few tokens: one launch
// Up to kFewTokens tokens need no order: every block puts all ids into a hash
// table in its shared memory (an id's first token and how many there are), and
// a warp takes 32·VEC columns of one token. If the token is its id's first, the
// warp sums the id's tokens in their order, a long run shared by the block's
// warps; the row of the compact gradient is the number of first tokens with
// smaller ids. Other warps write the zeros: 32 rows of the dense gradient
// each, looked up in the table, or the token's own place in the compact one
// where that lies past the last row. No scratch, and one launch instead of
// three that depend on one another: 1024 tokens x 768 bf16 into 2048 rows
// took 18.5 us in order of ids, 14.4 here; 333 x 256 fp32, rows met, 20 and 14.5.
// But a first token looks through all ids in every slice of its columns, so
// that the work grows with tokens^2 x slices: up to kFewWork of that, beyond it
// the order of ids is cheaper. A call, here and sorted: 1024 x 1024 bf16 14.6
// and 20.8 us, rows met 18.7 and 23.2 (8M); 1500 x 512 20.8 and 21.2, 25.1 and
// 24.0 (9M: the rows met are even there, and one limit does for both); 1024 x 301 fp32 18.0 and 20.9, 21.0 and 24.8 (10M); 1500 x 768
// bf16 23.0 and 21.3, 32.6 and 23.3 (13M); 2048 x 1023 fp32 105 and 25, 168
// and 35 (128M).
constexpr int kFewTokens = 2048;
constexpr int64_t kFewWork = 10 << 20;
constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewBlocks = 4;  // launched for an SM
constexpr int kFewRing = 8;
constexpr int kWholeRun = 32;  // tokens of a run that one warp sums
constexpr uint32_t kNoKey = 0xffffffffu;

struct FewArgs {
  const int32_t* ids;
  int n, words, slots;  // tokens, 32 of them a word, places of the table (a power of two)
  int64_t vocab, rows;
  int padding, dim, slices;
  int64_t ldy, ldg;
  float scale;
  int accumulate;
  int64_t token_units, units;
  int32_t* row_ids;  // of the compact gradient
  int32_t* count;
  int* bad_index;
};

size_t few_shared(int words, int slots) { return size_t(words) * 32 * 4 + size_t(words) * 4 + size_t(slots) * 12; }

template <typename TY, typename TG, int VEC>
__global__ void __launch_bounds__(kFewThreads) few_kernel(FewArgs a, const TY* __restrict__ dy, TG* grad) {
  extern __shared__ __align__(16) unsigned char memory[];
  uint32_t* keys = reinterpret_cast<uint32_t*>(memory);  // [words * 32]
  uint32_t* slot_key = keys + a.words * 32;              // [slots] each
  uint32_t* slot_first = slot_key + a.slots;
  uint32_t* slot_count = slot_first + a.slots;
  uint32_t* firsts = slot_count + a.slots;               // [words] bits: the token is its id's first
  __shared__ uint16_t list[kFewWarps][kFewTokens / kFewWarps];  // positions to sum
  __shared__ float part[kFewWarps][32 * VEC];
  __shared__ int shared_unit[kFewWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t slot_mask = a.slots - 1;
  auto slot_of = [&](uint32_t key) { return (key * 2654435761u >> 16) & slot_mask; };

  for (int i = tid; i < a.slots; i += kFewThreads) {
    slot_key[i] = kNoKey;
    slot_first[i] = kNoKey;
    slot_count[i] = 0;
  }
  for (int i = tid; i < a.words * 32; i += kFewThreads) {
    const uint32_t key = i < a.n ? token_key(a.ids[i], a.vocab, a.padding, a.bad_index) : uint32_t(a.vocab);
    keys[i] = key < a.vocab ? key : kNoKey;
  }
  __syncthreads();
  for (int i = tid; i < a.n; i += kFewThreads) {
    const uint32_t key = keys[i];
    if (key == kNoKey) continue;
    uint32_t s = slot_of(key);
    for (uint32_t was; (was = atomicCAS(&slot_key[s], kNoKey, key)) != kNoKey && was != key;) s = (s + 1) & slot_mask;
    atomicMin(&slot_first[s], uint32_t(i));
    atomicAdd(&slot_count[s], 1u);
  }
  __syncthreads();
  // the place of a key that may be in the table: slots, where it is not
  auto find = [&](uint32_t key) {
    uint32_t s = slot_of(key);
    while (slot_key[s] != key && slot_key[s] != kNoKey) s = (s + 1) & slot_mask;
    return slot_key[s] == key ? s : uint32_t(a.slots);
  };
  for (int i = tid; i < a.words * 32; i += kFewThreads) {
    const uint32_t key = keys[i];
    const unsigned bits = __ballot_sync(kFull, key != kNoKey && slot_first[find(key)] == uint32_t(i));
    if (lane == 0) firsts[i / 32] = bits;
  }
  __syncthreads();

  for (int64_t base = int64_t(blockIdx.x) * kFewWarps; base < a.units; base += int64_t(gridDim.x) * kFewWarps) {
    const int64_t unit = base + warp;
    const bool token = unit < a.token_units;
    // A frequent id's first token comes early: a block's warps take tokens far
    // apart, and the columns of a token meet in different blocks.
    const int64_t at = token ? unit : unit - a.token_units, across = token ? a.words * 32 : (a.rows + 31) / 32;
    const int slice = int(at / across), place_in = int(at % across);
    const int col = (slice * 32 + lane) * VEC;
    const bool in = col < a.dim && unit < a.units;
    const int t = token ? place_in % kFewWarps * (a.words * 32 / kFewWarps) + place_in / kFewWarps : 0;
    Pack<TG, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.set(i, 0.f);
    if (!token && unit < a.units) {  // 32 rows of the dense gradient
      const int64_t r0 = int64_t(place_in) * 32;
      const bool met = r0 + lane < a.rows && find(uint32_t(r0 + lane)) < uint32_t(a.slots);
      unsigned keep = __ballot_sync(kFull, met);
      if (a.rows - r0 < 32) keep |= kFull << (a.rows - r0);
      zero_kept<TG, VEC>(grad + r0 * a.ldg, keep, col, a.dim, a.ldg, lane);
    }
    // first tokens of a smaller key; of any key
    auto firsts_below = [&](uint32_t key) {
      int c = 0;
      for (int w = 0; w < a.words; ++w) c += (firsts[w] >> lane & 1) && keys[w * 32 + lane] < key;
      return __reduce_add_sync(kFull, c);
    };
    const bool first = token && (firsts[t / 32] >> t % 32 & 1);
    const uint32_t key = first ? keys[t] : 0;
    const int run = first ? int(slot_count[find(key)]) : 0;
    int64_t row = key;
    if (a.count && token && t < a.n) {
      if (first) row = firsts_below(key);
      const int met = firsts_below(kNoKey);
      const bool names = slice == 0 && lane == 0;
      if (first && names) a.row_ids[row] = int32_t(key);
      if (t >= met) {
        if (in) zero.store(grad + int64_t(t) * a.ldg + col);
        if (names) a.row_ids[t] = -1;
      }
      if (t == 0 && names) *a.count = met;
    }
    // sums the tokens of a key within some words of tokens, in their order
    const TY* y = dy + col;
    auto sum = [&](float (&acc)[VEC], uint32_t of, int word, int end, bool with) {
      int found = 0;
      for (; word < end; ++word) {
        const bool mine = keys[word * 32 + lane] == of;
        const unsigned who = __ballot_sync(kFull, mine);
        if (mine) list[warp][found + __popc(who & ((1u << lane) - 1))] = uint16_t(word * 32 + lane);
        found += __popc(who);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
      for (int i0 = 0; i0 < found; i0 += kFewRing) {
        Pack<TY, VEC> v[kFewRing];
#pragma unroll
        for (int u = 0; u < kFewRing; ++u)
          if (i0 + u < found && with) v[u].load(y + int64_t(list[warp][i0 + u]) * a.ldy);
#pragma unroll
        for (int u = 0; u < kFewRing; ++u)
          if (i0 + u < found)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += v[u].get(i);
      }
      __syncwarp();  // the list is read until here
    };
    float acc[VEC];
    if (first && run <= kWholeRun) {
      if (run == 1) {
        Pack<TY, VEC> v;
        if (in) v.load(y + int64_t(t) * a.ldy);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = v.get(i);
      } else {
        sum(acc, key, t / 32, a.words, in);
      }
      if (in) write_row<TG, VEC>(grad + row * a.ldg + col, acc, a.scale, a.accumulate);
    }
    if (lane == 0) shared_unit[warp] = first && run > kWholeRun ? t : -1;
    __syncthreads();
    for (int w = 0; w < kFewWarps; ++w) {
      const int of = shared_unit[w];
      if (of < 0) continue;
      const int share = (a.words + kFewWarps - 1) / kFewWarps, word = min(a.words, warp * share);
      // the columns are the unit's, not this warp's own
      const int c = (int((base + w) / (a.words * 32)) * 32 + lane) * VEC;
      y = dy + c;
      sum(acc, keys[of], word, min(a.words, word + share), c < a.dim);
#pragma unroll
      for (int i = 0; i < VEC; ++i) part[warp][lane * VEC + i] = acc[i];
      __syncthreads();
      if (warp == w && in) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
        for (int p = 0; p < kFewWarps; ++p)
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += part[p][lane * VEC + i];
        write_row<TG, VEC>(grad + row * a.ldg + col, acc, a.scale, a.accumulate);
      }
      __syncthreads();
    }
    __syncthreads();  // shared_unit is read until here
  }
}

int64_t blocks_of(int64_t n, int64_t per) { return (n + per - 1) / per; }
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

struct Scratch {
  cudaStream_t s;
  void* p = nullptr;
  explicit Scratch(cudaStream_t st) : s(st) {}
  ~Scratch() { scratch_free(p, s); }
};

// Both gradients: grad is [vocab, dim] and count null, or grad is [n, dim]
// with row_ids [n] and the count.
int embedding_grad(const void* dy, int dy_dtype, int64_t ldy, const int32_t* ids, int64_t n, int64_t vocab, int64_t dim,
                   float scale, int padding, void* grad, int grad_dtype, int64_t ldg, int accumulate, int32_t* row_ids,
                   int32_t* count, cudaStream_t s) {
  int* bad_index = nullptr;
  FG_TRY(device_index_word(&bad_index));
  const bool compact = count != nullptr;
  if (compact && n == 0) {
    FG_CUDA_TRY(cudaMemsetAsync(count, 0, sizeof(int32_t), s));
    return FG_OK;
  }
  const bool wide = grouped(dy, dy_dtype, dim, ldy, 4) && grouped(grad, grad_dtype, dim, ldg, 4);
  const int slices = int(blocks_of(dim, wide ? 128 : 32));
  if (n > 0 && n <= kFewTokens && n * n * slices <= kFewWork) {
    FewArgs f{};
    f.ids = ids;
    f.n = int(n);
    f.words = int(blocks_of(n, 32));
    f.slots = 64;
    while (f.slots < 2 * n) f.slots *= 2;
    f.vocab = vocab;
    f.rows = compact ? n : vocab;
    f.padding = padding;
    f.dim = int(dim);
    f.slices = slices;
    f.ldy = ldy;
    f.ldg = ldg;
    f.scale = scale;
    f.accumulate = accumulate;
    f.token_units = int64_t(f.words) * 32 * slices;
    f.units = f.token_units + (compact || accumulate ? 0 : blocks_of(vocab, 32) * (wide ? slices : 1));
    f.row_ids = row_ids;
    f.count = count;
    f.bad_index = bad_index;
    // Each block makes the table again, so no more than about what runs at once:
    // four an SM with 16-bit gradients or single columns and up to 1024 tokens;
    // three fit from there on (their tables take 57 KB), two where fp32 gradients
    // go in fours (128 registers), and the rest of a full grid follows them.
    const unsigned blocks = unsigned(std::min<int64_t>(blocks_of(f.units, kFewWarps), int64_t(sm_count()) * kFewBlocks));
    const size_t shared = few_shared(f.words, f.slots);
    return by_dtype(grad_dtype, [&](auto tg) {
      return by_dtype(dy_dtype, [&](auto ty) {
        using TG = typename decltype(tg)::type;
        using TY = typename decltype(ty)::type;
        static OncePerDevice ready;
        if (ready.first()) {
          const int most = int(few_shared(kFewTokens / 32, 2 * kFewTokens));
          FG_CUDA_TRY(cudaFuncSetAttribute(few_kernel<TY, TG, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
          FG_CUDA_TRY(cudaFuncSetAttribute(few_kernel<TY, TG, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
          ready.done();
        }
        const TY* y = static_cast<const TY*>(dy);
        if (wide)
          few_kernel<TY, TG, 4><<<blocks, kFewThreads, shared, s>>>(f, y, static_cast<TG*>(grad));
        else
          few_kernel<TY, TG, 1><<<blocks, kFewThreads, shared, s>>>(f, y, static_cast<TG*>(grad));
        FG_CUDA_TRY(cudaGetLastError());
        return FG_OK;
      });
    });
  }
  int bits = 1;
  while (bits < 31 && (int64_t(1) << bits) <= vocab) ++bits;  // keys reach vocab itself
  const int passes = (bits + kMaxDigit - 1) / kMaxDigit;
  const int digit = (bits + passes - 1) / passes;
  // few tokens are cut into shorter chunks, down to kMinChunk, until there are
  // 16 warps an SM: a chunk's rows arrive kRing at a time (measured on 333 tokens
  // x 256 fp32 in this form: sums 11 us in chunks of 32, 6.8 in chunks of 4)
  int chunk = kMaxChunk;
  while (chunk > kMinChunk && blocks_of(n, chunk) * slices < int64_t(sm_count()) * 16) chunk /= 2;
  const int64_t tiles = blocks_of(n, kSortTile), chunks = blocks_of(n, chunk);
  const bool marks = !compact && !accumulate && n > 0;
  const size_t met_bytes = marks ? round256(size_t(vocab) * sizeof(Mark)) : 0;
  const size_t list = round256(size_t(n) * 4), part = round256(size_t(chunks) * dim * 4);
  const bool grouped_here = n <= kMaxGroup;
  const size_t hist = grouped_here ? round256((kMaxBlocks * kWords + kMaxBlocks) * 4)
                                   : round256(size_t(tiles) * (size_t(1) << digit) * 4);
  Scratch ws(s);
  FG_TRY(scratch_alloc(&ws.p, 6 * list + hist + 2 * part + met_bytes, s));
  unsigned char* at = static_cast<unsigned char*>(ws.p);
  auto take = [&](size_t bytes) {
    void* r = at;
    at += bytes;
    return r;
  };
  uint32_t* key[2] = {static_cast<uint32_t*>(take(list)), static_cast<uint32_t*>(take(list))};
  uint32_t* pos[2] = {static_cast<uint32_t*>(take(list)), static_cast<uint32_t*>(take(list))};
  uint32_t* place = static_cast<uint32_t*>(take(list));
  uint32_t* long_runs = static_cast<uint32_t*>(take(list));  // at most one in kMinChunk + 1 tokens begins one
  uint32_t* counts = static_cast<uint32_t*>(take(hist));
  Mark* met = marks ? static_cast<Mark*>(take(met_bytes)) : nullptr;
  SumArgs a{};
  a.met = met;
  a.long_runs = long_runs;
  a.head = static_cast<float*>(take(part));
  a.tail = static_cast<float*>(take(part));
  // A large dense gradient's zeros are written while a cluster sorts (16 of the
  // SMs); the rows met are then marked beforehand.
  const bool zeros_first = met && grouped_here && vocab * dim * dtype_size(grad_dtype) >= kZerosFirst;
  if (zeros_first || (met && !grouped_here)) {
    FG_CUDA_TRY(cudaMemsetAsync(met, 0, met_bytes, s));
    met_kernel<<<kMarkBlocks, kMarkThreads, 0, s>>>(ids, n, vocab, padding, met);
    FG_CUDA_TRY(cudaGetLastError());
  }
  if (n > 0 && grouped_here) {
    GroupArgs g{ids, int(n), vocab, padding, passes, counts, {key[0], key[1]}, {pos[0], pos[1]}, zeros_first ? nullptr : met,
                compact ? place : nullptr, row_ids, count, long_runs, bad_index};
    FG_TRY(group_tokens(g, s));
  } else if (n > 0) {
    FG_CUDA_TRY(cudaMemsetAsync(long_runs, 0, sizeof(uint32_t), s));
    for (int p = 0; p < passes; ++p) {
      const uint32_t* k = p ? key[(p + 1) & 1] : nullptr;
      sort_count_kernel<<<unsigned(tiles), kSortThreads, 0, s>>>(ids, k, n, vocab, padding, p * digit, digit, counts, bad_index);
      scan_kernel<<<1, kScanThreads, 0, s>>>(counts, tiles << digit, nullptr);
      sort_move_kernel<<<unsigned(tiles), kSortThreads, 0, s>>>(ids, k, p ? pos[(p + 1) & 1] : nullptr, n, vocab, padding,
                                                               p * digit, digit, counts, key[p & 1], pos[p & 1], bad_index);
    }
  }
  a.keys = key[grouped_here ? 0 : (passes - 1) & 1];
  a.pos = pos[grouped_here ? 0 : (passes - 1) & 1];
  a.n = n;
  a.vocab = vocab;
  a.dim = int(dim);
  a.ldy = ldy;
  a.ldg = ldg;
  a.scale = scale;
  a.accumulate = accumulate;
  if (compact) a.place = place;
  if (compact && !grouped_here) {
    heads_count_kernel<<<unsigned(tiles), kSortThreads, 0, s>>>(a.keys, n, vocab, counts);
    scan_kernel<<<1, kScanThreads, 0, s>>>(counts, tiles, count);
    heads_place_kernel<<<unsigned(tiles), kSortThreads, 0, s>>>(a.keys, n, vocab, counts, place, row_ids);
    rest_ids_kernel<<<unsigned(blocks_of(n, 256)), 256, 0, s>>>(row_ids, n, count);
  }
  FG_CUDA_TRY(cudaGetLastError());
  a.chunk = chunk;
  a.slices = slices;
  a.rows = compact ? n : vocab;
  a.count = count;
  const int64_t sum_blocks = blocks_of(chunks * blocks_of(slices, wide ? 1 : kNarrowParts), kSumWarps);
  const int64_t all_zero_blocks = accumulate ? 0 : blocks_of(blocks_of(a.rows, 32) * (wide ? slices : 1), kSumWarps);
  const int64_t zero_blocks = zeros_first ? 0 : all_zero_blocks;
  if (sum_blocks + zero_blocks > INT32_MAX) return set_error(FG_EINVAL, "embedding gradient: too many tokens times columns");
  if (sum_blocks + zero_blocks == 0) return FG_OK;
  a.sum_blocks = int(sum_blocks);
  a.zero_blocks = int(zero_blocks);
  const unsigned threads = kSumWarps * 32, blocks = unsigned(sum_blocks + zero_blocks);
  // as many blocks as there may be long runs, up to two rounds of the SMs' blocks
  const unsigned join_blocks = unsigned(std::min<int64_t>(blocks_of(n / (chunk + 1), kSumWarps) * a.slices, int64_t(sm_count()) * 6));
  return by_dtype(grad_dtype, [&](auto tg) {
    using TG = typename decltype(tg)::type;
    TG* g = static_cast<TG*>(grad);
    if (zeros_first)
      FG_TRY(launch_after(wide ? zero_kernel<TG, 4> : zero_kernel<TG, 1>, unsigned(all_zero_blocks), threads, s, a, g));
    FG_TRY(by_dtype(dy_dtype, [&](auto ty) {
      using TY = typename decltype(ty)::type;
      return launch_after(wide ? sum_kernel<TY, TG, 4, 1> : sum_kernel<TY, TG, 1, kNarrowParts>, blocks, threads, s, a,
                          static_cast<const TY*>(dy), g);
    }));
    if (n <= chunk) return FG_OK;
    return launch_after(wide ? join_kernel<TG, 4> : join_kernel<TG, 1>, join_blocks, threads, s, a, g);
  });
}

// The refusals both gradients share.
int check_grad(const char* op, const void* dy, int dy_dtype, int64_t ldy, const int32_t* ids, int64_t n, int64_t vocab,
               int64_t dim, const void* grad, int grad_dtype, int64_t ldg, int64_t rows) {
  if (n < 0 || vocab < 0 || dim <= 0 || n >= INT32_MAX || vocab >= INT32_MAX || dim > (1 << 20))
    return set_error(FG_EINVAL, "%s: bad shape n=%lld vocab=%lld dim=%lld", op, (long long)n, (long long)vocab, (long long)dim);
  if (!known_dtype(dy_dtype) || !known_dtype(grad_dtype))
    return set_error(FG_EINVAL, "%s: unknown element type %d or %d", op, dy_dtype, grad_dtype);
  if (ldy < dim || ldg < dim) return set_error(FG_EINVAL, "%s: leading dimension smaller than the row", op);
  if (n > 0 && (!dy || !ids)) return set_error(FG_EINVAL, "%s: null operand", op);
  if (!grad && rows > 0) return set_error(FG_EINVAL, "%s: null operand", op);
  return FG_OK;
}

}  // namespace

}  // namespace fg

using namespace fg;

extern "C" {

int fg_embedding(const void* table, int table_dtype, int64_t vocab, int64_t dim, int64_t ldt, const int32_t* ids,
                 int64_t n, float scale, int padding, void* out, int out_dtype, int64_t ldo, void* stream) {
  clear_error();
  if (n < 0 || vocab < 0 || dim <= 0 || n >= INT32_MAX || vocab >= INT32_MAX || dim > (1 << 20))
    return set_error(FG_EINVAL, "fg_embedding: bad shape n=%lld vocab=%lld dim=%lld", (long long)n, (long long)vocab, (long long)dim);
  if (!known_dtype(table_dtype) || !known_dtype(out_dtype))
    return set_error(FG_EINVAL, "fg_embedding: unknown element type %d or %d", table_dtype, out_dtype);
  if (ldt < dim || ldo < dim) return set_error(FG_EINVAL, "fg_embedding: leading dimension smaller than the row");
  if (n == 0) return FG_OK;
  if (!ids || !out || (!table && vocab > 0)) return set_error(FG_EINVAL, "fg_embedding: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int* bad_index = nullptr;
  FG_TRY(device_index_word(&bad_index));
  const unsigned blocks = unsigned(blocks_of(n, kLookupWarps));
  const bool wide = grouped(table, table_dtype, dim, ldt, 4) && grouped(out, out_dtype, dim, ldo, 4);
  return by_dtype(table_dtype, [&](auto tw) {
    return by_dtype(out_dtype, [&](auto ty) {
      using TW = typename decltype(tw)::type;
      using TY = typename decltype(ty)::type;
      const TW* w = static_cast<const TW*>(table);
      TY* y = static_cast<TY*>(out);
      if (wide)
        lookup_kernel<TW, TY, 4><<<blocks, kLookupWarps * 32, 0, s>>>(w, vocab, int(dim), ldt, ids, n, scale, padding, y, ldo, bad_index);
      else
        lookup_kernel<TW, TY, 1><<<blocks, kLookupWarps * 32, 0, s>>>(w, vocab, int(dim), ldt, ids, n, scale, padding, y, ldo, bad_index);
      FG_CUDA_TRY(cudaGetLastError());
      return FG_OK;
    });
  });
}

int fg_embedding_grad(const void* dy, int dy_dtype, int64_t ldy, const int32_t* ids, int64_t n, int64_t vocab,
                      int64_t dim, float scale, int padding, void* grad, int grad_dtype, int64_t ldg, int accumulate,
                      void* stream) {
  clear_error();
  FG_TRY(check_grad("fg_embedding_grad", dy, dy_dtype, ldy, ids, n, vocab, dim, grad, grad_dtype, ldg, vocab));
  if (vocab == 0 && n == 0) return FG_OK;
  return embedding_grad(dy, dy_dtype, ldy, ids, n, vocab, dim, scale, padding, grad, grad_dtype, ldg, accumulate != 0,
                        nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

int fg_embedding_grad_rows(const void* dy, int dy_dtype, int64_t ldy, const int32_t* ids, int64_t n, int64_t vocab,
                           int64_t dim, float scale, int padding, int32_t* row_ids, void* rows, int rows_dtype,
                           int64_t ldr, int32_t* count, void* stream) {
  clear_error();
  FG_TRY(check_grad("fg_embedding_grad_rows", dy, dy_dtype, ldy, ids, n, vocab, dim, rows, rows_dtype, ldr, n));
  if (!count || (!row_ids && n > 0)) return set_error(FG_EINVAL, "fg_embedding_grad_rows: null operand");
  return embedding_grad(dy, dy_dtype, ldy, ids, n, vocab, dim, scale, padding, rows, rows_dtype, ldr, 0, row_ids, count,
                        static_cast<cudaStream_t>(stream));
}

}  // extern "C"
