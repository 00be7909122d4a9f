// The global norm of many gradients, and their clipping by it:
//
//   N = sqrt(Σ_i ‖g_i‖²),  out_i = c·g_i,  c = max_norm / N if max_norm < N < ∞, else 1
//
// N < ∞ is asked of the float32 that the caller gets, so that what it reads and
// what was done agree.
// Two passes over memory: a block sums the squares of its share of equal
// pieces and leaves one partial sum; every block of the second pass adds all
// partial sums in one order, so all have the same c, and scales its share,
// from the last piece to the first: what the first pass read last is still
// in L2. Bound by memory. Squares are added four or eight at a time in 32
// bits and these sums in 64 (squaring in 64 bits alone took 299 us for 302 M
// values, of 185 us for their bytes); where a thread's sum of a piece may have
// overflowed or lost small squares, it squares its values again in 64 bits, so
// that no gradient is too large or too small. 302 M fp32 values clipped into
// other buffers: 580 us, 6.3 TB/s of the three passes over memory that they
// need (1.2 GB do not stay on the chip between the two reads).
// The tensors' addresses travel in the kernel's arguments: no copy to the
// device, whatever their number.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fg_internal.h"
#include "fg_launch.cuh"
#include "fg_types.cuh"

namespace fg {

namespace {

constexpr int kNormThreads = 256;
constexpr int kPiece = 8192;      // values of a tensor that a block takes at once
constexpr int kFewTensors = 64;    // of a small call's launch: arguments are copied at every launch
constexpr int kMaxTensors = 1000;  // of a launch: 29 bytes each within the 32764 of a kernel's arguments

template <int N>
struct TensorList {
  const void* in[N];
  void* out[N];
  int64_t size[N];
  int first[N + 1];  // pieces before tensor i
  uint8_t dtype[N];
  int count;
};

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
  for (int w = 0; w < kNormThreads / 32; ++w) s += shared[w];
  __syncthreads();
  return s;
}

// The tensor a piece belongs to.
template <int N>
__device__ __forceinline__ int tensor_of(const TensorList<N>& t, int piece) {
  int lo = 0, hi = t.count;  // first[lo] <= piece < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= piece)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Calls f(offset in values, Pack) for the 16-byte groups of x's n values and
// g(offset) for the values before and after them. Whole pieces are loaded
// AHEAD groups a thread at a time.
template <int AHEAD, typename T, typename F, typename G>
__device__ __forceinline__ void for_groups(const T* x, int n, const F& f, const G& g) {
  constexpr int V = 16 / int(sizeof(T));
  const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  if (head == 0 && n == kPiece) {
    const int at = threadIdx.x * V;
#pragma unroll 1
    for (int i = at; i < kPiece; i += AHEAD * kNormThreads * V) {
      Pack<T, V> p[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) p[u].load_own(x + i + u * kNormThreads * V);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) f(i + u * kNormThreads * V, p[u]);
    }
    return;
  }
  const int groups = (n - head) / V, tail = head + groups * V;
#pragma unroll 1
  for (int i = threadIdx.x; i < groups; i += kNormThreads) {
    Pack<T, V> p;
    p.load_own(x + head + i * V);
    f(head + i * V, p);
  }
#pragma unroll 1
  for (int i = threadIdx.x; i < head + n - tail; i += kNormThreads) g(i < head ? i : tail + i - head);
}

template <typename T>
__device__ __forceinline__ double squares(const T* x, int n) {
  constexpr int V = 16 / int(sizeof(T));
  double sum = 0;
  uint32_t any = 0;  // bits of the values but their signs
  for_groups<4>(
      x, n,
      [&](int, const auto& p) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(p.get(j), p.get(j), s);
        any |= (p.part[0].x | p.part[0].y | p.part[0].z | p.part[0].w) & (V == 4 ? 0x7fffffffu : 0x7fff7fffu);
        sum += double(s);
      },
      [&](int i) {
        sum = fma(double(widen(x[i])), double(widen(x[i])), sum);
        any |= widen(x[i]) != 0.f;
      });
  if (any && !(sum > 0x1p-60 && sum < 0x1p+120)) {
    sum = 0;
    auto again = [&](int i) { sum = fma(double(widen(x[i])), double(widen(x[i])), sum); };
    for_groups<1>(
        x, n,
        [&](int i, const auto&) {
#pragma unroll 1
          for (int j = 0; j < V; ++j) again(i + j);
        },
        again);
  }
  return sum;
}

// C: float, or double for a factor below float's normal numbers, which has
// lost bits as a float.
template <typename T, typename C>
__device__ __forceinline__ void scale_piece(const T* x, T* y, int n, C c) {
  constexpr int V = 16 / int(sizeof(T));
  constexpr int kAheadOf = sizeof(C) == 4 ? 4 : 1;
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  for_groups<kAheadOf>(
      x, n,
      [&](int i, auto& p) {
#pragma unroll
        for (int j = 0; j < V; ++j) p.set(j, float(p.get(j) * c));
        if (alike) {
          p.store(y + i);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) y[i + j] = p.v[j];
        }
      },
      [&](int i) { y[i] = narrow<T>(float(widen(x[i]) * c)); });
}

// Piece `at` of a tensor, n of its values.
template <int N, typename C>
__device__ __forceinline__ void scale_any(const TensorList<N>& t, int i, int64_t at, int n, C c) {
  if (t.dtype[i] == FG_DT_F32)
    scale_piece(static_cast<const float*>(t.in[i]) + at, static_cast<float*>(t.out[i]) + at, n, c);
  else if (t.dtype[i] == FG_DT_BF16)
    scale_piece(static_cast<const __nv_bfloat16*>(t.in[i]) + at, static_cast<__nv_bfloat16*>(t.out[i]) + at, n, c);
  else
    scale_piece(static_cast<const __half*>(t.in[i]) + at, static_cast<__half*>(t.out[i]) + at, n, c);
}

template <int N>
__global__ void __launch_bounds__(kNormThreads, 8) squares_kernel(const __grid_constant__ TensorList<N> t, double* partial) {
  __shared__ double shared[kNormThreads / 32];
  double s = 0;
  for (int piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int i = tensor_of(t, piece);
    const int64_t at = int64_t(piece - t.first[i]) * kPiece;
    const int n = int(min(int64_t(kPiece), t.size[i] - at));
    if (t.dtype[i] == FG_DT_F32)
      s += squares(static_cast<const float*>(t.in[i]) + at, n);
    else if (t.dtype[i] == FG_DT_BF16)
      s += squares(static_cast<const __nv_bfloat16*>(t.in[i]) + at, n);
    else
      s += squares(static_cast<const __half*>(t.in[i]) + at, n);
  }
  s = block_sum(s, shared);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <int N>
__global__ void __launch_bounds__(kNormThreads, 4) clip_kernel(const __grid_constant__ TensorList<N> t,
                                                           const double* partial, int partials,
                                                           float max_norm, float* norm) {
  __shared__ double shared[kNormThreads / 32];
  wait_for_previous();
  double s = 0;
  for (int i = threadIdx.x; i < partials; i += kNormThreads) s += __ldcg(partial + i);
  const double total = sqrt(block_sum(s, shared));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(total);
  const bool clips = total > double(max_norm) && isfinite(float(total));
  const double factor = clips ? double(max_norm) / total : 1.0;
  const float c = float(factor);
  const bool small = factor > 0.0 && c < FLT_MIN;
  for (int piece = t.first[t.count] - 1 - blockIdx.x; piece >= 0; piece -= gridDim.x) {
    const int i = tensor_of(t, piece);
    if (!clips && t.in[i] == t.out[i]) continue;
    const int64_t at = int64_t(piece - t.first[i]) * kPiece;
    const int n = int(min(int64_t(kPiece), t.size[i] - at));
    if (small)
      scale_any(t, i, at, n, factor);
    else
      scale_any(t, i, at, n, c);
  }
}

template <int N>
int clip_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, void* const* outs,
                   float max_norm, float* norm, cudaStream_t s) {
  const int launches = std::max(1, (count + N - 1) / N);
  const int most = sm_count() * 8;  // blocks of a launch
  void* ws = nullptr;
  FG_TRY(scratch_alloc(&ws, size_t(launches) * most * sizeof(double), s));
  double* partial = static_cast<double*>(ws);
  int rc = FG_OK, partials = 0;
  TensorList<N> t;
  // the tensors of launch l; the number of its blocks
  auto list = [&](int l) {
    t.count = 0;
    t.first[0] = 0;
    for (int i = l * N; i < std::min(count, (l + 1) * N); ++i) {
      t.in[t.count] = grads[i];
      t.out[t.count] = outs ? outs[i] : const_cast<void*>(grads[i]);
      t.size[t.count] = sizes[i];
      t.dtype[t.count] = uint8_t(dtypes[i]);
      t.first[t.count + 1] = t.first[t.count] + int((sizes[i] + kPiece - 1) / kPiece);
      ++t.count;
    }
    return std::max(1, std::min(most, t.first[t.count]));
  };
  for (int l = 0; l < launches && rc == FG_OK; ++l) {
    const int blocks = list(l);
    squares_kernel<<<blocks, kNormThreads, 0, s>>>(t, partial + partials);
    partials += blocks;
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess)
      rc = set_error(FG_ECUDA, "fg_clip_grad_norm: %s", cudaGetErrorString(e));
  }
  for (int l = launches - 1; l >= 0 && rc == FG_OK; --l) {
    const int blocks = launches > 1 ? list(l) : std::max(1, std::min(most, t.first[t.count]));
    rc = launch_after(clip_kernel<N>, blocks, kNormThreads, s, t, partial, partials, max_norm, l == 0 ? norm : nullptr);
  }
  scratch_free(ws, s);
  return rc;
}

}  // namespace

}  // namespace fg

using namespace fg;

extern "C" {

int fg_clip_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, void* const* outs,
                      float max_norm, float* norm, void* stream) {
  clear_error();
  if (count < 0 || (count > 0 && (!grads || !sizes || !dtypes))) return set_error(FG_EINVAL, "fg_clip_grad_norm: bad tensor list");
  if (!(max_norm >= 0.f)) return set_error(FG_EINVAL, "fg_clip_grad_norm: max_norm must be at least 0");
  if (!norm) return set_error(FG_EINVAL, "fg_clip_grad_norm: null norm");
  int64_t pieces = 0;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0 || (pieces += sizes[i] / kPiece + 1) > INT32_MAX / 2) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d has %lld values", i, (long long)sizes[i]);
    if (!known_dtype(dtypes[i])) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d has unknown element type %d", i, dtypes[i]);
    if (sizes[i] > 0 && (!grads[i] || (outs && !outs[i]))) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d is null", i);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (count <= kFewTensors) return clip_grad_norm<kFewTensors>(count, grads, sizes, dtypes, outs, max_norm, norm, s);
  return clip_grad_norm<kMaxTensors>(count, grads, sizes, dtypes, outs, max_norm, norm, s);
}

}  // extern "C"
