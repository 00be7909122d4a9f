// The global norm of many gradients, and their clipping by it:
//
//   N = sqrt(Σ_i ‖g_i‖²),  out_i = c·g_i,  c = max_norm / N if max_norm < N < ∞, else 1
//
// Two passes over memory: a block sums the squares of its share of equal
// pieces in 64 bits (no gradient is too large or too small for its square)
// and leaves one partial sum; every block of the second pass adds all
// partial sums in one order, so all have the same c, and scales its share.
// The tensors' addresses travel in the kernel's arguments: no copy to the
// device, whatever their number.
#include <algorithm>
#include <cmath>

#include "fg_internal.h"
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

template <typename T>
__device__ __forceinline__ double squares(const T* x, int64_t n) {
  constexpr int V = 16 / int(sizeof(T));
  double s = 0;
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
    const int64_t groups = n / V;
    for (int64_t i = threadIdx.x; i < groups; i += kNormThreads) {
      Pack<T, V> p;
      p.load(x + i * V);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fma(double(p.get(j)), double(p.get(j)), s);
    }
    for (int64_t i = groups * V + threadIdx.x; i < n; i += kNormThreads) s = fma(double(widen(x[i])), double(widen(x[i])), s);
  } else {
    for (int64_t i = threadIdx.x; i < n; i += kNormThreads) s = fma(double(widen(x[i])), double(widen(x[i])), s);
  }
  return s;
}

template <typename T>
__device__ __forceinline__ void scale_piece(const T* x, T* y, int64_t n, float c) {
  constexpr int V = 16 / int(sizeof(T));
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
    const int64_t groups = n / V;
    for (int64_t i = threadIdx.x; i < groups; i += kNormThreads) {
      Pack<T, V> p;
      p.load_own(x + i * V);
#pragma unroll
      for (int j = 0; j < V; ++j) p.set(j, p.get(j) * c);
      p.store(y + i * V);
    }
    for (int64_t i = groups * V + threadIdx.x; i < n; i += kNormThreads) y[i] = narrow<T>(widen(x[i]) * c);
  } else {
    for (int64_t i = threadIdx.x; i < n; i += kNormThreads) y[i] = narrow<T>(widen(x[i]) * c);
  }
}

template <int N>
__global__ void __launch_bounds__(kNormThreads) squares_kernel(const __grid_constant__ TensorList<N> t, double* partial) {
  __shared__ double shared[kNormThreads / 32];
  double s = 0;
  for (int piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int i = tensor_of(t, piece);
    const int64_t at = int64_t(piece - t.first[i]) * kPiece;
    const int64_t n = min(int64_t(kPiece), t.size[i] - at);
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
__global__ void __launch_bounds__(kNormThreads) clip_kernel(const __grid_constant__ TensorList<N> t,
                                                           const double* __restrict__ partial, int partials,
                                                           float max_norm, float* norm) {
  __shared__ double shared[kNormThreads / 32];
  double s = 0;
  for (int i = threadIdx.x; i < partials; i += kNormThreads) s += partial[i];
  const double total = sqrt(block_sum(s, shared));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(total);
  const bool clips = total > double(max_norm) && isfinite(total);
  const float c = clips ? float(double(max_norm) / total) : 1.f;
  for (int piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int i = tensor_of(t, piece);
    if (!clips && t.in[i] == t.out[i]) continue;
    const int64_t at = int64_t(piece - t.first[i]) * kPiece;
    const int64_t n = min(int64_t(kPiece), t.size[i] - at);
    if (t.dtype[i] == FG_DT_F32)
      scale_piece(static_cast<const float*>(t.in[i]) + at, static_cast<float*>(t.out[i]) + at, n, c);
    else if (t.dtype[i] == FG_DT_BF16)
      scale_piece(static_cast<const __nv_bfloat16*>(t.in[i]) + at, static_cast<__nv_bfloat16*>(t.out[i]) + at, n, c);
    else
      scale_piece(static_cast<const __half*>(t.in[i]) + at, static_cast<__half*>(t.out[i]) + at, n, c);
  }
}

template <int N>
int clip_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, void* const* outs,
                   float max_norm, float* norm, cudaStream_t s) {
  const int launches = std::max(1, (count + N - 1) / N);
  const int blocks = sm_count() * 8;
  void* ws = nullptr;
  FG_TRY(scratch_alloc(&ws, size_t(launches) * blocks * sizeof(double), s));
  double* partial = static_cast<double*>(ws);
  int rc = FG_OK;
  for (int pass = 0; pass < 2 && rc == FG_OK; ++pass) {
    for (int l = 0; l < launches && rc == FG_OK; ++l) {
      TensorList<N> t;
      t.count = 0;
      t.first[0] = 0;
      for (int i = l * N; i < std::min(count, (l + 1) * N); ++i) {
        t.in[t.count] = grads[i];
        t.out[t.count] = outs ? outs[i] : const_cast<void*>(grads[i]);
        t.size[t.count] = sizes[i];
        t.dtype[t.count] = uint8_t(dtypes[i]);
        const int64_t next = t.first[t.count] + (sizes[i] + kPiece - 1) / kPiece;
        if (next > INT32_MAX / 2) {
          rc = set_error(FG_EINVAL, "fg_clip_grad_norm: too many values");
          break;
        }
        t.first[++t.count] = int(next);
      }
      if (rc != FG_OK) break;
      if (pass == 0)
        squares_kernel<<<blocks, kNormThreads, 0, s>>>(t, partial + l * blocks);
      else
        clip_kernel<<<blocks, kNormThreads, 0, s>>>(t, partial, launches * blocks, max_norm, l == 0 ? norm : nullptr);
      if (cudaError_t e = cudaGetLastError(); e != cudaSuccess)
        rc = set_error(FG_ECUDA, "fg_clip_grad_norm: %s", cudaGetErrorString(e));
    }
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
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] / kPiece > (1 << 28)) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d has %lld values", i, (long long)sizes[i]);
    if (!known_dtype(dtypes[i])) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d has unknown element type %d", i, dtypes[i]);
    if (sizes[i] > 0 && (!grads[i] || (outs && !outs[i]))) return set_error(FG_EINVAL, "fg_clip_grad_norm: tensor %d is null", i);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (count <= kFewTensors) return clip_grad_norm<kFewTensors>(count, grads, sizes, dtypes, outs, max_norm, norm, s);
  return clip_grad_norm<kMaxTensors>(count, grads, sizes, dtypes, outs, max_norm, norm, s);
}

}  // extern "C"
