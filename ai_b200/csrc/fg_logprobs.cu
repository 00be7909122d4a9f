// Log probabilities of given columns of rows of logits, with each row's
// entropy and its most probable columns, and the gradient.
//
//   z_j = scale·x_j, m = max_j z_j, s1 = Σ e^(z_j − m), s2 = Σ e^(z_j − m)·(z_j − m)
//   logprob = z_t − m − log s1,  H = log s1 − s2 / s1,  lse = m + log s1
//   dx_j = scale·(g·([j = t] − p_j) − h·p_j·(log p_j + H)),  p_j = e^(z_j − lse)
//
// A row whose entries are all −∞ has log probabilities −∞, entropy 0 and
// gradient 0; a row with a NaN or a +∞ has NaN in all of them.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fg_internal.h"
#include "fg_ptx.cuh"
#include "fg_types.cuh"

namespace fg {

namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxTop = FG_MAX_TOP;
constexpr unsigned kFull = 0xffffffffu;

// Order of the alternatives as one number: the value (NaN above +∞, −0 as
// 0) in the upper half, the lower index above the higher one in the lower.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  if (x != x) u = 0x7fc00000u;
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return uint64_t(u) << 32 | (0xffffffffu - index);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
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

// One block per row: the maximum, the sums, then one pass per alternative.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprobs_kernel(LogProbsArgs a, const T* __restrict__ logits) {
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float part[3][kWarps];
  __shared__ uint64_t best[kWarps];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * a.ld;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.width; j += kRowThreads) m = fmaxf(m, widen(x[j]));
  m = warp_max(m);
  if (lane == 0) part[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, part[0][w]);
  const bool empty = m == -INFINITY;
  const float m0 = empty ? 0.f : m;
  float s1 = 0.f, s2 = 0.f, bad = 0.f;
  for (int j = threadIdx.x; j < a.width; j += kRowThreads) {
    const float d = (widen(x[j]) - m0) * a.scale;
    const float e = __expf(d);
    s1 += e;
    s2 += e == 0.f ? 0.f : e * d;
    if (widen(x[j]) != widen(x[j])) bad = 1.f;
  }
  s1 = warp_sum(s1);
  s2 = warp_sum(s2);
  bad = warp_max(bad);
  if (lane == 0) {
    part[1][warp] = s1;
    part[2][warp] = s2;
  }
  const bool any_bad = __syncthreads_or(bad != 0.f);
  s1 = s2 = 0.f;
  for (int w = 0; w < kWarps; ++w) {
    s1 += part[1][w];
    s2 += part[2][w];
  }
  const bool void_row = empty && !any_bad;
  const float logs = logf(s1);
  if (threadIdx.x == 0) {
    const int t = a.targets[row];
    const bool none = t < 0 || t >= a.width;
    if (t >= a.width) atomicCAS(a.err, 0, kDevBadIndex);
    a.logprob[row] = none ? 0.f : void_row ? -INFINITY : (widen(x[t]) - m0) * a.scale - logs;
    a.entropy[row] = void_row ? 0.f : logs - s2 / s1;
    a.lse[row] = m0 * a.scale + logs;
  }
  uint64_t last = ~uint64_t(0);
  for (int k = 0; k < a.top; ++k) {
    uint64_t mine = 0;
    for (int j = threadIdx.x; j < a.width; j += kRowThreads) {
      const uint64_t key = rank_key(widen(x[j]), j);
      if (key < last && key > mine) mine = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t u = __shfl_xor_sync(kFull, mine, o);
      mine = u > mine ? u : mine;
    }
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    if (threadIdx.x == 0) {
      const uint32_t j = 0xffffffffu - uint32_t(mine);
      a.top_index[row * a.top + k] = int32_t(j);
      a.top_logprob[row * a.top + k] = void_row ? -INFINITY : (widen(x[j]) - m0) * a.scale - logs;
    }
    __syncthreads();
  }
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

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprobs_grad_kernel(LogProbsGradArgs a, const T* logits, T* dlogits) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * a.ld;
  T* dx = dlogits + row * a.ldd;
  const int t = a.targets[row];
  if (t >= a.width && threadIdx.x == 0) atomicCAS(a.err, 0, kDevBadIndex);
  const bool none = t < 0 || t >= a.width;
  const float lse = a.lse[row];
  const float g = none ? 0.f : a.dlogprob[row];
  const float h = a.dentropy ? a.dentropy[row] : 0.f, H = a.dentropy ? a.entropy[row] : 0.f;
  const bool empty = lse == -INFINITY;
  for (int j = threadIdx.x; j < a.width; j += kRowThreads) {
    float d = 0.f;
    if (!empty) {
      const float lp = fmaf(widen(x[j]), a.scale, -lse);
      const float p = __expf(lp);
      d = g * ((j == t ? 1.f : 0.f) - p);
      if (a.dentropy && p != 0.f) d -= h * p * (lp + H);
      d *= a.scale;
    }
    dx[j] = narrow<T>(d);
  }
}

}  // namespace

}  // namespace fg

using namespace fg;

extern "C" {

int fg_log_probs(const void* logits, int dtype, int64_t rows, int64_t width, int64_t ld, const int32_t* targets,
                 float scale, int top, float* logprob, float* entropy, float* lse, int32_t* top_index,
                 float* top_logprob, void* stream) {
  clear_error();
  if (rows < 0 || width <= 0 || rows >= INT32_MAX || width >= INT32_MAX)
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
    logprobs_kernel<T><<<unsigned(rows), kRowThreads, 0, s>>>(a, static_cast<const T*>(logits));
    FG_CUDA_TRY(cudaGetLastError());
    return FG_OK;
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
    logprobs_grad_kernel<T><<<unsigned(rows), kRowThreads, 0, s>>>(a, static_cast<const T*>(logits), static_cast<T*>(dlogits));
    FG_CUDA_TRY(cudaGetLastError());
    return FG_OK;
  });
}

}  // extern "C"
