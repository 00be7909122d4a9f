// Values of 32 or 16 bits in memory, 32 bits in registers: vector loads and
// stores of the element types the training operators take (FG_DT_*), and
// the dispatch from a type code to a template argument.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fg_internal.h"

namespace fg {

template <typename T>
struct TypeTag {
  using type = T;
};

// f(TypeTag<T>{}) for the element type of a FG_DT_* code.
template <typename F>
int by_dtype(int dt, const F& f) {
  switch (dt) {
    case FG_DT_F32: return f(TypeTag<float>{});
    case FG_DT_BF16: return f(TypeTag<__nv_bfloat16>{});
    case FG_DT_F16: return f(TypeTag<__half>{});
  }
  return set_error(FG_EINVAL, "unknown element type %d", dt);
}

inline bool known_dtype(int dt) { return dt == FG_DT_F32 || dt == FG_DT_BF16 || dt == FG_DT_F16; }
inline int64_t dtype_size(int dt) { return dt == FG_DT_F32 ? 4 : 2; }

// The bits of N consecutive values.
template <int BYTES>
struct Bits;
template <>
struct Bits<2> {
  uint16_t w;
};
template <>
struct Bits<4> {
  uint32_t w;
};
template <>
struct Bits<8> {
  uint2 w;
};
template <>
struct Bits<16> {
  uint4 w;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half narrow<__half>(float x) {
  return __float2half_rn(x);
}

// N values in their memory form: loaded together before they are widened,
// so that several can be in flight at the cost of their bytes.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = int(sizeof(T)) * N;
  static constexpr int kParts = kBytes > 16 ? kBytes / 16 : 1;
  using Part = decltype(Bits<kBytes / kParts>::w);
  union {
    Part part[kParts];
    T v[N];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) part[i] = __ldg(reinterpret_cast<const Part*>(p) + i);
  }
  // from memory that the kernel also writes
  __device__ __forceinline__ void load_own(const T* p) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) part[i] = reinterpret_cast<const Part*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kParts; ++i) reinterpret_cast<Part*>(p)[i] = part[i];
  }
  // not to be read again soon
  __device__ __forceinline__ void store_past(T* p) const {
#pragma unroll
    for (int i = 0; i < kParts; ++i) __stcs(reinterpret_cast<Part*>(p) + i, part[i]);
  }
  __device__ __forceinline__ float get(int i) const { return widen(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = narrow<T>(x); }
};

}  // namespace fg
