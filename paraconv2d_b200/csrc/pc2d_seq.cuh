// Shared pieces of the sequence operators (dropout, causal convolution, state
// space scan): element types, vector loads and the argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "pc2d_common.cuh"

namespace pc2d {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements of T held in registers, loaded and stored by the widest vectors
// (at most 16 bytes) that divide them.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = (int)sizeof(T) * N;
  static constexpr int kVec = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
  alignas(kVec) T v[N];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kVec == 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4 *>(v)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else if constexpr (kVec == 8) {
#pragma unroll
      for (int i = 0; i < kBytes / 8; ++i)
        reinterpret_cast<uint2 *>(v)[i] = __ldg(reinterpret_cast<const uint2 *>(p) + i);
    } else if constexpr (kVec == 4) {
#pragma unroll
      for (int i = 0; i < kBytes / 4; ++i)
        reinterpret_cast<unsigned *>(v)[i] = __ldg(reinterpret_cast<const unsigned *>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (kVec == 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(v)[i];
    } else if constexpr (kVec == 8) {
#pragma unroll
      for (int i = 0; i < kBytes / 8; ++i)
        reinterpret_cast<uint2 *>(p)[i] = reinterpret_cast<const uint2 *>(v)[i];
    } else if constexpr (kVec == 4) {
#pragma unroll
      for (int i = 0; i < kBytes / 4; ++i)
        reinterpret_cast<unsigned *>(p)[i] = reinterpret_cast<const unsigned *>(v)[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = v[i];
    }
  }
  __device__ __forceinline__ float f(int i) const { return to_f(v[i]); }
  // all N (even) at once: the 16-bit types round two per instruction
  __device__ __forceinline__ void set(const float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = x[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        if constexpr (std::is_same<T, __half>::value)
          *reinterpret_cast<__half2 *>(v + i) = __floats2half2_rn(x[i], x[i + 1]);
        else
          *reinterpret_cast<__nv_bfloat162 *>(v + i) = __floats2bfloat162_rn(x[i], x[i + 1]);
      }
    }
  }
};

// 1 / (1 + exp(-v)): 0 and 1 at the infinities.  The two hardware functions and
// the argument's rounding leave it off by 4 + |v| units of 2^-24 where v < 0, less
// elsewhere.
__device__ __forceinline__ float sigmoid_f(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// Element types the sequence operators take.
inline bool seq_dtype(int dtype) {
  return dtype == PC2D_DTYPE_F32 || dtype == PC2D_DTYPE_F16 || dtype == PC2D_DTYPE_BF16;
}
inline size_t seq_dtype_size(int dtype) { return dtype == PC2D_DTYPE_F32 ? 4 : 2; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Arrays that are read element by element: each on a boundary of its elements,
// off which any access faults.
inline int check_elements(const char *what, size_t bytes, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) {
      set_last_error("%s: an array of %zu-byte elements is not aligned to them", what, bytes);
      return PC2D_ERR_INVALID_ARGUMENT;
    }
  return PC2D_OK;
}

// Where a single-token step finds the state of batch row b: slots[b] of the
// `places` rows of the state array, or row b without slots.  -1: the row is
// padding (its output is 0).  A place outside the array, and one that an
// earlier row has already, cannot be served: the output is NaN and no state
// is touched, so that the mistake is seen and the result does not depend on
// which of two blocks came first.
//
// step_place gives a place that may be read (0 for rows that have none);
// step_twice, whether this thread's share of the earlier rows has it too; and
// step_served, which the whole block calls after its reads are on their way,
// whether it may be written.
enum StepKind { kStepServed, kStepPadding, kStepBad };
__device__ __forceinline__ int step_place(const int *slots, int b, int places, StepKind *kind) {
  const int place = slots ? slots[b] : b;
  *kind = place == -1 ? kStepPadding : place < 0 || place >= places ? kStepBad : kStepServed;
  return *kind == kStepServed ? place : 0;
}
__device__ __forceinline__ int step_twice(const int *slots, int b, int place, StepKind kind) {
  int twice = 0;
  if (slots && kind == kStepServed)
    for (int i = threadIdx.x; i < b; i += blockDim.x) twice |= slots[i] == place;
  return twice;
}
__device__ __forceinline__ StepKind step_served(int twice, StepKind kind) {
  return __syncthreads_or(twice) ? kStepBad : kind;
}
__device__ __forceinline__ float step_nothing(StepKind kind) {
  return kind == kStepBad ? __int_as_float(0x7fffffff) : 0.f;
}

}  // namespace pc2d
