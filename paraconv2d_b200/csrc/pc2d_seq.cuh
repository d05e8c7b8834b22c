// Shared pieces of the sequence operators (dropout, causal convolution, state
// space scan): element types, vector loads and the argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
};

// 1 / (1 + exp(-v)): 0 and 1 at the infinities.  __expf and __fdividef are off
// by a few units of the last place, far below the bf16/fp16 rounding and of
// the size of an fp32 sum's own roundings.
__device__ __forceinline__ float sigmoid_f(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

// Element types the sequence operators take.
inline bool seq_dtype(int dtype) {
  return dtype == PC2D_DTYPE_F32 || dtype == PC2D_DTYPE_F16 || dtype == PC2D_DTYPE_BF16;
}
inline size_t seq_dtype_size(int dtype) { return dtype == PC2D_DTYPE_F32 ? 4 : 2; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Where a single-token step finds the state of batch row b: slots[b] of the
// `places` rows of the state array, or row b without slots.  -1: the row is
// padding (its output is 0).  A place outside the array, and one that an
// earlier row has already, cannot be served: the output is NaN and no state
// is touched, so that the mistake is seen and the result does not depend on
// which of two blocks came first.  The whole block calls this.
__device__ __forceinline__ int step_place(const int *slots, int b, int places, bool *bad) {
  *bad = false;
  if (!slots) return b;
  const int place = slots[b];
  if (place == -1) return -1;
  int twice = place < 0 || place >= places;
  for (int i = threadIdx.x; i < b; i += blockDim.x) twice |= slots[i] == place;
  *bad = __syncthreads_or(twice) != 0;
  return *bad ? -1 : place;
}

}  // namespace pc2d
