// Dropout whose mask is never stored: both directions compute it again from a
// counter-based generator, Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011).
//
// Element i of the array takes 16 bits: the counter (i / 8, offset) under the
// key `seed` gives four 32-bit words, which are eight halves, and element i
// takes half i % 8 (the low half of word 0 first).  It is kept when its half
// is at least thr = round(65536 p), and then multiplied by 65536 / (65536 -
// thr), the inverse of the probability with which that happens, so that the
// expectation is exact for the rounded p.  A dropped element is 0 whatever it
// held (NaN too).  The mask depends on seed, offset and i alone: not on the
// type, the launch or the device.
//
// The kernel streams: 4 bytes an element at 16 bits (6 with a residual).
#include <math.h>

#include <algorithm>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace pc2d {
namespace {

// Two vectors in flight per thread and 16 blocks per SM: 66 us (6.1 TB/s) for
// 2^26 bf16 elements with a residual and 52 us (5.2 TB/s) without; one vector
// 65 and 55, four 77 and 54, 8 blocks per SM 69 and 53 us.  With 4 rounds of the
// generator instead of 10 it would be 63 and 42: its 20 wide products and 20
// exclusive-ors for eight elements, with five operations an element, come near
// the time of the traffic.
constexpr int kDropThreads = 256, kDropUnroll = 2, kDropBlocks = 16;

struct Words {
  unsigned w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint64_t seed) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
    c0 = (unsigned)(q >> 32) ^ c1 ^ k0;
    c1 = (unsigned)q;
    c2 = (unsigned)(p >> 32) ^ c3 ^ k1;
    c3 = (unsigned)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

__device__ __forceinline__ double to_acc(double v) { return v; }
template <typename T>
__device__ __forceinline__ float to_acc(T v) { return to_f(v); }
template <typename T, typename A>
__device__ __forceinline__ T from_acc(A v) {
  if constexpr (sizeof(T) == 8) return v;
  else return from_f<T>(v);
}

template <typename T>
struct Acc {
  using type = float;
};
template <>
struct Acc<double> {
  using type = double;
};

template <typename T, bool kResidual>
__device__ __forceinline__ typename Acc<T>::type drop_one(T x, T res, const Words &w, int i, unsigned thr,
                                                          typename Acc<T>::type scale) {
  using A = typename Acc<T>::type;
  // the half in the upper bits against the limit in the upper bits: what lies
  // below an upper half does not change the comparison
  const unsigned half = i & 1 ? w.w[i / 2] : w.w[i / 2] << 16;
  A v = half >= thr << 16 ? to_acc(x) * scale : A(0);
  if (kResidual) v += to_acc(res);
  return v;
}

template <typename T, bool kResidual>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const T *__restrict__ x, const T *__restrict__ res,
                                                              const int64_t *__restrict__ key, unsigned thr,
                                                              typename Acc<T>::type scale, int64_t n, bool vec,
                                                              T *__restrict__ out) {
  const uint64_t seed = (uint64_t)key[0], offset = (uint64_t)key[1];
  const int64_t stride = (int64_t)gridDim.x * kDropThreads;
  const int64_t whole = vec ? n / 8 : 0;  // groups that go by vectors
  for (int64_t g0 = (int64_t)blockIdx.x * kDropThreads + threadIdx.x; g0 < whole; g0 += stride * kDropUnroll) {
    Pack<T, 8> a[kDropUnroll], r[kDropUnroll];
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const int64_t g = g0 + k * stride;
      if (g < whole) {
        a[k].load(x + g * 8);
        if (kResidual) r[k].load(res + g * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const int64_t g = g0 + k * stride;
      if (g < whole) {
        const Words w = philox((uint64_t)g, offset, seed);
        Pack<T, 8> o;
        if constexpr (sizeof(T) == 2) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = drop_one<T, kResidual>(a[k].v[i], r[k].v[i], w, i, thr, scale);
          o.set(v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) o.v[i] = drop_one<T, kResidual>(a[k].v[i], r[k].v[i], w, i, thr, scale);
        }
        o.store(out + g * 8);
      }
    }
  }
  for (int64_t g = whole + (int64_t)blockIdx.x * kDropThreads + threadIdx.x; g * 8 < n; g += stride) {
    const Words w = philox((uint64_t)g, offset, seed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t e = g * 8 + i;
      if (e < n) out[e] = from_acc<T>(drop_one<T, kResidual>(x[e], kResidual ? res[e] : x[e], w, i, thr, scale));
    }
  }
}

__global__ void dropout_next_key_kernel(int64_t *state, int64_t *key) {
  key[0] = state[0];
  key[1] = (int64_t)atomicAdd(reinterpret_cast<unsigned long long *>(state + 1), 1ull);
}

template <typename T>
int launch_dropout(const void *x, const void *res, const int64_t *key, unsigned thr, double scale, int64_t n,
                   void *out, cudaStream_t stream) {
  const bool vec = aligned16(x) && aligned16(out) && (!res || aligned16(res));
  const int64_t blocks = ((n + 7) / 8 + kDropThreads - 1) / kDropThreads;
  const int grid = (int)std::min<int64_t>(blocks, (int64_t)device_sm_count() * kDropBlocks);
  using A = typename Acc<T>::type;
  if (res)
    dropout_kernel<T, true><<<grid, kDropThreads, 0, stream>>>((const T *)x, (const T *)res, key, thr, (A)scale, n,
                                                               vec, (T *)out);
  else
    dropout_kernel<T, false><<<grid, kDropThreads, 0, stream>>>((const T *)x, nullptr, key, thr, (A)scale, n, vec,
                                                                (T *)out);
  PC2D_LAUNCH_CHECK("dropout_kernel");
  return PC2D_OK;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" int pc2d_dropout(int dtype, const void *input, const void *residual, const int64_t *key, double p,
                            int64_t n, void *output, void *stream) {
  NvtxRange range("pc2d_dropout");
  if (!seq_dtype(dtype) && dtype != PC2D_DTYPE_F64) {
    set_last_error("pc2d_dropout: unsupported dtype %d", dtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (!(p >= 0.0 && p <= 1.0)) {
    set_last_error("pc2d_dropout: p must be in [0, 1], got %g", p);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (n < 0) {
    set_last_error("pc2d_dropout: invalid element count %lld", (long long)n);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  int st = pending_device_error();
  if (st != PC2D_OK) return st;
  if (n == 0) return PC2D_OK;
  if (!input || !key || !output) {
    set_last_error("pc2d_dropout: null pointer (input, key or output)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  const size_t size = dtype == PC2D_DTYPE_F64 ? 8 : seq_dtype_size(dtype);
  if ((st = check_elements("pc2d_dropout", size, {input, residual, output})) != PC2D_OK ||
      (st = check_elements("pc2d_dropout", 8, {key})) != PC2D_OK)
    return st;
  // round to even at a half, as Python's round() does
  const unsigned thr = (unsigned)nearbyint(p * 65536.0);
  const double scale = 65536.0 / (65536.0 - thr);  // (not used where every element is dropped)
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (thr == 65536u) {  // every element is dropped (the kernel's limits are below that)
    const size_t bytes = (size_t)n * size;
    if (residual) PC2D_CUDA_CHECK(cudaMemcpyAsync(output, residual, bytes, cudaMemcpyDeviceToDevice, s));
    else PC2D_CUDA_CHECK(cudaMemsetAsync(output, 0, bytes, s));
    return PC2D_OK;
  }
  switch (dtype) {
    case PC2D_DTYPE_F32: return launch_dropout<float>(input, residual, key, thr, scale, n, output, s);
    case PC2D_DTYPE_F64: return launch_dropout<double>(input, residual, key, thr, scale, n, output, s);
    case PC2D_DTYPE_F16: return launch_dropout<__half>(input, residual, key, thr, scale, n, output, s);
    default: return launch_dropout<__nv_bfloat16>(input, residual, key, thr, scale, n, output, s);
  }
}

extern "C" int pc2d_dropout_next_key(int64_t *state, int64_t *key, void *stream) {
  NvtxRange range("pc2d_dropout_next_key");
  if (!state || !key) {
    set_last_error("pc2d_dropout_next_key: null pointer");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  int st = check_elements("pc2d_dropout_next_key", 8, {state, key});
  if (st != PC2D_OK || (st = pending_device_error()) != PC2D_OK) return st;
  dropout_next_key_kernel<<<1, 1, 0, reinterpret_cast<cudaStream_t>(stream)>>>(state, key);
  PC2D_LAUNCH_CHECK("dropout_next_key_kernel");
  return PC2D_OK;
}
