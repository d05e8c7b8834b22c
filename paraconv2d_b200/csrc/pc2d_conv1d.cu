// Short causal convolution along the length of [batch][channels][length], one
// filter of K <= 8 taps per channel:
//
//   line  = [ state (K-1 values) | x_0 ... x_{n-1} ]       n: the row's length
//   pre_t = bias + sum_k w_k line[t + k]                   out_t = act(pre_t)
//   final = line[n ... n+K-2]
//
// with act the identity or silu(v) = v sigmoid(v).  Backward, with
// dpre = dout act'(pre):
//
//   dline[s] = sum_k w_k dpre[s - k]  (+ dfinal[s - n] for s >= n)
//   dw_k = sum dpre_t line[t + k]     dbias = sum dpre_t
//
// All of it is a few operations per element: the kernels stream.  A warp takes
// a run of one row, and a lane eight elements at a time, cut at the
// 8-element boundaries of the whole array rather than of the row: every load is
// then a 16-byte vector whatever the length is.  In the vectors that a row
// shares with its neighbours, and behind its last token, the foreign elements
// are replaced; only those vectors are stored element by element.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace pc2d {
namespace {

constexpr int kConvThreads = 128;
constexpr int kMaxTaps = 8;

struct ConvArgs {
  const void *x, *weight, *bias, *init;
  const int *lengths;
  int wdtype;
  int batch, channels, length, silu;
  int64_t rows;   // batch * channels
  int nseg;       // warps per row
  int seg;        // 8-element vectors per warp
  // forward
  void *out, *final_state;
  // backward
  const void *grad, *grad_final;
  void *dx, *dinit;
  float *part;    // [batch * nseg][K + 1][channels]
};

__device__ __forceinline__ float load_param(const void *p, int dtype, int64_t i) {
  if (dtype == PC2D_DTYPE_F32) return static_cast<const float *>(p)[i];
  if (dtype == PC2D_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_param(void *p, int dtype, int64_t i, float v) {
  if (dtype == PC2D_DTYPE_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == PC2D_DTYPE_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// Element j (0 .. n+K-2) of a row's line.
template <typename T, int K>
__device__ __forceinline__ float line_at(const T *row, const T *init, int j) {
  const int t = j - (K - 1);
  if (t >= 0) return to_f(row[t]);
  return init ? to_f(init[j]) : 0.f;
}

struct RowPlace {
  int64_t row;
  int seg, d, n;
  int64_t base;   // first element of the row in the array
  int e0;         // t of the first element of the row's vector 0: 0 or below
  int nvec;       // vectors that hold elements of the row
};

__device__ __forceinline__ bool place_of(const ConvArgs &a, RowPlace *p) {
  const int64_t w = ((int64_t)blockIdx.x * kConvThreads + threadIdx.x) >> 5;
  p->row = w / a.nseg;
  if (p->row >= a.rows) return false;
  p->seg = (int)(w - p->row * a.nseg);
  const int b = (int)(p->row / a.channels);
  p->d = (int)(p->row - (int64_t)b * a.channels);
  p->n = a.length;
  if (a.lengths) p->n = min(max(a.lengths[b], 0), a.length);
  p->base = p->row * a.length;
  const int over = (int)(p->base & 7);
  p->e0 = -over;
  p->nvec = (int)(((int64_t)a.length + over + 7) >> 3);
  return true;
}

// The last inputs before a vector that its windows reach: 4 or 8 of them, so
// that they are one aligned load.
template <int K>
constexpr int kBefore = K <= 5 ? 4 : 8;

// One vector of the array, and what its windows need of the one before.
template <typename T, int K>
struct Window {
  Pack<T, 8> cur;
  Pack<T, kBefore<K>> before;
  // `at`: the vector's first element in the array of `total`.  kInside: the
  // vector lies within the array.
  template <bool kInside>
  __device__ __forceinline__ void load(const T *array, int64_t at, int64_t total) {
    load8<kInside>(cur, array, at, total);
    // (before the array's first vector there is nothing: any values do, as they
    // are replaced)
    if (K > 1) {
      if (kInside) before.load(array + (at > 0 ? at - kBefore<K> : at));
      else if (at > 0) before.load(array + at - kBefore<K>);
    }
  }
  template <bool kInside>
  __device__ static __forceinline__ void load8(Pack<T, 8> &v, const T *array, int64_t at, int64_t total) {
    if (kInside || at + 8 <= total) {
      v.load(array + at);
    } else {  // the array's last elements
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < total) v.v[i] = array[at + i];
    }
  }
  // The 7 + K values of the row's line that the windows of its elements t0 ..
  // t0+7 cover: zeros behind the n tokens, the kept state's (or zeros) before.
  // kInside: no element lies behind them.
  template <bool kInside>
  __device__ __forceinline__ void get(float (&x)[K + 7], int t0, int n, const T *init) const {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) x[k] = before.f(kBefore<K> - (K - 1) + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[K - 1 + i] = cur.f(i);
    if (t0 < K - 1) {  // (the first one or two vectors of a row)
#pragma unroll
      for (int i = 0; i < K + 6; ++i) {
        const int t = t0 + i - (K - 1);
        if (t < 0) x[i] = init && t >= -(K - 1) ? to_f(init[t + K - 1]) : 0.f;
      }
    }
    if (!kInside && t0 + 8 > n) {
#pragma unroll
      for (int i = 0; i < K + 7; ++i)
        if (t0 + i - (K - 1) >= n) x[i] = 0.f;
    }
  }
};

template <int K>
__device__ __forceinline__ float filter(const float (&w)[K], float bias, const float (&x)[K + 7], int i) {
  float s = bias;
#pragma unroll
  for (int k = 0; k < K; ++k) s = fmaf(w[k], x[i + k], s);
  return s;
}

template <bool kInside, typename T>
__device__ __forceinline__ void store8(T *row, int t0, int length, const float (&y)[8]) {
  Pack<T, 8> o;
  o.set(y);
  if (t0 >= 0 && (kInside || t0 + 8 <= length)) {
    o.store(row + t0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (t0 + i >= 0 && t0 + i < length) row[t0 + i] = o.v[i];
  }
}

// Two vectors in flight per lane, and as many blocks per SM as hold them without
// spilling (4 x 4096 x 2048 bf16 with 4 taps: 32.8 us, 4.1 TB/s, against 33.2
// with the compiler's choice of registers and 37.3 with four vectors).
constexpr int kConvUnroll = 2;
template <typename T, int K>
constexpr int kConvFwdBlocks = sizeof(T) == 2 && K <= 5 ? 8 : 5;

template <typename T, int K>
__global__ void __launch_bounds__(kConvThreads, kConvFwdBlocks<T, K>) conv_forward_kernel(ConvArgs a) {
  constexpr int U = kConvUnroll;
  RowPlace p;
  if (!place_of(a, &p)) return;
  const int lane = threadIdx.x & 31;
  const T *array = static_cast<const T *>(a.x), *row = array + p.base;
  T *out = static_cast<T *>(a.out) + p.base;
  const T *init = a.init ? static_cast<const T *>(a.init) + p.row * (K - 1) : nullptr;
  const int64_t total = a.rows * a.length;
  float last = 0.f;
  const bool ends = a.final_state && p.seg == 0 && lane < K - 1;
  if (ends) last = line_at<T, K>(row, init, p.n + lane);
  float w[K];
#pragma unroll
  for (int k = 0; k < K; ++k) w[k] = load_param(a.weight, a.wdtype, (int64_t)p.d * K + k);
  const float bias = a.bias ? load_param(a.bias, a.wdtype, p.d) : 0.f;
  const int vb = min(p.nvec, (p.seg + 1) * a.seg);
  // U vectors per lane; kInside: all of them, in all lanes, within the tokens
  auto vectors = [&](int v0, auto inside) {
    constexpr bool kInside = decltype(inside)::value;
    Window<T, K> win[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + lane + 32 * u, t0 = p.e0 + v * 8;
      if (kInside || (v < vb && t0 < p.n)) win[u].template load<kInside>(array, p.base + t0, total);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + lane + 32 * u, t0 = p.e0 + v * 8;
      if (!kInside && v >= vb) break;
      float x[K + 7], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.f;
      if (kInside || t0 < p.n) {
        win[u].template get<kInside>(x, t0, p.n, init);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = filter<K>(w, bias, x, i);
          if (a.silu) y[i] *= sigmoid_f(y[i]);
        }
        if (!kInside && t0 + 8 > p.n) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (t0 + i >= p.n) y[i] = 0.f;
        }
      }
      store8<kInside>(out, t0, a.length, y);
    }
  };
  for (int v0 = p.seg * a.seg; v0 < vb; v0 += 32 * U) {
    if (v0 + 32 * U <= vb && p.e0 + (v0 + 32 * U) * 8 <= p.n) vectors(v0, std::true_type{});
    else vectors(v0, std::false_type{});
  }
  if (ends) static_cast<T *>(a.final_state)[p.row * (K - 1) + lane] = from_f<T>(last);
}

__device__ __forceinline__ float silu_slope(float v) {
  const float e = sigmoid_f(v);
  return e * fmaf(v, 1.f - e, 1.f);
}

// A vector's inputs of the backward pass.
template <typename T, int K>
struct BackWindow {
  Window<T, K> x;
  Pack<T, 8> g;
  template <bool kInside>
  __device__ __forceinline__ void load(const ConvArgs &a, int64_t at, int64_t total) {
    x.template load<kInside>(static_cast<const T *>(a.x), at, total);
    Window<T, K>::template load8<kInside>(g, static_cast<const T *>(a.grad), at, total);
  }
  // the values that its windows cover, and dpre (zeros outside [0, n))
  template <bool kInside>
  __device__ __forceinline__ void get(const ConvArgs &a, int t0, int n, const T *init, const float (&w)[K], float bias,
                                      float (&v)[K + 7], float *dp) const {
    x.template get<kInside>(v, t0, n, init);
#pragma unroll
    for (int i = 0; i < 8; ++i) dp[i] = g.f(i);
    if (a.silu) {
#pragma unroll
      for (int i = 0; i < 8; ++i) dp[i] *= silu_slope(filter<K>(w, bias, v, i));
    }
    if (t0 < 0 || (!kInside && t0 + 8 > n)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t0 + i < 0 || (!kInside && t0 + i >= n)) dp[i] = 0.f;
    }
  }
};

// dpre of token t (0 .. n-1) by itself.
template <typename T, int K>
__device__ __forceinline__ float dpre_at(const ConvArgs &a, const RowPlace &p, const T *init, const float (&w)[K],
                                         float bias, int t) {
  const float g = to_f(static_cast<const T *>(a.grad)[p.base + t]);
  if (!a.silu) return g;
  float s = bias;
#pragma unroll
  for (int k = 0; k < K; ++k) s = fmaf(w[k], line_at<T, K>(static_cast<const T *>(a.x) + p.base, init, t + k), s);
  return g * silu_slope(s);
}

// The lanes' sums of the K + 1 parameter gradients, lane k with the k-th, in a
// fixed order.
template <int K>
__device__ __forceinline__ float sum_params(const float (&dw)[K], float db, int lane) {
  float mine = 0.f;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    float s = k < K ? dw[k < K ? k : 0] : db;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == k) mine = s;
  }
  return mine;
}

// A warp's run once more, a token a lane, with the terms of the row's tokens
// only.  The vectors of conv_backward_kernel multiply the zeros of dpre outside
// of the row by whatever the window or the weights hold, and where that is an
// infinity the product is NaN; leaving the terms out there took 4 to 10 % more.
// Gives the sums of sum_params; `mine`: those that the vectors gave.
template <typename T, int K>
__device__ __noinline__ float conv_backward_again(const ConvArgs &a, float mine) {
  RowPlace p;
  place_of(a, &p);
  const int lane = threadIdx.x & 31;
  const T *row = static_cast<const T *>(a.x) + p.base;
  const T *init = a.init ? static_cast<const T *>(a.init) + p.row * (K - 1) : nullptr;
  const T *dfinal = a.grad_final ? static_cast<const T *>(a.grad_final) + p.row * (K - 1) : nullptr;
  const float bias = a.bias ? load_param(a.bias, a.wdtype, p.d) : 0.f;
  float w[K], dw[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = load_param(a.weight, a.wdtype, (int64_t)p.d * K + k);
    dw[k] = 0.f;
  }
  const int va = p.seg * a.seg, vb = min(p.nvec, va + a.seg), tb = min(a.length, p.e0 + vb * 8);
  __syncwarp();  // (other lanes wrote dx)
#pragma unroll 1
  for (int t = max(0, p.e0 + va * 8) + lane; t < tb; t += 32) {
    float g = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if (t + i < p.n) {
        const float d = dpre_at<T, K>(a, p, init, w, bias, t + i);
        g = fmaf(w[K - 1 - i], d, g);
        if (i == 0) {
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k] = fmaf(d, line_at<T, K>(row, init, t + k), dw[k]);
        }
      }
    }
    const int j = t + (K - 1) - p.n;
    if (dfinal && j >= 0 && t < p.n) g += to_f(dfinal[j]);
    static_cast<T *>(a.dx)[p.base + t] = from_f<T>(g);
  }
  const float again = sum_params<K>(dw, 0.f, lane);
  return lane < K ? again : mine;
}

// Blocks per SM, by the registers that they leave (4 x 4096 x 2048 bf16 with 4
// taps: 64 us, 3.1 TB/s, with 7; 69 with 6, 76 with 8).
template <typename T, int K>
constexpr int kConvBackBlocks = K <= 4 ? (sizeof(T) == 2 ? 7 : 6) : 4;

// A warp goes through its run from the end to the beginning, 32 vectors at a
// time: the K-1 values of dpre behind a lane's eight come from the next lane,
// and for lane 31 from lane 0 of the 32 vectors done before (for the first ones
// from a computation of the vector behind the run).  The inputs of 32 vectors
// are loaded while those before are computed.
template <typename T, int K>
__global__ void __launch_bounds__(kConvThreads, kConvBackBlocks<T, K>)
    conv_backward_kernel(const __grid_constant__ ConvArgs a) {
  RowPlace p;
  if (!place_of(a, &p)) return;
  const int lane = threadIdx.x & 31;
  const T *init = a.init ? static_cast<const T *>(a.init) + p.row * (K - 1) : nullptr;
  const T *dfinal = a.grad_final ? static_cast<const T *>(a.grad_final) + p.row * (K - 1) : nullptr;
  T *dx = static_cast<T *>(a.dx) + p.base;
  const int64_t total = a.rows * a.length;
  const int va = p.seg * a.seg, vb = min(p.nvec, va + a.seg);
  const int top = va + ((vb - va - 1) >> 5) * 32;
  BackWindow<T, K> next;
  // 32 vectors from v0 on: all of them within the row's tokens
  auto inside = [&](int v0) { return v0 + 32 <= vb && p.e0 + (v0 + 32) * 8 <= p.n; };
  auto fetch = [&](int v0) {
    const int t0 = p.e0 + (v0 + lane) * 8;
    if (inside(v0)) next.template load<true>(a, p.base + t0, total);
    else if (v0 + lane < vb && t0 < p.n) next.template load<false>(a, p.base + t0, total);
  };
  if (va < vb) fetch(top);
  float w[K], dw[K], db = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = load_param(a.weight, a.wdtype, (int64_t)p.d * K + k);
    dw[k] = 0.f;
  }
  const float bias = a.bias ? load_param(a.bias, a.wdtype, p.d) : 0.f;
  constexpr int B = K > 1 ? K - 1 : 1;
  float carry[B];  // dpre of the first elements of the vector behind
#pragma unroll
  for (int k = 0; k < B; ++k) carry[k] = 0.f;
  if (K > 1 && va < vb && vb < p.nvec && p.e0 + vb * 8 < p.n) {
    BackWindow<T, K> behind;
    float x[K + 7], dp[8];
    behind.template load<false>(a, p.base + p.e0 + vb * 8, total);
    behind.template get<false>(a, p.e0 + vb * 8, p.n, init, w, bias, x, dp);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) carry[k] = dp[k];
  }
  auto vectors = [&](int v0, auto all) {
    constexpr bool kInside = decltype(all)::value;
    const int v = v0 + lane, t0 = p.e0 + v * 8;
    float x[K + 7], dp[8 + B], g[8];
    if (kInside || (v < vb && t0 < p.n)) {
      next.template get<kInside>(a, t0, p.n, init, w, bias, x, dp);
    } else {
#pragma unroll
      for (int i = 0; i < K + 7; ++i) x[i] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) dp[i] = 0.f;
    }
    if (v0 > va) fetch(v0 - 32);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      // the last vector of the run may sit in any lane: lanes behind it hold
      // zeros, so it takes the carry itself
      const float behind = __shfl_down_sync(0xffffffffu, dp[k], 1);
      const float first = __shfl_sync(0xffffffffu, dp[k], 0);
      dp[8 + k] = lane == 31 || (!kInside && v == vb - 1) ? carry[k] : behind;
      carry[k] = first;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      db += dp[i];
#pragma unroll
      for (int k = 0; k < K; ++k) dw[k] = fmaf(dp[i], x[i + k], dw[k]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] = w[K - 1] * dp[i];
#pragma unroll
      for (int k = 1; k < K; ++k) g[i] = fmaf(w[K - 1 - k], dp[i + k], g[i]);
    }
    if (K > 1 && dfinal && t0 + 8 + K - 1 > p.n) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = t0 + i + (K - 1) - p.n;
        if (j >= 0 && t0 + i >= 0 && t0 + i < p.n) g[i] += to_f(dfinal[j]);
      }
    }
    // (behind the last token dpre is 0, and so is g)
    if (kInside || v < vb) store8<kInside>(dx, t0, a.length, g);
  };
  for (int v0 = top; v0 >= va && va < vb; v0 -= 32) {
    if (inside(v0)) vectors(v0, std::true_type{});
    else vectors(v0, std::false_type{});
  }
  float mine = sum_params<K>(dw, db, lane);  // the warp's share
  bool finite = fabsf(mine) < __int_as_float(0x7f800000);
#pragma unroll
  for (int k = 0; k < K; ++k) finite = finite && fabsf(w[k]) < __int_as_float(0x7f800000);
  if (!__all_sync(0xffffffffu, finite)) mine = conv_backward_again<T, K>(a, mine);
  const int64_t b = p.row / a.channels;
  if (lane <= K) a.part[((b * a.nseg + p.seg) * (K + 1) + lane) * a.channels + p.d] = mine;
  if (K > 1 && a.dinit && p.seg == 0) {
    // dline[s], s < K-1: lane j computes dpre[j] from its own window
    const float dpj = lane < K - 1 && lane < p.n ? dpre_at<T, K>(a, p, init, w, bias, lane) : 0.f;
    float g = 0.f;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const float other = __shfl_sync(0xffffffffu, dpj, (lane - k) & 31);
      if (lane >= k && lane - k < p.n) g = fmaf(w[k], other, g);
    }
    if (lane < K - 1) {
      if (dfinal && lane >= p.n) g += to_f(dfinal[lane - p.n]);
      static_cast<T *>(a.dinit)[p.row * (K - 1) + lane] = from_f<T>(g);
    }
  }
}

// Sums the warps' shares [groups][K+1][channels] over the groups, in 64 bits
// and in a fixed order: 8 lanes of threads per (k, channel), then those 8.
__global__ void __launch_bounds__(256) conv_param_kernel(const float *__restrict__ part, int groups, int taps,
                                                        int channels, int wdtype, void *dweight, void *dbias) {
  __shared__ double sums[8][32];
  const int d = blockIdx.x * 32 + threadIdx.x, k = blockIdx.y;
  double s = 0.0;
  if (d < channels) {
#pragma unroll 4
    for (int g = threadIdx.y; g < groups; g += 8) s += part[((int64_t)g * (taps + 1) + k) * channels + d];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || d >= channels) return;
  for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
  if (k < taps) {
    if (dweight) store_param(dweight, wdtype, (int64_t)d * taps + k, (float)s);
  } else if (dbias) {
    store_param(dbias, wdtype, d, (float)s);
  }
}

struct ConvStepArgs {
  const void *x, *weight, *bias;
  const int *slots;
  void *state, *out;
  int wdtype, batch, places, channels, silu;
};

// One token: thread = channel.  Reads and writes the K-1 kept inputs once.
template <typename T, int K>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(ConvStepArgs a) {
  const int nblk = (a.channels + kConvThreads - 1) / kConvThreads;
  const int b = blockIdx.x / nblk;
  StepKind kind;
  const int place = step_place(a.slots, b, a.places, &kind);
  const int twice = step_twice(a.slots, b, place, kind);
  const int d = (blockIdx.x - b * nblk) * kConvThreads + threadIdx.x;
  const bool valid = d < a.channels;
  const int64_t at = (int64_t)b * a.channels + d;
  T *kept = static_cast<T *>(a.state) + ((int64_t)place * a.channels + d) * (K - 1);
  T line[K];
  float s = 0.f;
  if (valid && kind == kStepServed) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) line[k] = kept[k];
    line[K - 1] = static_cast<const T *>(a.x)[at];
    if (a.bias) s = load_param(a.bias, a.wdtype, d);
#pragma unroll
    for (int k = 0; k < K; ++k) s = fmaf(load_param(a.weight, a.wdtype, (int64_t)d * K + k), to_f(line[k]), s);
  }
  kind = step_served(twice, kind);
  if (!valid) return;
  T *out = static_cast<T *>(a.out) + at;
  if (kind != kStepServed) {
    *out = from_f<T>(step_nothing(kind));
    return;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) kept[k] = line[k + 1];
  *out = from_f<T>(a.silu ? s * sigmoid_f(s) : s);
}

enum ConvWhat { kConvForward, kConvBackward };

// Vectors per warp: long runs amortise a warp's set-up (parameters, the vector
// behind the run), short ones fill the GPU when there are few rows.  Runs of a
// row are equally long, in whole groups of 32 vectors.
void conv_split(const ConvArgs &a, int *nseg, int *seg) {
  // (a row that starts off a vector boundary reaches into one vector more)
  const int nvec = a.length % 8 == 0 ? a.length / 8 : (int)(((int64_t)a.length + 14) >> 3);
  const int groups = std::max(1, (nvec + 31) / 32);
  int most = 8;
  while (most > 1 && a.rows * ((groups + most - 1) / most) < (int64_t)device_sm_count() * 32) most /= 2;
  const int runs = (groups + most - 1) / most;
  *seg = 32 * ((groups + runs - 1) / runs);
  *nseg = std::max(1, (nvec + *seg - 1) / *seg);
}

template <typename T, int K>
int launch_conv(ConvWhat what, const ConvArgs &a, cudaStream_t stream) {
  const int64_t blocks = (a.rows * a.nseg * 32 + kConvThreads - 1) / kConvThreads;
  if (what == kConvForward) conv_forward_kernel<T, K><<<(unsigned)blocks, kConvThreads, 0, stream>>>(a);
  else conv_backward_kernel<T, K><<<(unsigned)blocks, kConvThreads, 0, stream>>>(a);
  PC2D_LAUNCH_CHECK(what == kConvForward ? "conv_forward_kernel" : "conv_backward_kernel");
  return PC2D_OK;
}

template <typename T, int K>
int launch_conv_step(const ConvStepArgs &a, cudaStream_t stream) {
  const int nblk = (a.channels + kConvThreads - 1) / kConvThreads;
  conv_step_kernel<T, K><<<(unsigned)(nblk * a.batch), kConvThreads, 0, stream>>>(a);
  PC2D_LAUNCH_CHECK("conv_step_kernel");
  return PC2D_OK;
}

// f.template operator()<T, K>() for the call's type and taps
template <typename F>
int by_type_and_taps(int dtype, int taps, F &&f) {
#define PC2D_TAPS(T)                                            \
  switch (taps) {                                               \
    case 1: return f(T{}, std::integral_constant<int, 1>{});    \
    case 2: return f(T{}, std::integral_constant<int, 2>{});    \
    case 3: return f(T{}, std::integral_constant<int, 3>{});    \
    case 4: return f(T{}, std::integral_constant<int, 4>{});    \
    case 5: return f(T{}, std::integral_constant<int, 5>{});    \
    case 6: return f(T{}, std::integral_constant<int, 6>{});    \
    case 7: return f(T{}, std::integral_constant<int, 7>{});    \
    default: return f(T{}, std::integral_constant<int, 8>{});   \
  }
  if (dtype == PC2D_DTYPE_F32) { PC2D_TAPS(float) }
  if (dtype == PC2D_DTYPE_F16) { PC2D_TAPS(__half) }
  PC2D_TAPS(__nv_bfloat16)
#undef PC2D_TAPS
}

int check_conv(const char *what, int dtype, int wdtype, int batch, int channels, int length, int taps) {
  if (!seq_dtype(dtype)) {
    set_last_error("%s: unsupported dtype %d (float32, float16 and bfloat16)", what, dtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (wdtype != dtype && wdtype != PC2D_DTYPE_F32) {
    set_last_error("%s: weights of dtype %d beside inputs of dtype %d (the inputs' type or float32)", what, wdtype,
                   dtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (batch < 0 || channels < 0 || length < 0 || taps < 1) {
    set_last_error("%s: invalid batch %d, channels %d, length %d or taps %d", what, batch, channels, length, taps);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (taps > kMaxTaps) {
    set_last_error("%s: %d taps (at most %d)", what, taps, kMaxTaps);
    return PC2D_ERR_UNSUPPORTED;
  }
  // the vectors of a row are counted in 32 bits, the warps of a launch too
  if (length > 1 << 30 || (int64_t)batch * channels > (int64_t)1 << 30 ||
      (int64_t)batch * channels * (length / 256 + 2) > (int64_t)1 << 33) {
    set_last_error("%s: problem too large", what);
    return PC2D_ERR_UNSUPPORTED;
  }
  return PC2D_OK;
}

int check_aligned(const char *what, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (p && !aligned16(p)) {
      set_last_error("%s: the activations and their gradients must be 16-byte aligned", what);
      return PC2D_ERR_INVALID_ARGUMENT;
    }
  return PC2D_OK;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" int pc2d_causal_conv_forward(int dtype, int wdtype, const void *input, const void *weight, const void *bias,
                                        const void *initial_state, const int *lengths, int batch, int channels,
                                        int length, int taps, int silu, void *output, void *final_state,
                                        void *stream) {
  NvtxRange range("pc2d_causal_conv_forward");
  int st = check_conv("pc2d_causal_conv_forward", dtype, wdtype, batch, channels, length, taps);
  if (st != PC2D_OK) return st;
  if ((st = pending_device_error()) != PC2D_OK) return st;
  ConvArgs a{};
  a.rows = (int64_t)batch * channels;
  if (a.rows == 0 || (length == 0 && (!final_state || taps == 1))) return PC2D_OK;
  if (!weight || (length > 0 && (!input || !output))) {
    set_last_error("pc2d_causal_conv_forward: null pointer (input, weight or output)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_aligned("pc2d_causal_conv_forward", {input, output})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_forward", seq_dtype_size(dtype), {initial_state, final_state})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_forward", seq_dtype_size(wdtype), {weight, bias})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_forward", 4, {lengths})) != PC2D_OK)
    return st;
  a.x = input; a.weight = weight; a.bias = bias; a.init = taps > 1 ? initial_state : nullptr;
  a.lengths = lengths; a.wdtype = wdtype;
  a.batch = batch; a.channels = channels; a.length = length; a.silu = silu != 0;
  a.out = output; a.final_state = final_state;
  conv_split(a, &a.nseg, &a.seg);
  return by_type_and_taps(dtype, taps, [&](auto t, auto k) {
    return launch_conv<decltype(t), decltype(k)::value>(kConvForward, a, reinterpret_cast<cudaStream_t>(stream));
  });
}

extern "C" size_t pc2d_causal_conv_backward_workspace_size(int batch, int channels, int length, int taps) {
  if (check_conv("pc2d_causal_conv_backward_workspace_size", PC2D_DTYPE_F32, PC2D_DTYPE_F32, batch, channels, length,
                 taps) != PC2D_OK)
    return 0;
  ConvArgs a{};
  a.rows = (int64_t)batch * channels;
  a.length = length;
  int nseg, seg;
  conv_split(a, &nseg, &seg);
  return (size_t)a.rows * nseg * (taps + 1) * sizeof(float);
}

extern "C" int pc2d_causal_conv_backward(int dtype, int wdtype, const void *grad, const void *grad_final,
                                         const void *input, const void *weight, const void *bias,
                                         const void *initial_state, const int *lengths, int batch, int channels,
                                         int length, int taps, int silu, void *inputgrad, void *weightgrad,
                                         void *biasgrad, void *initialgrad, void *workspace, size_t workspace_bytes,
                                         void *stream) {
  NvtxRange range("pc2d_causal_conv_backward");
  int st = check_conv("pc2d_causal_conv_backward", dtype, wdtype, batch, channels, length, taps);
  if (st != PC2D_OK) return st;
  if ((st = pending_device_error()) != PC2D_OK) return st;
  if (channels == 0) return PC2D_OK;
  ConvArgs a{};
  a.rows = (int64_t)batch * channels;
  if (!weight || (a.rows > 0 && length > 0 && (!grad || !input || !inputgrad))) {
    set_last_error("pc2d_causal_conv_backward: null pointer (grad, input, weight or inputgrad)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_aligned("pc2d_causal_conv_backward", {grad, input, inputgrad})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_backward", seq_dtype_size(dtype),
                           {grad_final, initial_state, initialgrad})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_backward", seq_dtype_size(wdtype),
                           {weight, bias, weightgrad, biasgrad})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_backward", 4, {lengths})) != PC2D_OK)
    return st;
  const size_t need = pc2d_causal_conv_backward_workspace_size(batch, channels, length, taps);
  if (workspace_bytes < need || (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)))) {
    set_last_error("pc2d_causal_conv_backward: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", need,
                   workspace_bytes);
    return PC2D_ERR_WORKSPACE;
  }
  a.x = input; a.weight = weight; a.bias = bias; a.init = taps > 1 ? initial_state : nullptr;
  a.lengths = lengths; a.wdtype = wdtype;
  a.batch = batch; a.channels = channels; a.length = length; a.silu = silu != 0;
  a.grad = grad; a.grad_final = taps > 1 ? grad_final : nullptr;
  a.dx = inputgrad; a.dinit = taps > 1 ? initialgrad : nullptr;
  a.part = static_cast<float *>(workspace);
  conv_split(a, &a.nseg, &a.seg);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.rows > 0) {
    st = by_type_and_taps(dtype, taps, [&](auto t, auto k) {
      return launch_conv<decltype(t), decltype(k)::value>(kConvBackward, a, s);
    });
    if (st != PC2D_OK) return st;
  }
  if (!weightgrad && !biasgrad) return PC2D_OK;
  conv_param_kernel<<<dim3((channels + 31) / 32, taps + 1), dim3(32, 8), 0, s>>>(a.part, batch * a.nseg, taps,
                                                                               channels, wdtype, weightgrad, biasgrad);
  PC2D_LAUNCH_CHECK("conv_param_kernel");
  return PC2D_OK;
}

extern "C" int pc2d_causal_conv_step(int dtype, int wdtype, const void *input, void *state, const void *weight,
                                     const void *bias, const int *slots, int batch, int places, int channels, int taps,
                                     int silu, void *output, void *stream) {
  NvtxRange range("pc2d_causal_conv_step");
  int st = check_conv("pc2d_causal_conv_step", dtype, wdtype, batch, channels, 1, taps);
  if (st != PC2D_OK) return st;
  if (places < 0 || (!slots && batch > places)) {
    set_last_error("pc2d_causal_conv_step: %d rows of a batch without slots, but %d states", batch, places);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = pending_device_error()) != PC2D_OK) return st;
  if (batch == 0 || channels == 0) return PC2D_OK;
  if (!input || !weight || !output || (taps > 1 && !state && places > 0)) {
    set_last_error("pc2d_causal_conv_step: null pointer (input, state, weight or output)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_elements("pc2d_causal_conv_step", seq_dtype_size(dtype), {input, state, output})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_step", seq_dtype_size(wdtype), {weight, bias})) != PC2D_OK ||
      (st = check_elements("pc2d_causal_conv_step", 4, {slots})) != PC2D_OK)
    return st;
  ConvStepArgs a{};
  a.x = input; a.weight = weight; a.bias = bias; a.slots = slots; a.state = state; a.out = output;
  a.wdtype = wdtype; a.batch = batch; a.places = places; a.channels = channels; a.silu = silu != 0;
  return by_type_and_taps(dtype, taps, [&](auto t, auto k) {
    return launch_conv_step<decltype(t), decltype(k)::value>(a, reinterpret_cast<cudaStream_t>(stream));
  });
}
