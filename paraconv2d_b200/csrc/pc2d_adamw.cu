// AdamW over many tensors in one launch, with the moments in 32 or in 8 bits.
//
// Per element w with gradient g (times *grad_scale), at step t = ++*step:
//   m = beta1 m + (1 - beta1) g
//   v = beta2 v + (1 - beta2) g^2
//   w = (1 - lr rate decay wd) w - lr rate / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
// with a tensor's own rate (one below `split`, one from there on: the halves
// [h0 | h] and [p | p0] of a ParaConv2d layer) and decay factor.  m, v and w are
// computed in 32 bits, w from the new moments before these are rounded.
// With a master, w is held there in 32 bits and the parameter is its rounding.
//
// Moments in 8 bits: floats with 3 bits of mantissa, m with a sign and 4 bits
// of exponent, v with 5 bits (the same 16 binades for sqrt(v)).  256
// neighbouring elements share the exponent E of their smallest normal number,
// the one that brings their largest, rounded up, into the topmost binade: a code c below 8
// is c/8 of that number, any other 2^((c >> 3) - 1) (1 + (c & 7) / 8) of it.
// E is a byte, the exponent field of a 32-bit float; 255 says that the block
// had a value that is not finite, and all of its elements read as NaN.
// They are rounded stochastically, up with the probability of what is cut off
// (8 bits of it).  To the nearest, v would stand still: with beta2 = 0.999 it
// moves by 1e-3 of itself and less, and half a step is 3 to 6% of it.  A v
// that is not zero stays so (code 1 at least): the step is divided by its root,
// and an m of the same element, whose smallest code is about the root of v's,
// may have been rounded up.
// The random bits are Philox4x32-10's (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) under the key `seed`
// for the counter (element / 8, tensor, step): 16 bytes for the two moments of
// eight elements.
//
// Products and sums of the moments are rounded one by one (no fused
// operations): the codes are then the same whichever machine computes them.
#include <math.h>

#include <algorithm>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace pc2d {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;   // elements of a block of 8-bit moments: one warp, 8 a lane
constexpr int kChunk = 8192;  // elements of a thread block: 32 such blocks, four a warp
// Tensors of a launch: what the 32 KB that a launch may pass as parameters
// hold, and what 4 KB hold.
constexpr int kMany = 320, kFew = 36;

struct Item {
  void *param;
  const void *grad;
  void *m, *v;
  float *master;
  unsigned char *scales;
  int64_t n, split;
  float rate_first, rate_rest, decay;
  int index;  // the tensor's number in the counter
  int vec;    // every array on the boundary that vectors need
};

template <int N>
struct Items {
  Item item[N];
  int first[N];  // thread block that a tensor begins with
  int count;
};

static_assert(sizeof(Items<kMany>) <= 32000 && sizeof(Items<kFew>) <= 4000, "a launch's parameters");

// What every element needs of the step, made by one thread.  (In 32 bits: the
// GPU's 64-bit arithmetic is so slow that its latency showed in every block.)
struct Coef {
  float lr, lr1, root;  // lr, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  int pad;
  int64_t t;
};

struct Betas {
  float b1, c1, b2, c2, eps, wd;
  uint64_t seed;
};

// log1, log2: logarithms of the betas (1 - beta^t by expm1, which keeps its digits where it is small)
__global__ void adamw_coef_kernel(int64_t *step, const float *lr_device, float lr, float log1, float log2, Coef *coef) {
  const int64_t t = *step + 1;
  *step = t;
  if (lr_device) lr = *lr_device;
  coef->lr = lr;
  coef->lr1 = lr / -expm1f((float)t * log1);
  coef->root = rsqrtf(-expm1f((float)t * log2));
  coef->t = t;
}

template <int N>
__device__ __forceinline__ int find_item(const Items<N> &a, int block) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

struct Rates {
  float drop_first, drop_rest, lr_first, lr_rest, root, scale;  // drop: what the decay takes of a weight
  int64_t split;
};

__device__ __forceinline__ void moments(float &m, float &v, float g, const Betas &b) {
  m = __fadd_rn(__fmul_rn(m, b.b1), __fmul_rn(g, b.c1));
  v = __fadd_rn(__fmul_rn(v, b.b2), __fmul_rn(__fmul_rn(g, b.c2), g));
}
__device__ __forceinline__ float weight(float w, float m, float v, bool first, const Rates &r, const Betas &b) {
  // the hardware's square root and quotient: 2^-22 of the step, far below half a unit of w
  float s;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(s) : "f"(v));
  const float step = __fdividef(m, fmaf(s, r.root, b.eps));
  const float by = (first ? r.lr_first : r.lr_rest) * step;
  // What goes off, and then off the weight: 1 - lr wd in 32 bits would be lr wd rounded to a multiple of 2^-24, nothing
  // at all for lr wd = 1e-8.  (An infinite weight stays one.)
  const float decayed = fmaf(first ? r.drop_first : r.drop_rest, w, by);
  return w - (fabsf(w) == __int_as_float(0x7f800000) ? by : decayed);
}

// ------------------------------------------------------------- 8-bit moments

// 2^e, for e from -127 to 127
__device__ __forceinline__ constexpr unsigned exp2_bits(int e) { return e < -126 ? 1u << 22 : (unsigned)(e + 127) << 23; }
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(exp2_bits(e)); }

template <bool kSigned>
struct Code {
  static constexpr int kTop = kSigned ? 15 : 31;  // binades of normal numbers
  // E of a block whose largest absolute value has the bits `most`
  static __device__ __forceinline__ unsigned scale(unsigned most) {
    // (above 15/8 of its binade it may be rounded up into the next one)
    return most >= 0x7f800000u ? 255u : (unsigned)max((int)((most + 0xFFFFFu) >> 23) - (kTop - 1), 1);
  }
  // A code at bit 20 has the fields of a 32-bit float, small codes those of its
  // subnormal numbers: two exact products with powers of two (one would
  // overflow) bring the smallest normal number, 2^-126, to 2^(E - 127).
  static __device__ __forceinline__ float up(unsigned E) {
    return E == 255 ? __uint_as_float(0x7fffffffu) : exp2i((int)E - 127);
  }
  static __device__ __forceinline__ float decode(unsigned code, float up) {
    const unsigned bits = kSigned ? (code & 127u) << 20 | (code & 128u) << 24 : code << 20;
    return __uint_as_float(bits) * exp2i(126) * up;
  }
  // And back, with the rounding of the second product at the subnormal numbers'
  // step.  `low`: the 8 random bits, at bit 12.
  static __device__ __forceinline__ unsigned encode(float x, float down, unsigned low) {
    const unsigned bits = __float_as_uint(fabsf(x) * down * exp2i(-126));
    unsigned code = (bits + low + 2048u) >> 20;
    if (!kSigned && x > 0.f) code = max(code, 1u);
    return kSigned && x < 0.f ? code | 128u : code;
  }
};

struct Bytes16 {
  unsigned w[4];
};
__device__ __forceinline__ Bytes16 random16(uint64_t group, unsigned index, uint64_t t, uint64_t seed) {
  unsigned c0 = (unsigned)group, c1 = index, c2 = (unsigned)t, c3 = (unsigned)(t >> 32);
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
  return Bytes16{{c0, c1, c2, c3}};
}

// ------------------------------------------------------------------- kernels

// N elements of an array that is on a vector's boundary and whole, or else one
// by one, those of the `left` that there are.
template <typename T, int N>
__device__ __forceinline__ void fetch(Pack<T, N> &a, const T *p, bool whole, int left) {
  if (whole) {
    a.load(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = i < left ? p[i] : T(0);
  }
}
template <typename T, int N>
__device__ __forceinline__ void put(const float (&x)[N], T *p, bool whole, int left) {
  Pack<T, N> a;
  a.set(x);
  if (whole) {
    a.store(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = a.v[i];
  }
}

__device__ __forceinline__ Rates rates_of(const Item &it, const Coef *coef, const float *grad_scale, const Betas &b) {
  const float lr = coef->lr, lr1 = coef->lr1;
  Rates r;
  r.drop_first = lr * it.rate_first * b.wd * it.decay;
  r.drop_rest = lr * it.rate_rest * b.wd * it.decay;
  r.lr_first = lr1 * it.rate_first;
  r.lr_rest = lr1 * it.rate_rest;
  r.root = coef->root;
  r.scale = grad_scale ? *grad_scale : 1.f;
  r.split = it.split;
  return r;
}

// Moments in 32 bits: V elements a thread and vector, two vectors in flight.
// Memory bounds it: 92 million bfloat16 parameters with masters, 28 bytes each,
// take 395 us, 6.5 TB/s.  Small sets are bound by the two launches: 225,000
// float32 parameters in four tensors 8.5 us on the GPU, 20 with the host's share.
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Items<N> a, const Coef *coef,
                                                         const float *grad_scale, const Betas b) {
  constexpr int V = 4, U = 2;
  const int k = find_item(a, blockIdx.x);
  const Item &it = a.item[k];
  const Rates r = rates_of(it, coef, grad_scale, b);
  const int64_t begin = (int64_t)(blockIdx.x - a.first[k]) * kChunk, n = it.n;
  const int64_t end = min(begin + kChunk, n);
  P *param = (P *)it.param;
  const G *grad = (const G *)it.grad;
  float *ms = (float *)it.m, *vs = (float *)it.v;
  for (int64_t at = begin + threadIdx.x * V; at < end; at += kThreads * V * U) {
    Pack<G, V> g[U];
    Pack<float, V> m[U], v[U], w[U];
    Pack<P, V> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = at + u * kThreads * V;
      if (e < end) {
        const int left = (int)min(n - e, (int64_t)V);
        const bool whole = it.vec && left == V;
        fetch(g[u], grad + e, whole, left);
        fetch(m[u], ms + e, whole, left);
        fetch(v[u], vs + e, whole, left);
        if (it.master) fetch(w[u], it.master + e, whole, left);
        else fetch(p[u], param + e, whole, left);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = at + u * kThreads * V;
      if (e < end) {
        const int left = (int)min(n - e, (int64_t)V);
        const bool whole = it.vec && left == V;
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          moments(m[u].v[i], v[u].v[i], __fmul_rn(to_f(g[u].v[i]), r.scale), b);
          x[i] = weight(it.master ? w[u].v[i] : to_f(p[u].v[i]), m[u].v[i], v[u].v[i], e + i < r.split, r, b);
        }
        put<float, V>(m[u].v, ms + e, whole, left);
        put<float, V>(v[u].v, vs + e, whole, left);
        if (it.master) put<float, V>(x, it.master + e, whole, left);
        put<P, V>(x, param + e, whole, left);
      }
    }
  }
}

// Moments in 8 bits: a warp takes a block of 256 at a time, eight a lane (the
// generator's 16 bytes are for eight elements; the largest values meet in one
// instruction a warp).  Instructions bound it, not memory: 46 million bfloat16
// parameters, 10 bytes each, take 187 us, 2.5 TB/s.  Codes by comparisons and
// shifts instead of products took 242, two blocks an SM instead of three
// included.
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads, 3) adamw8_kernel(const __grid_constant__ Items<N> a, const Coef *coef,
                                                          const float *grad_scale, const Betas b) {
  constexpr int V = 8;
  const int k = find_item(a, blockIdx.x);
  const Item &it = a.item[k];
  const Rates r = rates_of(it, coef, grad_scale, b);
  const uint64_t t = (uint64_t)coef->t;
  const int64_t begin = (int64_t)(blockIdx.x - a.first[k]) * kChunk, n = it.n;
  const int64_t end = min(begin + kChunk, n);
  const int lane = threadIdx.x & 31;
  P *param = (P *)it.param;
  const G *grad = (const G *)it.grad;
  unsigned char *ms = (unsigned char *)it.m, *vs = (unsigned char *)it.v;
  for (int64_t block = begin + (threadIdx.x >> 5) * kBlock; block < end; block += kThreads / 32 * kBlock) {
    const int64_t e = block + lane * V;
    const int left = (int)max((int64_t)0, min(n - e, (int64_t)V));
    const bool whole = it.vec && left == V;
    Pack<G, V> g;
    Pack<P, V> p;
    Pack<float, V> w;
    Pack<unsigned char, V> mc, vc;
    fetch(g, grad + e, whole, left);
    fetch(mc, ms + e, whole, left);
    fetch(vc, vs + e, whole, left);
    if (it.master) fetch(w, it.master + e, whole, left);
    else fetch(p, param + e, whole, left);
    unsigned char *scale = it.scales + block / kBlock * 2;
    const float em = Code<true>::up(scale[0]), ev = Code<false>::up(scale[1]);
    const Bytes16 low = random16((uint64_t)(e / V), (unsigned)it.index, t, b.seed);
    float m[V], v[V], x[V];
    unsigned most_m = 0, most_v = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      m[i] = Code<true>::decode(mc.v[i], em);
      v[i] = Code<false>::decode(vc.v[i], ev);
      moments(m[i], v[i], __fmul_rn(to_f(g.v[i]), r.scale), b);
      x[i] = weight(it.master ? w.v[i] : to_f(p.v[i]), m[i], v[i], e + i < r.split, r, b);
      if (i < left) {
        most_m = max(most_m, __float_as_uint(fabsf(m[i])));
        most_v = max(most_v, __float_as_uint(fabsf(v[i])));
      }
    }
    if (it.master) put<float, V>(x, it.master + e, whole, left);
    put<P, V>(x, param + e, whole, left);
    const unsigned nm = Code<true>::scale(__reduce_max_sync(0xffffffffu, most_m));
    const unsigned nv = Code<false>::scale(__reduce_max_sync(0xffffffffu, most_v));
    // (values that are not finite have code 0: their exponent says what they are)
    const float dm = nm == 255 ? 0.f : exp2i(127 - (int)nm), dv = nv == 255 ? 0.f : exp2i(127 - (int)nv);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const unsigned rm = low.w[i / 4], rv = low.w[2 + i / 4], mask = 255u << 12;
      mc.v[i] = (unsigned char)Code<true>::encode(m[i], dm, (i % 4 < 2 ? rm << (12 - 8 * (i % 4)) : rm >> (8 * (i % 4) - 12)) & mask);
      vc.v[i] = (unsigned char)Code<false>::encode(v[i], dv, (i % 4 < 2 ? rv << (12 - 8 * (i % 4)) : rv >> (8 * (i % 4) - 12)) & mask);
    }
    if (nm == 255)
#pragma unroll
      for (int i = 0; i < V; ++i) mc.v[i] = 0;
    if (nv == 255)
#pragma unroll
      for (int i = 0; i < V; ++i) vc.v[i] = 0;
    if (whole) {
      mc.store(ms + e);
      vc.store(vs + e);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) {
          ms[e + i] = mc.v[i];
          vs[e + i] = vc.v[i];
        }
    }
    if (lane == 0) {
      scale[0] = (unsigned char)nm;
      scale[1] = (unsigned char)nv;
    }
  }
}

// 8-bit moments read out: m into `param`, v into `master` of an item.  Memory
// bounds it: 46 million to bfloat16 in 42 us, 6.6 TB/s.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) adamw_values_kernel(const __grid_constant__ Items<N> a) {
  constexpr int V = 8;
  const int k = find_item(a, blockIdx.x);
  const Item &it = a.item[k];
  const int64_t begin = (int64_t)(blockIdx.x - a.first[k]) * kChunk, n = it.n;
  const int64_t end = min(begin + kChunk, n);
  const unsigned char *ms = (const unsigned char *)it.m, *vs = (const unsigned char *)it.v;
  T *mo = (T *)it.param, *vo = (T *)it.master;
  for (int64_t e = begin + threadIdx.x * V; e < end; e += kThreads * V) {
    const int left = (int)min(n - e, (int64_t)V);
    const bool whole = it.vec && left == V;
    Pack<unsigned char, V> mc, vc;
    fetch(mc, ms + e, whole, left);
    fetch(vc, vs + e, whole, left);
    const float em = Code<true>::up(it.scales[e / kBlock * 2]), ev = Code<false>::up(it.scales[e / kBlock * 2 + 1]);
    float m[V], v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      m[i] = Code<true>::decode(mc.v[i], em);
      v[i] = Code<false>::decode(vc.v[i], ev);
    }
    put<T, V>(m, mo + e, whole, left);
    put<T, V>(v, vo + e, whole, left);
  }
}

bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Calls run(Items<N>, grid) for the tensors that `take` chooses, as many to a
// launch as its parameters hold.  fill(item, tensor) completes an item.
template <typename Take, typename Fill, typename RunFew, typename RunMany>
int in_launches(const pc2d_adamw_tensor *tensors, int count, Take &&take, Fill &&fill, RunFew &&few, RunMany &&many) {
  int chosen = 0;
  for (int i = 0; i < count; ++i) chosen += take(tensors[i]);
  const bool small = chosen <= kFew;
  Items<kFew> a;
  static thread_local Items<kMany> b;  // (28 KB)
  Item *items = small ? a.item : b.item;
  int *first = small ? a.first : b.first;
  int used = 0;
  int64_t blocks = 0;
  auto launch = [&]() -> int {
    if (!used) return PC2D_OK;
    (small ? a.count : b.count) = used;
    const int st = small ? few(a, (unsigned)blocks) : many(b, (unsigned)blocks);
    used = 0;
    blocks = 0;
    return st;
  };
  for (int i = 0; i < count; ++i) {
    if (!take(tensors[i])) continue;
    const int64_t need = (tensors[i].n + kChunk - 1) / kChunk;
    if (used == (small ? kFew : kMany) || blocks + need > 0x7fffffff) {
      const int st = launch();
      if (st != PC2D_OK) return st;
    }
    Item it{};
    it.m = tensors[i].exp_avg;
    it.v = tensors[i].exp_avg_sq;
    it.scales = tensors[i].scales;
    it.n = tensors[i].n;
    it.index = i;
    fill(it, tensors[i]);
    items[used] = it;
    first[used++] = (int)blocks;
    blocks += need;
  }
  return launch();
}

template <typename P, typename G>
int launch_group(int bits, const pc2d_adamw_tensor *tensors, int count, const int64_t *numbers, int dtype,
                 int grad_dtype, const Coef *coef, const float *grad_scale, const Betas &b, cudaStream_t stream) {
  auto take = [&](const pc2d_adamw_tensor &t) { return t.n > 0 && t.dtype == dtype && t.grad_dtype == grad_dtype; };
  auto fill = [&](Item &it, const pc2d_adamw_tensor &t) {
    it.param = t.param;
    it.grad = t.grad;
    it.master = t.master;
    it.split = t.split;
    if (numbers) it.index = (int)numbers[&t - tensors];
    it.rate_first = (float)t.rate_first;
    it.rate_rest = (float)t.rate_rest;
    it.decay = (float)t.decay;
    const size_t state = bits == 8 ? 8 : 16;
    it.vec = aligned_to(t.param, 16) && aligned_to(t.grad, 16) && aligned_to(t.exp_avg, state) &&
             aligned_to(t.exp_avg_sq, state) && aligned_to(t.master, 16);
  };
  auto run = [&](auto &items, unsigned grid) -> int {
    constexpr int N = sizeof(items.first) / sizeof(int);
    if (bits == 8) adamw8_kernel<P, G, N><<<grid, kThreads, 0, stream>>>(items, coef, grad_scale, b);
    else adamw_kernel<P, G, N><<<grid, kThreads, 0, stream>>>(items, coef, grad_scale, b);
    PC2D_LAUNCH_CHECK("adamw_kernel");
    return PC2D_OK;
  };
  return in_launches(tensors, count, take, fill, run, run);
}

int refuse(const char *fmt, int i) {
  set_last_error(fmt, i);
  return PC2D_ERR_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" size_t pc2d_adamw_workspace_size(void) { return sizeof(Coef); }

extern "C" int pc2d_adamw_step(int state_bits, const pc2d_adamw_tensor *tensors, int count, int64_t *step,
                               const float *lr_device, double lr, double beta1, double beta2, double eps,
                               double weight_decay, const float *grad_scale, int64_t seed, void *workspace,
                               size_t workspace_bytes, void *stream) {
  return pc2d_adamw_step_numbered(state_bits, tensors, count, nullptr, step, lr_device, lr, beta1, beta2, eps,
                                  weight_decay, grad_scale, seed, workspace, workspace_bytes, stream);
}

extern "C" int pc2d_adamw_step_numbered(int state_bits, const pc2d_adamw_tensor *tensors, int count,
                                        const int64_t *numbers, int64_t *step, const float *lr_device, double lr,
                                        double beta1, double beta2, double eps, double weight_decay,
                                        const float *grad_scale, int64_t seed, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  NvtxRange range("pc2d_adamw_step");
  if (state_bits != 8 && state_bits != 32) return refuse("pc2d_adamw_step: states of 32 or 8 bits, got %d", state_bits);
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) ||
      (!lr_device && !(lr >= 0.0))) {
    set_last_error("pc2d_adamw_step: lr, eps and weight_decay must be non-negative and the betas in [0, 1)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (count < 0 || (count && !tensors)) return refuse("pc2d_adamw_step: invalid count %d or null tensors", count);
  for (int i = 0; i < count; ++i) {
    const pc2d_adamw_tensor &t = tensors[i];
    if (!seq_dtype(t.dtype) || (t.grad_dtype != t.dtype && t.grad_dtype != PC2D_DTYPE_F32))
      return refuse("pc2d_adamw_step: tensor %d: parameters of float32, float16 or bfloat16, gradients of the same or "
                    "float32", i);
    if (t.n < 0 || t.n > (int64_t)1 << 34 || t.split < 0) return refuse("pc2d_adamw_step: tensor %d: invalid size", i);
    if (numbers && (numbers[i] < 0 || numbers[i] > 0x7fffffff))
      return refuse("pc2d_adamw_step: tensor %d: its number must be from 0 to 2^31 - 1", i);
    if (!isfinite(t.rate_first) || !isfinite(t.rate_rest) || !isfinite(t.decay))
      return refuse("pc2d_adamw_step: tensor %d: factors must be finite", i);
    if (t.master && t.dtype == PC2D_DTYPE_F32) return refuse("pc2d_adamw_step: tensor %d: a float32 parameter needs no "
                                                             "master", i);
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (state_bits == 8 && !t.scales))
      return refuse("pc2d_adamw_step: tensor %d: null pointer", i);
    int st;
    if ((st = check_elements("pc2d_adamw_step", seq_dtype_size(t.dtype), {t.param})) != PC2D_OK ||
        (st = check_elements("pc2d_adamw_step", seq_dtype_size(t.grad_dtype), {t.grad})) != PC2D_OK ||
        (st = check_elements("pc2d_adamw_step", 4, {t.master})) != PC2D_OK ||
        (state_bits == 32 && (st = check_elements("pc2d_adamw_step", 4, {t.exp_avg, t.exp_avg_sq})) != PC2D_OK))
      return st;
  }
  if (!step) return refuse("pc2d_adamw_step: null step (of %d tensors)", count);
  if (!workspace || workspace_bytes < sizeof(Coef) || !aligned16(workspace)) {
    set_last_error("pc2d_adamw_step: workspace of %zu bytes on a 16-byte boundary needed", sizeof(Coef));
    return PC2D_ERR_WORKSPACE;
  }
  int st = check_elements("pc2d_adamw_step", 8, {step});
  if (st != PC2D_OK || (st = check_elements("pc2d_adamw_step", 4, {lr_device, grad_scale})) != PC2D_OK ||
      (st = pending_device_error()) != PC2D_OK)
    return st;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Coef *coef = static_cast<Coef *>(workspace);
  adamw_coef_kernel<<<1, 1, 0, s>>>(step, lr_device, (float)lr, (float)log(beta1), (float)log(beta2), coef);
  PC2D_LAUNCH_CHECK("adamw_coef_kernel");
  const Betas b{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, (float)weight_decay,
                (uint64_t)seed};
  auto group = [&](auto p, auto g, int dtype, int grad_dtype) -> int {
    return launch_group<decltype(p), decltype(g)>(state_bits, tensors, count, numbers, dtype, grad_dtype, coef, grad_scale,
                                                  b, s);
  };
  const int F = PC2D_DTYPE_F32, H = PC2D_DTYPE_F16, B = PC2D_DTYPE_BF16;
  const float f32{};
  const __half f16{};
  const __nv_bfloat16 bf16{};
  if ((st = group(f32, f32, F, F)) != PC2D_OK || (st = group(f16, f16, H, H)) != PC2D_OK ||
      (st = group(f16, f32, H, F)) != PC2D_OK || (st = group(bf16, bf16, B, B)) != PC2D_OK ||
      (st = group(bf16, f32, B, F)) != PC2D_OK)
    return st;
  return PC2D_OK;
}

extern "C" int pc2d_adamw_state_values(int dtype, const pc2d_adamw_tensor *tensors, int count, void *const *exp_avgs,
                                       void *const *exp_avg_sqs, void *stream) {
  NvtxRange range("pc2d_adamw_state_values");
  if (dtype != PC2D_DTYPE_F32 && dtype != PC2D_DTYPE_BF16)
    return refuse("pc2d_adamw_state_values: float32 or bfloat16, got dtype %d", dtype);
  if (count < 0 || (count && (!tensors || !exp_avgs || !exp_avg_sqs)))
    return refuse("pc2d_adamw_state_values: invalid count %d or null arrays", count);
  const size_t size = seq_dtype_size(dtype);
  int st;
  for (int i = 0; i < count; ++i) {
    const pc2d_adamw_tensor &t = tensors[i];
    if (t.n < 0 || t.n > (int64_t)1 << 34) return refuse("pc2d_adamw_state_values: tensor %d: invalid size", i);
    if (t.n == 0) continue;
    if (!t.exp_avg || !t.exp_avg_sq || !t.scales || !exp_avgs[i] || !exp_avg_sqs[i])
      return refuse("pc2d_adamw_state_values: tensor %d: null pointer", i);
    if ((st = check_elements("pc2d_adamw_state_values", size, {exp_avgs[i], exp_avg_sqs[i]})) != PC2D_OK) return st;
  }
  if ((st = pending_device_error()) != PC2D_OK) return st;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto take = [](const pc2d_adamw_tensor &t) { return t.n > 0; };
  auto fill = [&](Item &it, const pc2d_adamw_tensor &t) {
    const int64_t i = &t - tensors;
    it.param = exp_avgs[i];
    it.master = (float *)exp_avg_sqs[i];
    it.vec = aligned_to(it.param, 16) && aligned_to(it.master, 16) && aligned_to(t.exp_avg, 8) &&
             aligned_to(t.exp_avg_sq, 8);
  };
  auto run = [&](auto &items, unsigned grid) -> int {
    constexpr int N = sizeof(items.first) / sizeof(int);
    if (dtype == PC2D_DTYPE_F32) adamw_values_kernel<float, N><<<grid, kThreads, 0, s>>>(items);
    else adamw_values_kernel<__nv_bfloat16, N><<<grid, kThreads, 0, s>>>(items);
    PC2D_LAUNCH_CHECK("adamw_values_kernel");
    return PC2D_OK;
  };
  return in_launches(tensors, count, take, fill, run, run);
}
