// State space scan over [batch][channels][length], with N states per channel
// and inputs B, C shared by the channels of a group:
//
//   D_t = softplus(delta_t + bias)         (or delta_t + bias)
//   h_t[n] = exp(D_t A[n]) h_{t-1}[n] + D_t u_t B_t[n]
//   y_t = sum_n C_t[n] h_t[n] + skip u_t           out_t = y_t silu(z_t)
//
// Backward, with dy = dout silu(z) and a_t = exp(D_t A):
//
//   dh_t = C_t dy_t + r_t       r_{t-1} = a_t dh_t  (r behind the last token: dfinal)
//   dC_t[n] = sum_channels dy_t h_t[n]      dB_t[n] = sum_channels dh_t[n] D_t u_t
//   through_t = sum_n dh_t[n] B_t[n]        m_t[n] = r_{t-1}[n] h_{t-1}[n]
//   du_t = D_t through_t + skip dy_t        dD_t = u_t through_t + sum_n A[n] m_t[n]
//   dA[n] = sum_t D_t m_t[n]     dskip = sum dy_t u_t     dz_t = dout_t y_t silu'(z_t)
//   ddelta_t = dD_t softplus'(delta_t + bias)             dbias = sum ddelta_t
//
// P lanes share a channel and hold four of its states each (P the power of
// two that covers N); a block of 128 threads has 128 / P channels of one
// group and goes through the length in tiles.  Per tile the inputs come in by
// vectors along the length, D_t, D_t u_t (and dy_t) go to shared memory as
// 32-bit rows of the warp that uses them, B and C, which the whole block
// reads, as [t][n] so that a lane takes its four states in one 16-byte read.
// The recurrence stays in registers; sums over the states are made four (or
// eight) tokens at a time, each exchange halving what a lane still holds.
//
// The bound is the arithmetic: an exp per channel, state and token (two in
// the backward pass) at 16 a clock and SM, against 8 to 14 bytes of traffic
// per channel and token.  4 x 2048 x 2048 bf16 with 16 states and a gate take
// 181 us forwards and 494 backwards: 256 blocks are 7 warps per SM, whose
// issue slots are half used and no pipe is full; with 14 warps (one row of
// 16384 tokens in segments) 64 % are used.
//
// Few rows leave SMs empty.  Then the length is cut into segments that run at
// the same time, after a first pass that gives each segment's end state from
// zero and its sum of D_t: as the decay over a segment is exp(A sum D_t), a
// segment gets its true state from those of the segments before it.  The
// backward pass does the same with r, from the end.
//
// For the backward pass the forward one keeps the state at the start of each
// of that pass's tiles; within a tile the states are computed again.
#include <float.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace pc2d {
namespace {

constexpr int kS = 4, kH = kS / 2;  // states per lane, and pairs of them (packed registers)
constexpr int kRun = 8;             // tokens of an inner run
constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();

// How a block is laid out: P lanes per channel, and the tiles' lengths.  A
// forward tile holds whole backward ones.  kMany: for grids that fill the GPU
// several times, registers for four blocks per SM and a shorter tile; else for
// two, which the compiler spends on overlapping more of a run (16384 tokens of
// 2048 channels in 9 segments: 287 against 330 us; 4 x 2048 tokens of 2048
// channels, 1.7 blocks per SM: 209 against 184 us).
// kWhole: every row of the arrays starts on a 16-byte boundary.
template <int P_, bool kWhole_, bool kMany_ = false>
struct Layout {
  static constexpr bool kWhole = kWhole_, kMany = kMany_;
  static constexpr int P = P_, NP = kS * P, CB = kThreads / P;
  static constexpr int TF = P == 1 ? 16 : P == 2 || P >= 16 || kMany ? 32 : 64;
  static constexpr int TB = P == 1 || P >= 16 ? 16 : 32;
  static constexpr int kFwdBlocks = P >= 16 ? 2 : kMany ? 4 : 2;
};
constexpr int kBwdBlocks = 2;
inline int lanes_of(int states) {
  int p = 1;
  while (p * kS < states) p *= 2;
  return p;
}
inline int bwd_tile_of(int states) {
  const int p = lanes_of(states);
  return p == 1 || p >= 16 ? 16 : 32;
}

struct ScanArgs {
  const void *u, *delta, *z, *B, *C;
  const float *A, *skip, *bias, *init;
  const int *lengths;
  int batch, channels, length, states, groups, per_group, softplus;
  int nblk;            // blocks of channels per group
  int nseg, seg_len;   // segments of the length, in tokens
  void *out;
  float *final_state;  // [batch][channels][states]
  float *ckpt;         // [batch][tiles][channels][states], state at each backward tile's start
  float *seg_state;    // [batch][nseg][channels][states]
  float *seg_sum;      // [batch][nseg][channels]
  // backward
  const void *grad;
  const float *grad_final;
  void *du, *ddelta, *dz;
  float *dinit;
  float *part_bc;      // [batch][groups][nblk][2 states][length]: dB, then dC
  float *part_par;     // [batch * nseg][par_stride]: dA, dskip, dbias
  // rows of dA, dskip and dbias start on a 16-byte boundary
  __host__ __device__ int64_t par_stride() const { return ((int64_t)channels * (states + 2) + 3) / 4 * 4; }
};

__device__ __forceinline__ float exp2_f(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two states at a time: the packed 32-bit instructions do twice the work of
// the scalar ones per issue.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  }
  __device__ __forceinline__ float x() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return a;
  }
  __device__ __forceinline__ float y() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return b;
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Decays.  The hardware exponential is off by up to 2.4 units of 2^-24 and, on
// average over its table, low by 0.1 to 0.8 of one (measured on [-2, 0]).  A
// state that decays (or grows) slowly would add that bias up over all the tokens it
// remembers, a thousand or more.  So each tile of up to 32 tokens ends with a
// correction: what is left of the state that entered the tile, by the decays
// that were used, is replaced by exp of the tile's sum,
//   h += h_entry exp2(A2 sum d) - left,       left = h_entry a_1 a_2 ...
// and the bias no longer grows beyond a tile.  (The decays' product by itself,
// from 1 on, would not do: of (1 - a)(1 - b) the small a b is rounded off, always
// to the same side; a state's own digits round to both.  With the product,
// states that remember 20000 tokens were off by 1600 units.)  exp2_tile, for
// that one value a tile, takes 1 + x q(x) for |x| < 1/8 with the interpolation
// of (2^x - 1)/x at the four Chebyshev nodes of [-1/8, 1/8] as q (no bias where
// many tiles are remembered), else the hardware's.
__device__ __forceinline__ F2 exp2_2(F2 x) { return F2(exp2_f(x.x()), exp2_f(x.y())); }
__device__ __forceinline__ float exp2_tile(float x) {
  float q = fmaf(0.009620536f, x, 0.055524945f);
  q = fmaf(q, x, 0.2402265f);
  q = fmaf(q, x, 0.6931471f);
  return fabsf(x) < 0.125f ? fmaf(q, x, 1.f) : exp2_f(x);
}
// The same for two values.
__device__ __forceinline__ F2 exp2_tile2(F2 x) {
  F2 q = fma2(F2(0.009620536f, 0.009620536f), x, F2(0.055524945f, 0.055524945f));
  q = fma2(q, x, F2(0.2402265f, 0.2402265f));
  q = fma2(q, x, F2(0.6931471f, 0.6931471f));
  q = fma2(q, x, F2(1.f, 1.f));
  return F2(fabsf(x.x()) < 0.125f ? q.x() : exp2_f(x.x()), fabsf(x.y()) < 0.125f ? q.y() : exp2_f(x.y()));
}
// h corrected for the tile: x = A2 sum d.  Not for an infinite state, nor where
// the decays overflowed.
__device__ __forceinline__ float correct_tile(float h, float entry, float x, float left) {
  const float by = fmaf(entry, exp2_tile(x), -left);
  return fabsf(by) < kInf ? h + by : h;
}
__device__ __forceinline__ F2 correct_tile2(F2 h, F2 entry, F2 x, F2 left) {
  return F2(correct_tile(h.x(), entry.x(), x.x(), left.x()), correct_tile(h.y(), entry.y(), x.y(), left.y()));
}

// Two pairs from, and to, 16 aligned bytes.
__device__ __forceinline__ void load_pairs(const float *p, F2 (&f)[kH]) {
  const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(p);
  f[0].v = q.x;
  f[1].v = q.y;
}
__device__ __forceinline__ void put_pairs(float *p, const F2 (&f)[kH]) {
  *reinterpret_cast<ulonglong2 *>(p) = make_ulonglong2(f[0].v, f[1].v);
}
// sum of a[i] b[i] over a lane's states
__device__ __forceinline__ float dot(const F2 (&a)[kH], const F2 (&b)[kH]) {
  const F2 s = fma2(a[1], b[1], mul2(a[0], b[0]));
  return s.x() + s.y();
}
template <int n>
__device__ __forceinline__ void load_row_f(const float *p, float (&v)[n]) {
#pragma unroll
  for (int i = 0; i < n; i += 4) {
    const float4 a = *reinterpret_cast<const float4 *>(p + i);
    v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
  }
}

// softplus(v) = max(v, 0) + log(1 + e) with e = exp(-|v|), and its slope.
// exp2 takes v log2(e) in two parts, so that e is off by 3 units of 2^-24
// whatever v is; log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3, by the
// interpolation of 2 atanh(s) / s at five Chebyshev nodes of s^2 in [0, 1/9]
// (4e-9): it keeps its relative accuracy where e is small.
__device__ __forceinline__ float exp_neg_abs(float v) {
  const float a = -fabsf(v), hi = a * kLog2e;
  const float lo = fmaf(a, 1.925963033e-8f, fmaf(a, kLog2e, -hi));
  const float e = exp2_f(hi);
  return hi < -126.f ? 0.f : fmaf(e, lo * 0.6931471806f, e);
}
// softplus and its slope, the logistic function, from one exponential
__device__ __forceinline__ float softplus_f(float v, float *slope) {
  const float e = exp_neg_abs(v);
  const float s = __fdividef(e, 2.f + e), w = s * s;
  float q = fmaf(0.2815778f, w, 0.27965158f);
  q = fmaf(q, w, 0.40024596f);
  q = fmaf(q, w, 0.6666632f);
  q = fmaf(q, w, 2.f);
  *slope = __fdividef(v < 0.f ? e : 1.f, 1.f + e);
  return fmaf(q, s, fmaxf(v, 0.f));
}
__device__ __forceinline__ float softplus_f(float v) {
  float unused;
  return softplus_f(v, &unused);
}

// Sums of v0..v3 over the P lanes of a channel.  P >= 4: lane p ends with
// that of v[p % 4]; P = 2: with those of v[p] and v[p + 2]; P = 1: all four.
template <int P>
struct Sum4 {
  static constexpr int kLeft = P >= 4 ? 1 : 4 / P;
  float r[kLeft];
  __device__ __forceinline__ Sum4(float v0, float v1, float v2, float v3, int p) {
    if constexpr (P == 1) {
      r[0] = v0;
      r[1] = v1;
      r[2] = v2;
      r[3] = v3;
    } else if constexpr (P == 2) {
      const bool odd = p & 1;
      r[0] = (odd ? v1 : v0) + __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 1);
      r[1] = (odd ? v3 : v2) + __shfl_xor_sync(0xffffffffu, odd ? v2 : v3, 1);
    } else {
      const bool high = p & 2, odd = p & 1;
      float k0 = (high ? v2 : v0) + __shfl_xor_sync(0xffffffffu, high ? v0 : v2, 2);
      float k1 = (high ? v3 : v1) + __shfl_xor_sync(0xffffffffu, high ? v1 : v3, 2);
      float s = (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 1);
#pragma unroll
      for (int o = 4; o < P; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      r[0] = s;
    }
  }
  // writes the four sums to dst[0..3], each by one lane
  __device__ __forceinline__ void put(float *dst, int p) const {
    if (P > 4 && p >= 4) return;
#pragma unroll
    for (int i = 0; i < kLeft; ++i) dst[p + i * P] = r[i];
  }
};

// An array of `total` elements whose rows are read along their length.
template <typename T>
struct Rows {
  const T *array;
  int64_t total;
};

// E elements of a row, on their way: load() only issues the reads, get() gives
// the elements (0 at and behind `end`, where nothing is read).  Where rows may
// start anywhere, the aligned vectors that hold the elements are read and
// shifted by the elements before them when they are wanted; reads of single
// elements, which are packed as they arrive, would wait for each other and for
// memory (4 x 2048 x 2047 bf16 forwards: 317 us, when 2048 tokens took 181).
template <typename T, int E, bool kWhole>
struct RowLoad {
  static constexpr int V = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
  static constexpr bool kShift = !kWhole && V > 1;
  static constexpr int NV = E / V + (kShift ? 1 : 0), kPer = kShift ? V * (int)sizeof(T) / 4 : 1;
  Pack<T, V> q[NV];

  // whether the vectors can be read whole (kShift: one more than the elements fill)
  __device__ static __forceinline__ bool vectors(const Rows<T> &r, int64_t row, int t, int end) {
    return kWhole ? t + E <= end : kShift && t < end && row + t + E + V <= r.total;
  }
  __device__ __forceinline__ void load(const Rows<T> &r, int64_t row, int t, int end) {
    const int64_t at = row + t;
    if (vectors(r, row, t, end)) {
      const T *p = r.array + (kShift ? at & ~(int64_t)(V - 1) : at);
#pragma unroll
      for (int i = 0; i < NV; ++i) q[i].load(p + i * V);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) q[i / V].v[i % V] = t + i < end ? r.array[at + i] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(const Rows<T> &r, int64_t row, int t, int end, Pack<T, E> &v) const {
    if constexpr (!kShift) {
#pragma unroll
      for (int i = 0; i < E; ++i) v.v[i] = q[i / V].v[i % V];
    } else {
      // (without vectors the elements lie unshifted)
      const int m = vectors(r, row, t, end) ? (int)((row + t) & (V - 1)) : 0;
      unsigned w[NV * kPer];
#pragma unroll
      for (int i = 0; i < NV * kPer; ++i) w[i] = reinterpret_cast<const unsigned *>(q[i / kPer].v)[i % kPer];
#pragma unroll
      for (int e = V / 2; e * (int)sizeof(T) >= 4; e /= 2) {
        const int step = e * (int)sizeof(T) / 4;
#pragma unroll
        for (int i = 0; i + step < NV * kPer; ++i) w[i] = m & e ? w[i + step] : w[i];
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i + 1 < NV * kPer; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (m & 1) * 16);
      }
#pragma unroll
      for (int i = 0; i < E * (int)sizeof(T) / 4; ++i) reinterpret_cast<unsigned *>(v.v)[i] = w[i];
      if (t + E > end) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (t + i >= end) v.v[i] = from_f<T>(0.f);
      }
    }
  }
};

template <bool kWhole, typename T, int E>
__device__ __forceinline__ void store_row(const Pack<T, E> &v, T *array, int64_t row, int t, int end) {
  T *dst = array + row + t;
  if (kWhole && t + E <= end) {
    v.store(dst);
  } else if (!kWhole && sizeof(T) == 2 && E >= 2 && t + E <= end) {
    // two elements a store, from an even one on
    const int odd = (int)((row + t) & 1);
    const unsigned *w = reinterpret_cast<const unsigned *>(v.v);
    if (odd) {
      dst[0] = v.v[0];
#pragma unroll
      for (int i = 0; i + 1 < E / 2; ++i) reinterpret_cast<unsigned *>(dst + 1)[i] = __funnelshift_r(w[i], w[i + 1], 16);
      dst[E - 1] = v.v[E - 1];
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) reinterpret_cast<unsigned *>(dst)[i] = w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + i < end) dst[i] = v.v[i];
  }
}

// A lane's four values of B or C as they lie in shared memory.
template <typename T>
struct Four;
template <>
struct Four<float> {
  F2 f[kH];
  __device__ __forceinline__ void unpack(F2 (&o)[kH]) const {
    o[0] = f[0];
    o[1] = f[1];
  }
};
template <>
struct Four<__half> {
  __half2 h[kH];
  __device__ __forceinline__ void unpack(F2 (&o)[kH]) const {
#pragma unroll
    for (int i = 0; i < kH; ++i) {
      const float2 v = __half22float2(h[i]);
      o[i] = F2(v.x, v.y);
    }
  }
};
template <>
struct Four<__nv_bfloat16> {
  unsigned w[kH];
  __device__ __forceinline__ void unpack(F2 (&o)[kH]) const {
#pragma unroll
    for (int i = 0; i < kH; ++i) o[i] = F2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};

// A block's tile of B and C, loaded along the length by vectors and kept in
// their own type, a token a row: for each lane its four values of B, then of C,
// which it takes in one read (two for float).  The rows of a vector's tokens
// are followed by 16 bytes, so that the lanes of a warp, which store the same
// element of their vectors, meet different banks.
template <typename T, class G, int TT>
struct TileBC {
  static constexpr int NP = G::NP, kCount = NP * TT;
  static constexpr int kEach = kCount / kThreads > 0 ? kCount / kThreads : 1;
  static constexpr int kVec = kEach * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : kEach;
  static constexpr int kNum = kEach / kVec;
  static constexpr int kPad = 16 / (int)sizeof(T), kElems = TT * 2 * NP + TT / kVec * kPad;
  static constexpr int kFloats = (kElems * (int)sizeof(T) + 3) / 4;
  __device__ static __forceinline__ int row(int t) { return t * 2 * NP + t / kVec * kPad; }
  // row(t + j) for t a multiple of n and a constant j < n
  template <int n>
  __device__ static __forceinline__ int row_in(int t, int j) {
    return kVec < n ? row(t) + j * 2 * NP + j / kVec * kPad : row(t) + j * 2 * NP;
  }
  using Load = RowLoad<T, kVec, G::kWhole>;
  Load b[kNum], c[kNum];
  // at: where the group's first state's row begins
  __device__ __forceinline__ void load(const Rows<T> &B, const Rows<T> *C, int64_t at, int states, int length, int t0,
                                       int end) {
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int e = (i * kThreads + threadIdx.x) * kVec, n = e / TT, t = t0 + e % TT;
      const int stop = n < states && e < kCount ? end : t;  // nothing to read for missing states
      b[i].load(B, at + (int64_t)n * length, t, stop);
      if (C) c[i].load(*C, at + (int64_t)n * length, t, stop);
    }
  }
  // (with the arguments of the load)
  __device__ __forceinline__ void put(T *tile, const Rows<T> &B, const Rows<T> *C, int64_t at, int states, int length,
                                      int t0, int end) const {
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int e = (i * kThreads + threadIdx.x) * kVec, n = e / TT, t = e % TT;
      if (e < kCount) {
        const int stop = n < states ? end : t0 + t;
        T *dst = tile + row(t) + n / kS * (2 * kS) + n % kS;
        Pack<T, kVec> vb, vc;
        b[i].get(B, at + (int64_t)n * length, t0 + t, stop, vb);
        if (C) c[i].get(*C, at + (int64_t)n * length, t0 + t, stop, vc);
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          dst[k * 2 * NP] = vb.v[k];
          if (C) dst[k * 2 * NP + kS] = vc.v[k];
        }
      }
    }
  }
  struct alignas(16) Both {
    Four<T> b, c;
  };
  // the first of a lane's two; both
  __device__ static __forceinline__ Four<T> first(const T *tile, int at, int p) {
    Four<T> r;
    const T *src = tile + at + p * 2 * kS;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(src);
    else *reinterpret_cast<uint2 *>(&r) = *reinterpret_cast<const uint2 *>(src);
    return r;
  }
  __device__ static __forceinline__ Both both(const T *tile, int at, int p) {
    Both r;
    const T *src = tile + at + p * 2 * kS;
#pragma unroll
    for (int i = 0; i < (int)sizeof(Both) / 16; ++i)
      reinterpret_cast<uint4 *>(&r)[i] = reinterpret_cast<const uint4 *>(src)[i];
    return r;
  }
};

// What a thread is: lane p of a channel, in a segment of the length.
template <class G>
struct ScanPlace {
  int p, c, d, b, g, blk, seg, len;
  bool valid;
  int64_t row;   // batch row * channels + channel
  __device__ __forceinline__ ScanPlace(const ScanArgs &a) {
    p = threadIdx.x % G::P;
    c = threadIdx.x / G::P;
    int i = blockIdx.x;
    seg = i % a.nseg;
    i /= a.nseg;
    blk = i % a.nblk;
    i /= a.nblk;
    g = i % a.groups;
    b = i / a.groups;
    const int in_group = blk * G::CB + c;
    valid = in_group < a.per_group;
    // a thread without a channel computes on its group's last one and writes nothing
    d = g * a.per_group + (valid ? in_group : a.per_group - 1);
    row = (int64_t)b * a.channels + d;
    len = a.length;
    if (a.lengths) len = min(max(a.lengths[b], 0), a.length);
  }
};

// A lane's states of a channel's row of them (0 for those beyond the last).
__device__ __forceinline__ void load_states(const float *src, int states, int p, F2 (&h)[kH]) {
  if (states % kS == 0 && p * kS < states) {
    // (rows of a multiple of four states in a 16-byte aligned array)
    const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(src + p * kS);
    h[0].v = q.x;
    h[1].v = q.y;
    return;
  }
#pragma unroll
  for (int s = 0; s < kH; ++s) {
    const int n = p * kS + 2 * s;
    h[s] = F2(n < states ? src[n] : 0.f, n + 1 < states ? src[n + 1] : 0.f);
  }
}
__device__ __forceinline__ void store_states(float *dst, int states, int p, const F2 (&h)[kH]) {
  if (states % kS == 0) {
    if (p * kS < states) put_pairs(dst + p * kS, h);
  } else {
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      const int n = p * kS + 2 * s;
      if (n < states) dst[n] = h[s].x();
      if (n + 1 < states) dst[n + 1] = h[s].y();
    }
  }
}
// A log2(e); the lowest (largest) number for an infinite one, so that a step of
// d = 0, and the places of a tile that have no token, change nothing.
__device__ __forceinline__ float decay_rate(float A) {
  const float x = A * kLog2e;
  return x < -FLT_MAX ? -FLT_MAX : x > FLT_MAX ? FLT_MAX : x;
}
__device__ __forceinline__ void load_decay_rates(const float *A, int states, int p, F2 (&A2)[kH]) {
  load_states(A, states, p, A2);
#pragma unroll
  for (int s = 0; s < kH; ++s) A2[s] = F2(decay_rate(A2[s].x()), decay_rate(A2[s].y()));
}

// A segment's state after it: `own`, from zero, and the state h that entered it,
// decayed by exp2(x).  The decay may leave 32 bits where the product does not,
// so it goes in two halves then; 0 stays 0, and an infinite state infinite (as
// it would token by token), whatever the decay.
__device__ __forceinline__ float join_segment(float x, float h, float own) {
  if (h == 0.f) return own;
  if (fabsf(h) == kInf) return h + own;
  if (fabsf(x) <= 126.f) return fmaf(exp2_tile(x), h, own);
  const float half = exp2_f(0.5f * x);
  return fmaf(half, half * h, own);
}
// Takes the states h of a lane through the segments from `i` on, up to `stop` or
// down to it; state and sum: those of the row's segment 0.  (Not inlined: called
// once, it would only take registers from the kernels' loops.)
struct LaneStates {
  F2 h[kH];
};
__device__ __noinline__ LaneStates join_segments(const float *state, const float *sum, int64_t channels, int N, int p,
                                                 F2 A0, F2 A1, int i, int stop, LaneStates in) {
  const F2 A2[kH] = {A0, A1};
  const int step = i < stop ? 1 : -1;
  F2 h[kH] = {in.h[0], in.h[1]};
  float largest = 0.f;
  auto load = [&](int k, F2 (&own)[kH], F2 (&x)[kH]) {
    load_states(state + k * channels * N, N, p, own);
    const float d = sum[k * channels];
#pragma unroll
    for (int s = 0; s < kH; ++s) x[s] = mul2(F2(d, d), A2[s]);
  };
#pragma unroll 8
  for (int k = i; k != stop; k += step) {
    F2 own[kH], x[kH];
    load(k, own, x);
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      largest = fmaxf(largest, fmaxf(fabsf(h[s].x()), fabsf(h[s].y())));
      h[s] = fma2(exp2_tile2(x[s]), h[s], own[s]);
    }
  }
  // An infinity or NaN may come of a decay alone (and stays).  A decay that
  // underflows loses less than 2^-86 of what is at most 2^40.
  const float sum_of = fabsf(h[0].x()) + fabsf(h[0].y()) + fabsf(h[1].x()) + fabsf(h[1].y());
  if (!(sum_of < kInf) || largest > 0x1p40f) {
    h[0] = in.h[0];
    h[1] = in.h[1];
#pragma unroll 1
    for (int k = i; k != stop; k += step) {
      F2 own[kH], x[kH];
      load(k, own, x);
#pragma unroll
      for (int s = 0; s < kH; ++s)
        h[s] = F2(join_segment(x[s].x(), h[s].x(), own[s].x()), join_segment(x[s].y(), h[s].y(), own[s].y()));
    }
  }
  return LaneStates{{h[0], h[1]}};
}
template <class G>
__device__ __forceinline__ void enter_segment(const ScanArgs &a, const ScanPlace<G> &q, const F2 (&A2)[kH], int from,
                                              F2 (&h)[kH]) {
  if (from == q.seg) return;
  const int64_t at = (int64_t)q.b * a.nseg * a.channels + q.d;
  const LaneStates r = join_segments(a.seg_state + at * a.states, a.seg_sum + at, a.channels, a.states, q.p, A2[0],
                                     A2[1], from, q.seg, LaneStates{{h[0], h[1]}});
  h[0] = r.h[0];
  h[1] = r.h[1];
}

// Forward pass; kStateOnly: the first pass over segments (end state from zero
// and sum of D_t, no outputs).
template <typename T, class G, bool kStateOnly>
__global__ void __launch_bounds__(kThreads, G::kFwdBlocks) scan_forward_kernel(ScanArgs a) {
  constexpr int P = G::P, TT = G::TF, TB = G::TB, E = TT / P, DP = TT + 4;
  using BC = TileBC<T, G, TT>;
  __shared__ __align__(16) float s_d[G::CB * DP], s_x[G::CB * DP], s_o[kStateOnly ? 4 : G::CB * DP];
  __shared__ __align__(16) T s_bc[BC::kElems];
  const ScanPlace<G> q(a);
  const int p = q.p, N = a.states, L = a.length;
  const int64_t row = q.row * L, all = (int64_t)a.batch * a.channels * L, all_bc = (int64_t)a.batch * a.groups * N * L;
  const Rows<T> u{static_cast<const T *>(a.u), all}, dl{static_cast<const T *>(a.delta), all};
  const Rows<T> zr{static_cast<const T *>(a.z), all};
  const int64_t bg = ((int64_t)q.b * a.groups + q.g) * N * L;
  const Rows<T> B{static_cast<const T *>(a.B), all_bc}, C{static_cast<const T *>(a.C), all_bc};
  const bool z = a.z != nullptr;
  T *out = static_cast<T *>(a.out);
  const float bias = a.bias ? a.bias[q.d] : 0.f, skip = a.skip ? a.skip[q.d] : 0.f;
  const int t_begin = q.seg * a.seg_len, t_stop = min(L, t_begin + a.seg_len), t_end = min(t_stop, q.len);
  F2 A2[kH], h[kH];
  load_decay_rates(a.A + (int64_t)q.d * N, N, p, A2);
#pragma unroll
  for (int s = 0; s < kH; ++s) h[s] = F2(0.f, 0.f);
  if (!kStateOnly) {
    if (a.init) load_states(a.init + q.row * N, N, p, h);
    enter_segment(a, q, A2, 0, h);
  }
  float total = 0.f;
  float *row_d = s_d + q.c * DP, *row_x = s_x + q.c * DP, *row_o = s_o + (kStateOnly ? 0 : q.c * DP);
  RowLoad<T, E, G::kWhole> nu, nd, nz;   // the next tile's inputs, on their way
  BC nbc;
  auto fetch = [&](int t0) {
    nu.load(u, row, t0 + p * E, t_end);
    nd.load(dl, row, t0 + p * E, t_end);
    if (!kStateOnly && z) nz.load(zr, row, t0 + p * E, t_end);
    nbc.load(B, kStateOnly ? nullptr : &C, bg, N, L, t0, t_end);
  };
  if (t_begin < t_end) fetch(t_begin);
  for (int t0 = t_begin; t0 < t_stop; t0 += TT) {
    if (t0 >= t_end) {  // nothing but padding from here on
      if (!kStateOnly && q.valid) {
        Pack<T, E> o;
#pragma unroll
        for (int i = 0; i < E; ++i) o.v[i] = from_f<T>(0.f);
        store_row<G::kWhole>(o, out, row, t0 + p * E, t_stop);
      }
      continue;
    }
    Pack<T, E> cu, cd, cz;
    nu.get(u, row, t0 + p * E, t_end, cu);
    nd.get(dl, row, t0 + p * E, t_end, cd);
    if (!kStateOnly && z) nz.get(zr, row, t0 + p * E, t_end, cz);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float v = cd.f(i) + bias;
      if (a.softplus) v = softplus_f(v);
      if (t0 + p * E + i >= t_end) v = 0.f;
      row_d[p * E + i] = v;
      row_x[p * E + i] = v * cu.f(i);
    }
    nbc.put(s_bc, B, kStateOnly ? nullptr : &C, bg, N, L, t0, t_end);
    __syncthreads();
    if (t0 + TT < t_end) fetch(t0 + TT);
#pragma unroll 1
    for (int tb = 0; tb < TT; tb += TB) {
      if (!kStateOnly && a.ckpt && t0 + tb < t_end && q.valid)
        store_states(a.ckpt + (((int64_t)q.b * ((L + TB - 1) / TB) + (t0 + tb) / TB) * a.channels + q.d) * N, N, p, h);
      F2 entry[kH], left[kH];
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < kH; ++s) {
        entry[s] = left[s] = h[s];
      }
#pragma unroll 1
      for (int t = tb; t < tb + TB; t += kRun) {
        float y[kRun], dd[kRun], xx[kRun];
        load_row_f(row_d + t, dd);
        load_row_f(row_x + t, xx);
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          F2 b[kH];
          const F2 d2(dd[j], dd[j]), x2(xx[j], xx[j]);
          const int at = BC::template row_in<kRun>(t, j);
          typename BC::Both bc;
          if (kStateOnly) bc.b = BC::first(s_bc, at, p);
          else bc = BC::both(s_bc, at, p);
          bc.b.unpack(b);
          sum += dd[j];
#pragma unroll
          for (int s = 0; s < kH; ++s) {
            const F2 dec = exp2_2(mul2(d2, A2[s]));
            left[s] = mul2(left[s], dec);
            h[s] = fma2(dec, h[s], mul2(x2, b[s]));
          }
          if (!kStateOnly) {
            F2 c[kH];
            bc.c.unpack(c);
            y[j] = dot(h, c);
          }
        }
        if (!kStateOnly) {
#pragma unroll
          for (int j = 0; j < kRun; j += 4) Sum4<P>(y[j], y[j + 1], y[j + 2], y[j + 3], p).put(row_o + t + j, p);
        }
      }
#pragma unroll
      for (int s = 0; s < kH; ++s) h[s] = correct_tile2(h[s], entry[s], mul2(F2(sum, sum), A2[s]), left[s]);
      total += sum;
    }
    if (!kStateOnly) {
      __syncwarp();
      if (q.valid) {
        Pack<T, E> o;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float v = fmaf(skip, cu.f(i), row_o[p * E + i]);
          if (z) v *= cz.f(i) * sigmoid_f(cz.f(i));
          if (t0 + p * E + i >= t_end) v = 0.f;
          o.v[i] = from_f<T>(v);
        }
        store_row<G::kWhole>(o, out, row, t0 + p * E, t_stop);
      }
    }
    __syncthreads();
  }
  if (kStateOnly) {
    if (q.valid) {
      const int64_t at = ((int64_t)q.b * a.nseg + q.seg) * a.channels + q.d;
      store_states(a.seg_state + at * N, N, p, h);
      if (p == 0) a.seg_sum[at] = total;
    }
  } else if (a.final_state && q.seg == a.nseg - 1 && q.valid) {
    store_states(a.final_state + q.row * N, N, p, h);
  }
}

// First pass of the backward over segments: r from zero behind the segment,
// and the sum of D_t.
template <typename T, class G>
__global__ void __launch_bounds__(kThreads, G::kFwdBlocks) scan_carry_kernel(ScanArgs a) {
  constexpr int P = G::P, TT = G::TB, E = TT >= P ? TT / P : 1, DP = TT + 4;
  using BC = TileBC<T, G, TT>;
  __shared__ __align__(16) float s_d[G::CB * DP], s_y[G::CB * DP];
  __shared__ __align__(16) T s_c[BC::kElems];
  const ScanPlace<G> q(a);
  const int p = q.p, N = a.states, L = a.length;
  const int64_t row = q.row * L, all = (int64_t)a.batch * a.channels * L, all_bc = (int64_t)a.batch * a.groups * N * L;
  const Rows<T> dl{static_cast<const T *>(a.delta), all}, grad{static_cast<const T *>(a.grad), all};
  const Rows<T> zr{static_cast<const T *>(a.z), all}, C{static_cast<const T *>(a.C), all_bc};
  const int64_t bg = ((int64_t)q.b * a.groups + q.g) * N * L;
  const bool z = a.z != nullptr;
  const float bias = a.bias ? a.bias[q.d] : 0.f;
  F2 A2[kH], r[kH];
  load_decay_rates(a.A + (int64_t)q.d * N, N, p, A2);
#pragma unroll
  for (int s = 0; s < kH; ++s) r[s] = F2(0.f, 0.f);
  const int t_begin = q.seg * a.seg_len, t_end = min(min(L, t_begin + a.seg_len), q.len);
  float total = 0.f;
  float *row_d = s_d + q.c * DP, *row_y = s_y + q.c * DP;
  RowLoad<T, E, G::kWhole> nd, ng, nz;
  BC nc;
  auto fetch = [&](int t0) {
    if (p * E < TT) {
      nd.load(dl, row, t0 + p * E, t_end);
      ng.load(grad, row, t0 + p * E, t_end);
      if (z) nz.load(zr, row, t0 + p * E, t_end);
    }
    nc.load(C, nullptr, bg, N, L, t0, t_end);
  };
  const int last = t_begin + (t_end - t_begin - 1) / TT * TT;
  if (t_begin < t_end) fetch(last);
  for (int t0 = last; t0 >= t_begin && t_begin < t_end; t0 -= TT) {
    if (p * E < TT) {
      Pack<T, E> cd, cg, cz;
      nd.get(dl, row, t0 + p * E, t_end, cd);
      ng.get(grad, row, t0 + p * E, t_end, cg);
      if (z) nz.get(zr, row, t0 + p * E, t_end, cz);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float v = cd.f(i) + bias;
        if (a.softplus) v = softplus_f(v);
        if (t0 + p * E + i >= t_end) v = 0.f;
        row_d[p * E + i] = v;
        float dy = cg.f(i);
        if (z) dy *= cz.f(i) * sigmoid_f(cz.f(i));
        row_y[p * E + i] = dy;
      }
    }
    nc.put(s_c, C, nullptr, bg, N, L, t0, t_end);
    __syncthreads();
    if (t0 > t_begin) fetch(t0 - TT);
    F2 entry[kH], left[kH];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      entry[s] = left[s] = r[s];
    }
#pragma unroll 1
    for (int t = TT - kRun; t >= 0; t -= kRun) {
      float dd[kRun], yy[kRun];
      load_row_f(row_d + t, dd);
      load_row_f(row_y + t, yy);
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        F2 c[kH];
        BC::first(s_c, BC::template row_in<kRun>(t, j), p).unpack(c);
        const F2 d2(dd[j], dd[j]), y2(yy[j], yy[j]);
        sum += dd[j];
#pragma unroll
        for (int s = 0; s < kH; ++s) {
          const F2 dec = exp2_2(mul2(d2, A2[s]));
          left[s] = mul2(left[s], dec);
          r[s] = mul2(dec, fma2(c[s], y2, r[s]));
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kH; ++s) r[s] = correct_tile2(r[s], entry[s], mul2(F2(sum, sum), A2[s]), left[s]);
    total += sum;
    __syncthreads();
  }
  if (q.valid) {
    const int64_t at = ((int64_t)q.b * a.nseg + q.seg) * a.channels + q.d;
    store_states(a.seg_state + at * N, N, p, r);
    if (p == 0) a.seg_sum[at] = total;
  }
}

constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

template <typename T, class G>
struct BwdSmem {
  static constexpr int TT = G::TB, DP = TT + 4, kPart = 2 * G::NP + 4;
  // D, D u, dy, the slopes of softplus and of the gate, and three sums over states
  static constexpr int kRows = G::CB * DP;
  static constexpr int kStart = TT / kRun * kThreads * kS;     // states at the start of each run
  static constexpr int kBC = (TileBC<T, G, TT>::kFloats + 3) / 4 * 4;
  static constexpr int kSums = 8 * kRows + kStart + kBC + (kThreads / 32) * TT * kPart;  // dskip, dbias of each thread
  static constexpr int kFloats = kSums + 4 * kThreads;
};

// Sums of v[0..7] over the lanes of a warp that hold the same states of
// different channels (lanes i, i + P, i + 2P ...): each step halves what a
// lane holds.  Leaves kLeft values, the first of index `first`.
template <int P>
struct SumChannels {
  static constexpr int kValues = 2 * kS, kChannels = 32 / P;
  static constexpr int kLevels = log2_of(kChannels < kValues ? kChannels : kValues);
  static constexpr int kLeft = kValues >> kLevels;
  __device__ static __forceinline__ int first(int lane) {
    int f = 0;
#pragma unroll
    for (int i = 0; i < kLevels; ++i)
      if (lane & (P << i)) f += kValues >> (i + 1);
    return f;
  }
  __device__ static __forceinline__ void sum(float (&v)[kValues], int lane) {
#pragma unroll
    for (int i = 0; i < kLevels; ++i) {
      const bool hi = lane & (P << i);
      const int half = kValues >> (i + 1);
#pragma unroll
      for (int k = 0; k < half; ++k) {
        const float keep = hi ? v[half + k] : v[k], send = hi ? v[k] : v[half + k];
        v[k] = keep + __shfl_xor_sync(0xffffffffu, send, P << i);
      }
    }
    if constexpr (kLeft == 1) {
#pragma unroll
      for (int o = P << kLevels; o < 32; o <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  // with more channels than values several lanes end with the same sum: one writes it
  __device__ static __forceinline__ bool writes(int lane) { return lane < (P << kLevels); }
};

// The gradients behind the last token, in its tile: 0.
template <typename T, class G>
__device__ __noinline__ void clear_rest(const ScanArgs &a) {
  constexpr int TT = G::TB;
  const ScanPlace<G> q(a);
  const int t_begin = q.seg * a.seg_len, t_stop = min(a.length, t_begin + a.seg_len);
  const int to = min(t_stop, t_begin + (q.len - t_begin + TT - 1) / TT * TT), N = a.states, L = a.length;
  if (q.valid) {
    for (int t = q.len + q.p; t < to; t += G::P) {
      const int64_t at = q.row * L + t;
      static_cast<T *>(a.du)[at] = static_cast<T *>(a.ddelta)[at] = from_f<T>(0.f);
      if (a.z) static_cast<T *>(a.dz)[at] = from_f<T>(0.f);
    }
  }
  float *part = a.part_bc + (((int64_t)q.b * a.groups + q.g) * a.nblk + q.blk) * 2 * N * L;
  for (int n = threadIdx.x; n < 2 * N; n += kThreads)
    for (int t = q.len; t < to; ++t) part[(int64_t)n * L + t] = 0.f;
}

// A warp's shares of dA and dbias (with the channel's first lane) once more, a
// token at a time, for rows where the products of the last tile's places
// without a token were NaN.  (Conditions in the loops cost the backward pass of
// 4 x 2048 x 2048 bf16 up to a tenth.)
struct RateShares {
  F2 dA[kH];
  double dbias;
};
template <typename T, class G>
__device__ __noinline__ RateShares rate_shares(const ScanArgs &a) {
  constexpr int P = G::P, TT = G::TB;
  const ScanPlace<G> q(a);
  const int N = a.states, L = a.length, t_begin = q.seg * a.seg_len, t_end = min(min(L, t_begin + a.seg_len), q.len);
  const int64_t row = q.row * L, bg = ((int64_t)q.b * a.groups + q.g) * N * L;
  const float bias = a.bias ? a.bias[q.d] : 0.f;
  F2 A2[kH], r[kH] = {F2(0.f, 0.f), F2(0.f, 0.f)};
  load_decay_rates(a.A + (int64_t)q.d * N, N, q.p, A2);
  if (a.grad_final) load_states(a.grad_final + q.row * N, N, q.p, r);
  enter_segment(a, q, A2, a.nseg - 1, r);
  RateShares sums{{F2(0.f, 0.f), F2(0.f, 0.f)}, 0.0};
  auto at = [&](const void *array, int64_t i) { return to_f(static_cast<const T *>(array)[i]); };
  auto states_of = [&](const void *array, int t, F2 (&v)[kH]) {
    float f[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) f[s] = q.p * kS + s < N ? at(array, bg + (int64_t)(q.p * kS + s) * L + t) : 0.f;
    v[0] = F2(f[0], f[1]);
    v[1] = F2(f[2], f[3]);
  };
  auto step = [&](int t, float *slope) {
    const float d = at(a.delta, row + t) + bias;
    *slope = 1.f;
    return a.softplus ? softplus_f(d, slope) : d;
  };
#pragma unroll 1
  for (int t0 = t_begin + (t_end - t_begin - 1) / TT * TT; t0 >= t_begin; t0 -= TT) {
    const int n = min(TT, t_end - t0);
    F2 before[TT][kH], b[kH], c[kH], h[kH];
    float slope;
    load_states(a.ckpt + (((int64_t)q.b * ((L + TT - 1) / TT) + t0 / TT) * a.channels + q.d) * N, N, q.p, h);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const float d = step(t0 + j, &slope), x = d * at(a.u, row + t0 + j);
      states_of(a.B, t0 + j, b);
#pragma unroll
      for (int s = 0; s < kH; ++s) {
        before[j][s] = h[s];
        h[s] = fma2(exp2_2(mul2(F2(d, d), A2[s])), h[s], mul2(F2(x, x), b[s]));
      }
    }
    F2 tile_dA[kH] = {F2(0.f, 0.f), F2(0.f, 0.f)}, left[kH] = {r[0], r[1]}, dh[kH], m[kH];
    const F2 entry[kH] = {r[0], r[1]};
    float sum = 0.f;
#pragma unroll 1
    for (int j = n - 1; j >= 0; --j) {
      const float d = step(t0 + j, &slope);
      float dy = at(a.grad, row + t0 + j);
      if (a.z) {
        const float z = at(a.z, row + t0 + j);
        dy *= z * sigmoid_f(z);
      }
      states_of(a.B, t0 + j, b);
      states_of(a.C, t0 + j, c);
      sum += d;
#pragma unroll
      for (int s = 0; s < kH; ++s) {
        const F2 dec = exp2_2(mul2(F2(d, d), A2[s]));
        dh[s] = fma2(F2(dy, dy), c[s], r[s]);
        r[s] = mul2(dec, dh[s]);
        m[s] = mul2(r[s], before[j][s]);
        left[s] = mul2(left[s], dec);
        tile_dA[s] = fma2(m[s], F2(d, d), tile_dA[s]);
      }
      float through = dot(dh, b), moved = dot(m, A2);
#pragma unroll
      for (int o = 1; o < P; o <<= 1) {
        through += __shfl_xor_sync(0xffffffffu, through, o);
        moved += __shfl_xor_sync(0xffffffffu, moved, o);
      }
      if (q.p == 0) sums.dbias += fmaf(at(a.u, row + t0 + j), through, moved * (1.f / kLog2e)) * slope;
    }
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      sums.dA[s] = add2(sums.dA[s], tile_dA[s]);
      r[s] = correct_tile2(r[s], entry[s], mul2(F2(sum, sum), A2[s]), left[s]);
    }
  }
  return sums;
}

template <typename T, class G>
__global__ void __launch_bounds__(kThreads, kBwdBlocks)
    scan_backward_kernel(const __grid_constant__ ScanArgs a) {
  using M = BwdSmem<T, G>;
  constexpr int P = G::P, NP = G::NP;
  constexpr int TT = M::TT, E = TT >= P ? TT / P : 1, DP = M::DP;
  using BC = TileBC<T, G, TT>;
  extern __shared__ __align__(16) float smem[];
  float *s_d = smem, *s_x = s_d + M::kRows, *s_y = s_x + M::kRows;
  float *s_o = s_y + M::kRows, *s_start = s_o + 5 * M::kRows;
  T *s_bc = reinterpret_cast<T *>(s_start + M::kStart);
  float *s_part = s_start + M::kStart + M::kBC;
  const ScanPlace<G> q(a);
  const int p = q.p, N = a.states, L = a.length, lane = threadIdx.x & 31;
  const int64_t row = q.row * L, all = (int64_t)a.batch * a.channels * L, all_bc = (int64_t)a.batch * a.groups * N * L;
  const Rows<T> u{static_cast<const T *>(a.u), all}, dl{static_cast<const T *>(a.delta), all};
  const Rows<T> grad{static_cast<const T *>(a.grad), all}, zr{static_cast<const T *>(a.z), all};
  const int64_t bg = ((int64_t)q.b * a.groups + q.g) * N * L;
  const Rows<T> B{static_cast<const T *>(a.B), all_bc}, C{static_cast<const T *>(a.C), all_bc};
  const bool z = a.z != nullptr;
  T *du = static_cast<T *>(a.du), *ddl = static_cast<T *>(a.ddelta), *dz = static_cast<T *>(a.dz);
  float *part = a.part_bc + (((int64_t)q.b * a.groups + q.g) * a.nblk + q.blk) * 2 * N * L;
  const bool loads = p * E < TT;  // (more lanes than tokens of a tile)
  const float bias = a.bias ? a.bias[q.d] : 0.f, skip = a.skip ? a.skip[q.d] : 0.f;
  // dskip and dbias: a tile's sum in 32 bits, the row's in 64 (kept where it
  // takes no registers from the loops)
  double2 *sums = reinterpret_cast<double2 *>(smem + M::kSums) + threadIdx.x;
  *sums = make_double2(0.0, 0.0);
  F2 A2[kH], r[kH], dA[kH];
  // a thread without a channel has states of 0 that stay 0: nothing of the
  // channel whose inputs it reads reaches the sums over channels
  const int own = q.valid ? N : 0;
  load_decay_rates(a.A + (int64_t)q.d * N, own, p, A2);
#pragma unroll
  for (int s = 0; s < kH; ++s) r[s] = dA[s] = F2(0.f, 0.f);
  if (a.grad_final) load_states(a.grad_final + q.row * N, own, p, r);
  if (q.valid) enter_segment(a, q, A2, a.nseg - 1, r);
  const int t_begin = q.seg * a.seg_len, t_stop = min(L, t_begin + a.seg_len), t_end = min(t_stop, q.len);
  float *row_d = s_d + q.c * DP, *row_x = s_x + q.c * DP, *row_y = s_y + q.c * DP;
  float *row_sy = s_o + q.c * DP, *row_sb = row_sy + M::kRows, *row_sm = row_sb + M::kRows;
  float *row_ds = row_sm + M::kRows, *row_gs = row_ds + M::kRows;
  float *my_part = s_part + (threadIdx.x / 32) * TT * M::kPart;
  RowLoad<T, E, G::kWhole> nu, nd, ng, nz;
  F2 nh[kH];
  BC nbc;
  auto fetch = [&](int t0) {
    load_states(a.ckpt + (((int64_t)q.b * ((L + TT - 1) / TT) + t0 / TT) * a.channels + q.d) * N, own, p, nh);
    if (loads) {
      nu.load(u, row, t0 + p * E, t_end);
      nd.load(dl, row, t0 + p * E, t_end);
      ng.load(grad, row, t0 + p * E, t_end);
      if (z) nz.load(zr, row, t0 + p * E, t_end);
    }
    nbc.load(B, &C, bg, N, L, t0, t_end);
  };
  const int last_live = t_begin + (t_end - t_begin - 1) / TT * TT;
  if (t_begin < t_end) fetch(last_live);
  for (int t0 = t_begin + (t_stop - t_begin - 1) / TT * TT; t0 >= t_begin; t0 -= TT) {
    if (t0 >= t_end) {  // padding: no gradient
      if (q.valid && loads) {
        Pack<T, E> o;
#pragma unroll
        for (int i = 0; i < E; ++i) o.v[i] = from_f<T>(0.f);
        store_row<G::kWhole>(o, du, row, t0 + p * E, t_stop);
        store_row<G::kWhole>(o, ddl, row, t0 + p * E, t_stop);
        if (z) store_row<G::kWhole>(o, dz, row, t0 + p * E, t_stop);
      }
      for (int e = threadIdx.x; e < 2 * N * TT; e += kThreads) {
        const int n = e / TT, t = t0 + e % TT;
        if (t < t_stop) part[(int64_t)n * L + t] = 0.f;
      }
      continue;
    }
    Pack<T, E> cu;
    F2 h0[kH] = {nh[0], nh[1]};
    if (loads) {
      Pack<T, E> cd, cg, cz;
      nu.get(u, row, t0 + p * E, t_end, cu);
      nd.get(dl, row, t0 + p * E, t_end, cd);
      ng.get(grad, row, t0 + p * E, t_end, cg);
      if (z) nz.get(zr, row, t0 + p * E, t_end, cz);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool live = t0 + p * E + i < t_end;
        float v = cd.f(i) + bias, slope = 1.f, dy = cg.f(i);
        if (a.softplus) v = softplus_f(v, &slope);
        if (z) {
          const float zz = cz.f(i), e = sigmoid_f(zz);
          row_gs[p * E + i] = dy * (e * fmaf(zz, 1.f - e, 1.f));
          dy *= zz * e;
        }
        if (!live) v = slope = 0.f;
        row_d[p * E + i] = v;
        row_ds[p * E + i] = slope;
        // a thread without a channel adds nothing to the sums over channels
        row_x[p * E + i] = q.valid ? v * cu.f(i) : 0.f;
        row_y[p * E + i] = q.valid ? dy : 0.f;
      }
    }
    nbc.put(s_bc, B, &C, bg, N, L, t0, t_end);
    __syncthreads();
    if (t0 > t_begin) fetch(t0 - TT);
    // the states at the start of each run of kRun tokens
    float *start = s_start + threadIdx.x * kS;
    put_pairs(start, h0);
#pragma unroll 1
    for (int k = 1; k < TT / kRun; ++k) {
      float dd[kRun], xx[kRun];
      load_row_f(row_d + (k - 1) * kRun, dd);
      load_row_f(row_x + (k - 1) * kRun, xx);
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        F2 b[kH];
        BC::first(s_bc, BC::template row_in<kRun>((k - 1) * kRun, j), p).unpack(b);
        const F2 d2(dd[j], dd[j]), x2(xx[j], xx[j]);
#pragma unroll
        for (int s = 0; s < kH; ++s) h0[s] = fma2(exp2_2(mul2(d2, A2[s])), h0[s], mul2(x2, b[s]));
      }
      put_pairs(start + k * kThreads * kS, h0);
    }
    F2 tile_dA[kH], entry[kH], left[kH];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      tile_dA[s] = F2(0.f, 0.f);
      entry[s] = left[s] = r[s];
    }
#pragma unroll 1
    for (int k = TT / kRun - 1; k >= 0; --k) {
      F2 h[kRun + 1][kH], dec[kRun][kH];
      typename BC::Both bc[kRun];
      float y[kRun], s1[kRun], s2[kRun], dd[kRun], xx[kRun], yy[kRun];
      load_row_f(row_d + k * kRun, dd);
      load_row_f(row_x + k * kRun, xx);
      load_row_f(row_y + k * kRun, yy);
      load_pairs(start + k * kThreads * kS, h[0]);
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        F2 b[kH], c[kH];
        bc[j] = BC::both(s_bc, BC::template row_in<kRun>(k * kRun, j), p);
        bc[j].b.unpack(b);
        bc[j].c.unpack(c);
        const F2 d2(dd[j], dd[j]), x2(xx[j], xx[j]);
        sum += dd[j];
#pragma unroll
        for (int s = 0; s < kH; ++s) {
          dec[j][s] = exp2_2(mul2(d2, A2[s]));
          left[s] = mul2(left[s], dec[j][s]);
          h[j + 1][s] = fma2(dec[j][s], h[j][s], mul2(x2, b[s]));
        }
        y[j] = dot(h[j + 1], c);
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        F2 b[kH], c[kH], dh[kH], m[kH];
        bc[j].b.unpack(b);
        bc[j].c.unpack(c);
        const F2 d2(dd[j], dd[j]), x2(xx[j], xx[j]), dy2(yy[j], yy[j]);
        float v[2 * kS];  // dB of the lane's states, then dC
#pragma unroll
        for (int s = 0; s < kH; ++s) {
          dh[s] = fma2(dy2, c[s], r[s]);
          const F2 vb = mul2(dh[s], x2), vc = mul2(dy2, h[j + 1][s]);
          v[2 * s] = vb.x();
          v[2 * s + 1] = vb.y();
          v[kS + 2 * s] = vc.x();
          v[kS + 2 * s + 1] = vc.y();
          r[s] = mul2(dec[j][s], dh[s]);
          m[s] = mul2(r[s], h[j][s]);
          tile_dA[s] = fma2(m[s], d2, tile_dA[s]);
        }
        s1[j] = dot(dh, b);
        s2[j] = dot(m, A2);
        SumChannels<P>::sum(v, lane);
        if (SumChannels<P>::writes(lane)) {
          const int f = SumChannels<P>::first(lane);
#pragma unroll
          for (int i = 0; i < SumChannels<P>::kLeft; ++i) {
            const int idx = f + i;
            my_part[(k * kRun + j) * M::kPart + (idx / kS) * NP + p * kS + idx % kS] = v[i];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kRun; j += 4) {
        Sum4<P>(y[j], y[j + 1], y[j + 2], y[j + 3], p).put(row_sy + k * kRun + j, p);
        Sum4<P>(s1[j], s1[j + 1], s1[j + 2], s1[j + 3], p).put(row_sb + k * kRun + j, p);
        Sum4<P>(s2[j], s2[j + 1], s2[j + 2], s2[j + 3], p).put(row_sm + k * kRun + j, p);
      }
    }
    // dA: a tile's sum at a time, as what a long sum of 32-bit numbers loses
    // grows with the number of its terms
#pragma unroll
    for (int s = 0; s < kH; ++s) {
      dA[s] = add2(dA[s], tile_dA[s]);
      r[s] = correct_tile2(r[s], entry[s], mul2(F2(sum, sum), A2[s]), left[s]);
    }
    __syncwarp();
    if (q.valid && loads) {
      Pack<T, E> ou, od, oz;
      float tile_skip = 0.f, tile_bias = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        // (behind the last token D, the slopes and dy are 0)
        const float uu = cu.f(i), dy = row_y[p * E + i], through = row_sb[p * E + i];
        const float dd = fmaf(uu, through, row_sm[p * E + i] * (1.f / kLog2e)) * row_ds[p * E + i];
        ou.v[i] = from_f<T>(fmaf(row_d[p * E + i], through, skip * dy));
        od.v[i] = from_f<T>(dd);
        if (z) oz.v[i] = from_f<T>(row_gs[p * E + i] * fmaf(skip, uu, row_sy[p * E + i]));
        tile_skip = fmaf(dy, uu, tile_skip);
        tile_bias += dd;
      }
      *sums = make_double2(sums->x + tile_skip, sums->y + tile_bias);
      store_row<G::kWhole>(ou, du, row, t0 + p * E, t_stop);
      store_row<G::kWhole>(od, ddl, row, t0 + p * E, t_stop);
      if (z) store_row<G::kWhole>(oz, dz, row, t0 + p * E, t_stop);
    }
    __syncthreads();
    // the warps' sums over their channels, added in order, four states at a time
    for (int e = threadIdx.x; e < 2 * P * TT; e += kThreads) {
      const int n = e / TT * kS, t = e % TT;  // n: 0 .. 2 NP, dB's states and dC's
      const float *src = s_part + t * M::kPart + n;
      F2 v[kH];
      load_pairs(src, v);
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) {
        F2 o[kH];
        load_pairs(src + w * TT * M::kPart, o);
        v[0] = add2(v[0], o[0]);
        v[1] = add2(v[1], o[1]);
      }
      const float f[kS] = {v[0].x(), v[0].y(), v[1].x(), v[1].y()};
      const int first = n < NP ? n : n - NP;  // state
      float *dst = part + ((int64_t)(n < NP ? 0 : N) + first) * L + t0 + t;
#pragma unroll
      for (int s = 0; s < kS; ++s)
        if (first + s < N && t0 + t < t_stop) dst[(int64_t)s * L] = f[s];
    }
    // (the next tile's first barrier comes before anything overwrites s_part)
  }
  float dskip = (float)sums->x, dbias = (float)sums->y;
  if (t_begin < t_end && (t_end - t_begin) % TT != 0) {
    // The last tile went over places without a token.  D, dy and the inputs are
    // 0 there, but the state, r or skip may be infinite: then the products NaN.
    const float size = fabsf(dA[0].x()) + fabsf(dA[0].y()) + fabsf(dA[1].x()) + fabsf(dA[1].y()) + fabsf(dbias);
    if (__syncthreads_or(!(size < kInf && fabsf(skip) < kInf))) {
      const RateShares again = rate_shares<T, G>(a);
      dA[0] = again.dA[0];
      dA[1] = again.dA[1];
      dbias = (float)again.dbias;
      clear_rest<T, G>(a);
    }
  }
#pragma unroll
  for (int o = 1; o < P; o <<= 1) {
    dskip += __shfl_xor_sync(0xffffffffu, dskip, o);
    dbias += __shfl_xor_sync(0xffffffffu, dbias, o);
  }
  if (q.valid) {
    float *par = a.part_par + ((int64_t)q.b * a.nseg + q.seg) * a.par_stride();
    store_states(par + (int64_t)q.d * N, N, p, dA);
    if (p == 0) {
      par[(int64_t)a.channels * N + q.d] = dskip;
      par[(int64_t)a.channels * (N + 1) + q.d] = dbias;
    }
    if (a.dinit && q.seg == 0) store_states(a.dinit + q.row * N, N, p, r);
  }
}

// Adds up the blocks' shares of dB and dC (in 32 bits, over the blocks of a
// group) and those of dA, dskip and dbias (in 64 bits, over the batch and the
// segments).  `ways` threads share a column (V neighbouring ones of dB and dC),
// add every ways-th share and are then added in order: short chains of loads,
// many of them at a time.  A block of the first kind stays within one batch
// row and group (per_bg blocks each).
constexpr int kParThreads = 256, kParWays = 8;

template <typename T, int V>
__global__ void __launch_bounds__(kParThreads) scan_params_kernel(ScanArgs a, T *dB, T *dC, float *dA, float *dskip,
                                                                 float *dbias, unsigned bc_blocks, unsigned per_bg,
                                                                 int bc_ways) {
  __shared__ __align__(16) double sums[kParThreads * V / 2 + kParThreads / 2];
  const int N = a.states;
  if (blockIdx.x < bc_blocks) {
    const int ways = bc_ways, cols = kParThreads / ways;
    const int way = threadIdx.x / cols, col = threadIdx.x - way * cols;
    const int64_t half = (int64_t)N * a.length, per = 2 * half;
    const int64_t bg = blockIdx.x / per_bg, e = ((int64_t)(blockIdx.x - bg * per_bg) * cols + col) * V;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (e < per) {
      const float *src = a.part_bc + bg * a.nblk * per + e;
#pragma unroll 8
      for (int k = way; k < a.nblk; k += ways) {
        Pack<float, V> w;
        w.load(src + k * per);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += w.v[j];
      }
    }
    float *mine = reinterpret_cast<float *>(sums) + threadIdx.x * V;
    if (ways > 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) mine[j] = v[j];
      __syncthreads();
    }
    if (way != 0 || e >= per) return;
    for (int w = 1; w < ways; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += mine[w * cols * V + j];
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = from_f<T>(v[j]);
    o.store(e < half ? dB + bg * half + e : dC + bg * half + e - half);
    return;
  }
  constexpr int cols = kParThreads / kParWays;
  const int way = threadIdx.x / cols, col = threadIdx.x - way * cols;
  const int64_t i = (int64_t)(blockIdx.x - bc_blocks) * cols + col;
  const int64_t count = (int64_t)a.channels * (N + 2), stride = a.par_stride();
  double s = 0.0;
  if (i < count) {
#pragma unroll 8
    for (int k = way; k < a.batch * a.nseg; k += kParWays) s += a.part_par[k * stride + i];
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (way != 0 || i >= count) return;
  for (int w = 1; w < kParWays; ++w) s += sums[w * cols + col];
  const int64_t dn = (int64_t)a.channels * N;
  if (i < dn) dA[i] = (float)s;
  else if (i < dn + a.channels) {
    if (dskip) dskip[i - dn] = (float)s;
  } else if (dbias) {
    dbias[i - dn - a.channels] = (float)s;
  }
}

struct ScanStepArgs {
  const void *u, *delta, *z, *B, *C;
  const float *A, *skip, *bias;
  const int *slots;
  float *state;
  void *out;
  int batch, places, channels, states, groups, per_group, softplus, nblk;
};

// One token: reads and writes each state once (8 bytes a state: what bounds
// it).  A lane has eight states, so that what a channel needs once (softplus,
// the gate) is not computed by more lanes than need be.  All reads are on their
// way before the block learns whether it may write.
constexpr int kStepThreads = 64, kStepQuads = 2;
inline int step_lanes_of(int states) {
  int p = 1;
  while (p * kStepQuads * kS < states) p *= 2;
  return p;
}

template <typename T, int P>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(ScanStepArgs a) {
  constexpr int CB = kStepThreads / P, Q = kStepQuads;
  const int b = blockIdx.x / a.nblk, blk = blockIdx.x - b * a.nblk;
  const int p = threadIdx.x % P, d = blk * CB + threadIdx.x / P, N = a.states;
  const bool valid = d < a.channels;
  StepKind kind;
  const int place = step_place(a.slots, b, a.places, &kind);
  const int twice = step_twice(a.slots, b, place, kind);
  const int64_t i = (int64_t)b * a.channels + (valid ? d : 0);
  const int dd = valid ? d : 0, g = a.groups == 1 ? 0 : dd / a.per_group;
  float *state = a.state + ((int64_t)place * a.channels + dd) * N;
  F2 h[Q][kH];
  float y = 0.f, u = 0.f, z = 0.f;
  if (kind == kStepServed) {
    F2 A2[Q][kH];
    Pack<T, kS> vb[Q], vc[Q];
    const T *B = static_cast<const T *>(a.B) + ((int64_t)b * a.groups + g) * N;
    const T *C = static_cast<const T *>(a.C) + ((int64_t)b * a.groups + g) * N;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int n = (p * Q + k) * kS;
      if (N % kS == 0 && n < N) {
        load_pairs(state + n, h[k]);
        load_pairs(a.A + (int64_t)dd * N + n, A2[k]);
        vb[k].load(B + n);
        vc[k].load(C + n);
      } else {
        load_states(state, N, p * Q + k, h[k]);
        load_states(a.A + (int64_t)dd * N, N, p * Q + k, A2[k]);
#pragma unroll
        for (int s = 0; s < kS; ++s) {
          vb[k].v[s] = n + s < N ? B[n + s] : from_f<T>(0.f);
          vc[k].v[s] = n + s < N ? C[n + s] : from_f<T>(0.f);
        }
      }
    }
    u = to_f(static_cast<const T *>(a.u)[i]);
    float delta = to_f(static_cast<const T *>(a.delta)[i]) + (a.bias ? a.bias[dd] : 0.f);
    if (a.z) z = to_f(static_cast<const T *>(a.z)[i]);
    if (a.softplus) delta = softplus_f(delta);
    const F2 d2(delta * kLog2e, delta * kLog2e), x2(delta * u, delta * u);
    if (delta != 0.f) {  // (a step of 0 changes nothing, also where A is infinite)
#pragma unroll
      for (int k = 0; k < Q; ++k)
#pragma unroll
        for (int s = 0; s < kH; ++s)
          h[k][s] = fma2(exp2_tile2(mul2(d2, A2[k][s])), h[k][s],
                         mul2(x2, F2(vb[k].f(2 * s), vb[k].f(2 * s + 1))));
    }
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      F2 c2[kH];
#pragma unroll
      for (int s = 0; s < kH; ++s) c2[s] = F2(vc[k].f(2 * s), vc[k].f(2 * s + 1));
      y += dot(h[k], c2);
    }
  }
#pragma unroll
  for (int o = 1; o < P; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  kind = step_served(twice, kind);
  if (!valid) return;
  if (kind == kStepServed) {
#pragma unroll
    for (int k = 0; k < Q; ++k) store_states(state, N, p * Q + k, h[k]);
    if (a.skip) y = fmaf(a.skip[dd], u, y);
    if (a.z) y *= z * sigmoid_f(z);
  } else {
    y = step_nothing(kind);
  }
  if (p == 0) static_cast<T *>(a.out)[i] = from_f<T>(y);
}

// --------------------------------------------------------------------- host

PerContext<uint64_t> g_scan_attr;

// f(T{}, Layout{}) for the call's type, states and length
template <bool kWhole, typename F>
int by_type_and_states(int dtype, int states, F &&f) {
#define PC2D_LAYOUT(T)                             \
  switch (lanes_of(states)) {                      \
    case 1: return f(T{}, Layout<1, kWhole>{});    \
    case 2: return f(T{}, Layout<2, kWhole>{});    \
    case 4: return f(T{}, Layout<4, kWhole>{});    \
    case 8: return f(T{}, Layout<8, kWhole>{});    \
    case 16: return f(T{}, Layout<16, kWhole>{});  \
    default: return f(T{}, Layout<32, kWhole>{});  \
  }
  if (dtype == PC2D_DTYPE_F32) { PC2D_LAYOUT(float) }
  if (dtype == PC2D_DTYPE_F16) { PC2D_LAYOUT(__half) }
  PC2D_LAYOUT(__nv_bfloat16)
#undef PC2D_LAYOUT
}
template <typename F>
int by_type_and_layout(int dtype, int states, int length, F &&f) {
  if (length * (int64_t)seq_dtype_size(dtype) % 16 == 0) return by_type_and_states<true>(dtype, states, f);
  return by_type_and_states<false>(dtype, states, f);
}

constexpr int kMaxStates = 128;

int check_scan(const char *what, int dtype, int batch, int channels, int length, int states, int groups) {
  if (!seq_dtype(dtype)) {
    set_last_error("%s: unsupported dtype %d (float32, float16 and bfloat16)", what, dtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (batch < 0 || channels < 0 || length < 0 || states < 1 || groups < 1 || channels % groups != 0) {
    set_last_error("%s: invalid batch %d, channels %d, length %d, states %d or groups %d (channels in equal groups)",
                   what, batch, channels, length, states, groups);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (states > kMaxStates) {
    set_last_error("%s: %d states per channel (at most %d)", what, states, kMaxStates);
    return PC2D_ERR_UNSUPPORTED;
  }
  if (length > 1 << 30 || (int64_t)batch * channels > (int64_t)1 << 24) {
    set_last_error("%s: problem too large", what);
    return PC2D_ERR_UNSUPPORTED;
  }
  return PC2D_OK;
}

// Blocks and segments.  Segments cost the first pass over the inputs and its
// exps again, so the length is cut only when the rows alone leave most of the
// GPU idle, into as many as give each SM the blocks that it holds at a time
// (four forwards, two backwards) and at least two tiles of the longer (forward)
// kind each.  Two segments are not made (2 x 2048 x 2048 bf16, 128 blocks
// backwards: 358 us as it is, 326 with two).
template <bool kBackward>
void scan_split(ScanArgs *a) {
  const int CB = kThreads / lanes_of(a->states);
  a->per_group = a->channels / a->groups;
  a->nblk = std::max(1, (a->per_group + CB - 1) / CB);
  const int64_t blocks = (int64_t)a->batch * a->groups * a->nblk;
  const int sms = device_sm_count();
  constexpr int kStep = 64;  // a multiple of every tile
  a->nseg = 1;
  a->seg_len = std::max(kStep, (a->length + kStep - 1) / kStep * kStep);
  if (blocks > 0 && blocks < sms + sms / 2) {
    const int want = (int)std::min<int64_t>(64, (int64_t)sms * (kBackward ? kBwdBlocks : 4) / blocks);
    const int len = std::max(2 * kStep, (int)((((int64_t)a->length + want - 1) / want + kStep - 1) / kStep * kStep));
    const int n = std::max(1, (int)(((int64_t)a->length + len - 1) / len));
    if (n > 2) {
      a->nseg = n;
      a->seg_len = len;
    }
  }
}

size_t scan_segment_bytes(const ScanArgs &a) {
  if (a.nseg == 1) return 0;
  return align_up((size_t)a.batch * a.nseg * a.channels * a.states * 4, 256) +
         align_up((size_t)a.batch * a.nseg * a.channels * 4, 256);
}
size_t scan_part_bc_bytes(const ScanArgs &a) {
  return align_up((size_t)a.batch * a.groups * a.nblk * 2 * a.states * a.length * 4, 256);
}
size_t scan_part_par_bytes(const ScanArgs &a) {
  return align_up((size_t)a.batch * a.nseg * a.par_stride() * 4, 256);
}
char *take_segments(ScanArgs *a, char *ws) {
  if (a->nseg == 1) return ws;
  a->seg_state = reinterpret_cast<float *>(ws);
  ws += align_up((size_t)a->batch * a->nseg * a->channels * a->states * 4, 256);
  a->seg_sum = reinterpret_cast<float *>(ws);
  return ws + align_up((size_t)a->batch * a->nseg * a->channels * 4, 256);
}

int check_ws(const char *what, const void *ws, size_t got, size_t need) {
  if (got < need || (need > 0 && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255)))) {
    set_last_error("%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", what, need, got);
    return PC2D_ERR_WORKSPACE;
  }
  return PC2D_OK;
}

int check_aligned(const char *what, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (p && !aligned16(p)) {
      set_last_error("%s: arrays must be 16-byte aligned", what);
      return PC2D_ERR_INVALID_ARGUMENT;
    }
  return PC2D_OK;
}

ScanArgs scan_problem(int batch, int channels, int length, int states, int groups) {
  ScanArgs a{};
  a.batch = batch;
  a.channels = channels;
  a.length = length;
  a.states = states;
  a.groups = groups;
  return a;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" size_t pc2d_ssm_scan_checkpoint_size(int batch, int channels, int length, int states) {
  if (check_scan("pc2d_ssm_scan_checkpoint_size", PC2D_DTYPE_F32, batch, channels, length, states, 1) != PC2D_OK)
    return 0;
  const int tile = bwd_tile_of(states);
  return (size_t)batch * (((size_t)length + tile - 1) / tile) * channels * states * sizeof(float);
}

extern "C" size_t pc2d_ssm_scan_forward_workspace_size(int batch, int channels, int length, int states, int groups) {
  if (check_scan("pc2d_ssm_scan_forward_workspace_size", PC2D_DTYPE_F32, batch, channels, length, states, groups) !=
      PC2D_OK)
    return 0;
  ScanArgs a = scan_problem(batch, channels, length, states, groups);
  scan_split<false>(&a);
  return scan_segment_bytes(a);
}

extern "C" int pc2d_ssm_scan_forward(int dtype, const void *u, const void *delta, const float *A, const void *B,
                                     const void *C, const float *skip, const void *z, const float *delta_bias,
                                     const float *initial_state, const int *lengths, int delta_softplus, int batch,
                                     int channels, int length, int states, int groups, void *output,
                                     float *final_state, float *checkpoints, void *workspace, size_t workspace_bytes,
                                     void *stream) {
  NvtxRange range("pc2d_ssm_scan_forward");
  int st = check_scan("pc2d_ssm_scan_forward", dtype, batch, channels, length, states, groups);
  if (st != PC2D_OK) return st;
  if ((st = pending_device_error()) != PC2D_OK) return st;
  if (batch == 0 || channels == 0) return PC2D_OK;
  if (!A || (length > 0 && (!u || !delta || !B || !C || !output))) {
    set_last_error("pc2d_ssm_scan_forward: null pointer (u, delta, A, B, C or output)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_aligned("pc2d_ssm_scan_forward",
                          {u, delta, z, B, C, output, initial_state, final_state, checkpoints, A})) != PC2D_OK ||
      (st = check_elements("pc2d_ssm_scan_forward", 4, {skip, delta_bias, lengths})) != PC2D_OK)
    return st;
  ScanArgs a = scan_problem(batch, channels, length, states, groups);
  scan_split<false>(&a);
  if ((st = check_ws("pc2d_ssm_scan_forward", workspace, workspace_bytes, scan_segment_bytes(a))) != PC2D_OK) return st;
  a.u = u; a.delta = delta; a.z = z; a.B = B; a.C = C;
  a.A = A; a.skip = skip; a.bias = delta_bias; a.init = initial_state; a.lengths = lengths;
  a.softplus = delta_softplus != 0;
  a.out = output; a.final_state = final_state; a.ckpt = checkpoints;
  take_segments(&a, static_cast<char *>(workspace));
  const unsigned grid = (unsigned)((int64_t)batch * groups * a.nblk * a.nseg);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return by_type_and_layout(dtype, states, length, [&](auto t, auto layout) -> int {
    using T = decltype(t);
    using G = decltype(layout);
    if (a.nseg > 1) {
      scan_forward_kernel<T, G, true><<<grid, kThreads, 0, s>>>(a);
      PC2D_LAUNCH_CHECK("scan_forward_kernel (segments)");
    }
    // more blocks than two per SM: the layout for four (the rule goes by the grid; rows of a ragged batch that end
    // early may leave less, and then it costs up to a tenth: 7 x 1002 channels of 24 states over up to 777 tokens,
    // fp16, 91 against 84 us; with all 777 in every row 131 against 157)
    if constexpr (G::P == 4 || G::P == 8) {
      if (grid > 2u * device_sm_count()) {
        scan_forward_kernel<T, Layout<G::P, G::kWhole, true>, false><<<grid, kThreads, 0, s>>>(a);
        PC2D_LAUNCH_CHECK("scan_forward_kernel (many blocks)");
        return PC2D_OK;
      }
    }
    scan_forward_kernel<T, G, false><<<grid, kThreads, 0, s>>>(a);
    PC2D_LAUNCH_CHECK("scan_forward_kernel");
    return PC2D_OK;
  });
}

extern "C" size_t pc2d_ssm_scan_backward_workspace_size(int batch, int channels, int length, int states, int groups) {
  if (check_scan("pc2d_ssm_scan_backward_workspace_size", PC2D_DTYPE_F32, batch, channels, length, states, groups) !=
      PC2D_OK)
    return 0;
  ScanArgs a = scan_problem(batch, channels, length, states, groups);
  scan_split<true>(&a);
  return scan_segment_bytes(a) + scan_part_bc_bytes(a) + scan_part_par_bytes(a);
}

extern "C" int pc2d_ssm_scan_backward(int dtype, const void *grad, const float *grad_final, const void *u,
                                      const void *delta, const float *A, const void *B, const void *C,
                                      const float *skip, const void *z, const float *delta_bias, const int *lengths,
                                      const float *checkpoints, int delta_softplus, int batch, int channels,
                                      int length, int states, int groups, void *ugrad, void *deltagrad, float *Agrad,
                                      void *Bgrad, void *Cgrad, float *skipgrad, void *zgrad, float *biasgrad,
                                      float *initialgrad, void *workspace, size_t workspace_bytes, void *stream) {
  NvtxRange range("pc2d_ssm_scan_backward");
  int st = check_scan("pc2d_ssm_scan_backward", dtype, batch, channels, length, states, groups);
  if (st != PC2D_OK) return st;
  if ((st = pending_device_error()) != PC2D_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (channels == 0) {  // B and C reach nothing
    const size_t bytes = (size_t)batch * groups * states * length * seq_dtype_size(dtype);
    if (bytes && Bgrad) PC2D_CUDA_CHECK(cudaMemsetAsync(Bgrad, 0, bytes, s));
    if (bytes && Cgrad) PC2D_CUDA_CHECK(cudaMemsetAsync(Cgrad, 0, bytes, s));
    return PC2D_OK;
  }
  const bool any = batch > 0 && length > 0;
  if (!A || !Agrad || (any && (!grad || !u || !delta || !B || !C || !checkpoints || !ugrad || !deltagrad || !Bgrad ||
                               !Cgrad || (z && !zgrad)))) {
    set_last_error("pc2d_ssm_scan_backward: null pointer");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_aligned("pc2d_ssm_scan_backward", {grad, u, delta, z, B, C, ugrad, deltagrad, Bgrad, Cgrad, zgrad, checkpoints,
                                                     grad_final, initialgrad, A})) != PC2D_OK ||
      (st = check_elements("pc2d_ssm_scan_backward", 4,
                           {skip, delta_bias, lengths, Agrad, skipgrad, biasgrad})) != PC2D_OK)
    return st;
  ScanArgs a = scan_problem(batch, channels, length, states, groups);
  scan_split<true>(&a);
  const size_t need = scan_segment_bytes(a) + scan_part_bc_bytes(a) + scan_part_par_bytes(a);
  if ((st = check_ws("pc2d_ssm_scan_backward", workspace, workspace_bytes, need)) != PC2D_OK) return st;
  a.u = u; a.delta = delta; a.z = z; a.B = B; a.C = C;
  a.A = A; a.skip = skip; a.bias = delta_bias; a.lengths = lengths;
  a.softplus = delta_softplus != 0;
  a.ckpt = const_cast<float *>(checkpoints);
  a.grad = grad; a.grad_final = grad_final;
  a.du = ugrad; a.ddelta = deltagrad; a.dz = zgrad; a.dinit = initialgrad;
  char *ws = take_segments(&a, static_cast<char *>(workspace));
  a.part_bc = reinterpret_cast<float *>(ws);
  a.part_par = reinterpret_cast<float *>(ws + scan_part_bc_bytes(a));
  const unsigned grid = (unsigned)((int64_t)batch * groups * a.nblk * a.nseg);
  return by_type_and_layout(dtype, states, length, [&](auto t, auto layout) -> int {
    using T = decltype(t);
    using G = decltype(layout);
    if (grid > 0) {
      constexpr int bytes = BwdSmem<T, G>::kFloats * 4;
      // one bit per instance: 3 types x 6 lane counts x 2
      int bit = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 1 : 2;
      bit += 3 * log2_of(G::P) + (G::kWhole ? 0 : 18);
      const int attr = once_per_context(g_scan_attr, (uint64_t)1 << bit, []() -> int {
        PC2D_CUDA_CHECK(cudaFuncSetAttribute(scan_backward_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             bytes));
        return PC2D_OK;
      });
      if (attr != PC2D_OK) return attr;
      if (a.nseg > 1) {
        scan_carry_kernel<T, G><<<grid, kThreads, 0, s>>>(a);
        PC2D_LAUNCH_CHECK("scan_carry_kernel");
      }
      scan_backward_kernel<T, G><<<grid, kThreads, bytes, s>>>(a);
      PC2D_LAUNCH_CHECK("scan_backward_kernel");
    }
    const int ways = a.nblk >= 16 ? 8 : a.nblk >= 8 ? 4 : a.nblk >= 4 ? 2 : 1;
    const int64_t half = (int64_t)states * length;
    const bool four = half % 4 == 0;  // then every row of dB and dC starts on a vector of four
    const unsigned per_bg = (unsigned)ceil_div(2 * half, (int64_t)kParThreads / ways * (four ? 4 : 1));
    const unsigned bc = per_bg * (unsigned)(batch * groups);
    const unsigned par = (unsigned)ceil_div((int64_t)channels * (states + 2), kParThreads / kParWays);
    if (four)
      scan_params_kernel<T, 4><<<bc + par, kParThreads, 0, s>>>(a, static_cast<T *>(Bgrad), static_cast<T *>(Cgrad),
                                                               Agrad, skipgrad, biasgrad, bc, per_bg, ways);
    else
      scan_params_kernel<T, 1><<<bc + par, kParThreads, 0, s>>>(a, static_cast<T *>(Bgrad), static_cast<T *>(Cgrad),
                                                               Agrad, skipgrad, biasgrad, bc, per_bg, ways);
    PC2D_LAUNCH_CHECK("scan_params_kernel");
    return PC2D_OK;
  });
}

extern "C" int pc2d_ssm_scan_step(int dtype, const void *u, const void *delta, float *state, const float *A,
                                  const void *B, const void *C, const float *skip, const void *z,
                                  const float *delta_bias, const int *slots, int delta_softplus, int batch, int places,
                                  int channels, int states, int groups, void *output, void *stream) {
  NvtxRange range("pc2d_ssm_scan_step");
  int st = check_scan("pc2d_ssm_scan_step", dtype, batch, channels, 1, states, groups);
  if (st != PC2D_OK) return st;
  if (places < 0 || (!slots && batch > places)) {
    set_last_error("pc2d_ssm_scan_step: %d rows of a batch without slots, but %d states", batch, places);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = pending_device_error()) != PC2D_OK) return st;
  if (batch == 0 || channels == 0) return PC2D_OK;
  if (!u || !delta || (!state && places > 0) || !A || !B || !C || !output) {
    set_last_error("pc2d_ssm_scan_step: null pointer (u, delta, state, A, B, C or output)");
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_aligned("pc2d_ssm_scan_step", {state, A, B, C})) != PC2D_OK ||
      (st = check_elements("pc2d_ssm_scan_step", seq_dtype_size(dtype), {u, delta, z, output})) != PC2D_OK ||
      (st = check_elements("pc2d_ssm_scan_step", 4, {skip, delta_bias, slots})) != PC2D_OK)
    return st;
  ScanStepArgs a{};
  a.u = u; a.delta = delta; a.z = z; a.B = B; a.C = C; a.A = A; a.skip = skip; a.bias = delta_bias;
  a.slots = slots; a.state = state; a.out = output;
  a.batch = batch; a.places = places; a.channels = channels; a.states = states; a.groups = groups;
  a.per_group = channels / groups;
  a.softplus = delta_softplus != 0;
  const int cb = kStepThreads / step_lanes_of(states);
  a.nblk = (channels + cb - 1) / cb;
  // (as many lanes as a layout for that many states' quads has)
  return by_type_and_states<true>(dtype, step_lanes_of(states) * kS, [&](auto t, auto layout) -> int {
    scan_step_kernel<decltype(t), decltype(layout)::P>
        <<<(unsigned)((int64_t)a.nblk * batch), kStepThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    PC2D_LAUNCH_CHECK("scan_step_kernel");
    return PC2D_OK;
  });
}
