// Linear attention with a decay for each head.  Per batch row and head, over
// tokens t with queries and keys of dk and values of dv numbers:
//
//   S_t = exp(g_t) S_(t-1) + k_t v_t^T        (dk x dv, in 32 bits)
//   o_t = scale S_t^T q_t
//
// Whole sequences go by chunks of C tokens.  With b_t the sum of the g of a
// chunk's tokens up to t, S the state before the chunk and b_C the whole sum:
//
//   o_t = scale (exp(b_t) S^T q_t + sum_(s <= t) exp(b_t - b_s) (q_t k_s) v_s)
//   S' = exp(b_C) S + sum_s exp(b_C - b_s) k_s v_s^T
//
// which are matrix products.  The b are kept as pairs of 32-bit numbers, so that
// a difference b_t - b_s is off by a rounding of itself and not of the b, which
// may be far larger.  (In 64 bits, which are slow on this GPU, the chain of sums
// and an exponential took longer than a chunk's products.)  A decay to nothing
// (g = -inf) counts as -kNothing, whose exponential is 0 too.
//
// Gradients, with D_t that of S_t and do_t that of o_t:
//
//   D_t = exp(g_(t+1)) D_(t+1) + scale q_t do_t^T
//   dq_t = scale S_t do_t,  dk_t = D_t v_t,  dv_t = D_t^T k_t
//   dg_t = exp(g_t) <S_(t-1), D_t>: every pair of a token (or the entering
//          state) before t and a token (or the leaving state) from t on
//
// The matrix products run on 16-bit matrix instructions, with 32-bit operands
// taken apart into `planes`, numbers of 8 bits of mantissa whose sum they are
// (bfloat16: one plane for the inputs; float16, of 11 bits: two; float32:
// three), and the products of planes that matter: mma.sync with operands that
// stay in registers from one product to the next.  (bfloat16 planes and not
// float16 ones for float16 inputs too: states and scores outgrow its range.)
// The state, which is scaled at every chunk and multiplied as an operand of the
// next product, never leaves a warp's registers that way; in tensor memory
// (tcgen05) it would be read, scaled, split and written again for each.
//
// Measured (one B200).  4 rows of 32 heads of 64 at 2048 tokens, bfloat16, a
// training step: 474 us, of these outputs 101, states of the segments 37,
// gradients' states 38 + 44, gradients 250.  16 heads of 128 at 16384 tokens:
// 337 us, states of the segments 100 (tensor pipe half busy: it multiplies
// three planes), outputs 242 (each kernel's time from a cold cache).  Everywhere the steps from one product to the
// next (loads from shared memory, splits, exponentials) leave the tensor pipe
// idle; what helped was more warps for an SM, fewer instructions between
// products (no calls, fixed strides) and no 64-bit arithmetic.
#include <math.h>

#include <algorithm>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace pc2d {
namespace {

constexpr int kMaxDim = 128;
constexpr float kNothing = 1e5f;  // in powers of two: exp2(-1e5) is 0 in 32 bits

// How many planes the operands of a type have: its inputs; scores and states
// that meet inputs in the outputs; the decayed values in the state's update,
// whose result is a state of 32 bits; states in the backward pass, whose
// products make the decays' gradients of 32 bits.  With bfloat16 a score or
// state is off by 2^-15 of itself at most, so that outputs are rounded once, to
// their type, as far as that shows (errors in norm 1.67e-3, which the rounding
// alone has too; with one plane, 2^-8, 2.35e-3, and a training step of 4 rows of
// 32 heads of 64 at 2048 tokens 448 us instead of 468).
template <typename T>
struct Planes;
template <>
struct Planes<__nv_bfloat16> {
  static constexpr int in = 1, out = 2, update = 3, back = 3, chunk = 64;
};
template <>
struct Planes<__half> {
  static constexpr int in = 2, out = 2, update = 3, back = 3, chunk = 32;
};
template <>
struct Planes<float> {
  static constexpr int in = 3, out = 3, update = 3, back = 3, chunk = 32;
};

struct Args {
  const void *q, *k, *v, *grad;
  const float *g;
  int64_t g_batch, g_head, g_token;  // strides
  const float *initial, *last_grad;
  const int *lengths;
  void *out;            // o
  float *final_state;   // or the gradient of the initial one
  float *states;        // [batch][heads][chunks][dk][dv]: S before each chunk
  float *dstates;       // likewise: D behind each chunk
  float *starts;        // [batch][heads][segments][dk][dv]: of segments, then their starts
  float *decays;        // [batch][heads][segments]: a segment's decay
  void *dq, *dk_, *dv_;
  float *dq_heads, *dk_heads;  // [batch][heads][dk][length] where heads share queries and keys
  float *dg;            // [batch][heads][length]
  int batch, heads, groups, length, dk, dv, chunks;
  int slabs, slab;      // of values
  int segments, per_segment;  // chunks of a segment
  float scale;
  bool vec;             // rows start on a vector's boundary
};

// ---------------------------------------------------------------- instructions

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pair(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ float2 unpair(uint32_t p) {
  return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
// Two numbers as N planes: upper halves, of 8 bits of mantissa, and the rests'
// in turn; the last one is rounded.  (The rest of an infinity is NaN.)
template <int N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + 1 == N) {
      p[i] = pair(x, y);
    } else {
      const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
      p[i] = __byte_perm(u, v, 0x7632);
      x -= __uint_as_float(u & 0xffff0000u);
      y -= __uint_as_float(v & 0xffff0000u);
    }
  }
}

// A matrix in shared memory: rows of RB bytes (0: of `bytes`, 128 or 256) of
// 16-bit numbers, their 16-byte pieces exchanged within the row so that the eight
// rows of an ldmatrix are in different banks.  Planes follow one another.
template <int RB>
struct Tile {
  uint32_t at;
  int plane, bytes;
  __device__ __forceinline__ Tile(uint32_t at, int plane, int bytes = RB) : at(at), plane(plane), bytes(bytes) {}
  __device__ __forceinline__ int row_bytes() const { return RB ? RB : bytes; }
  static __device__ __forceinline__ int turn(int row) { return RB == 64 ? row >> 1 & 3 : row & 7; }
  __device__ __forceinline__ uint32_t piece(int row, int col8, int p = 0) const {
    return at + p * plane + row * row_bytes() + ((col8 ^ turn(row)) << 4);
  }
  // The address that this lane gives an ldmatrix of the 16x16 numbers at (row, col), both multiples of 16: of its
  // four 8x8 parts, the second one to the right (kRight) or below.
  template <bool kRight>
  __device__ __forceinline__ uint32_t part(int row, int col, int p) const {
    const int lane = threadIdx.x & 31, w = lane & 7, i = lane >> 3, down = kRight ? i >> 1 : i & 1, right = kRight ? i & 1 : i >> 1;
    return at + (down * 8 + w) * row_bytes() + p * plane + row * row_bytes() + ((col >> 3 ^ (right ^ turn(w))) << 4);
  }
};
// The 16x16 operand A (rows m, columns k) of a product, stored [m][k] or (trans) [k][m].
template <bool kTrans, int RB>
__device__ __forceinline__ void load_a(uint32_t (&r)[4], const Tile<RB> &t, int m, int k, int p) {
  if (kTrans) ldsm_t(r, t.template part<true>(k, m, p));
  else ldsm(r, t.template part<false>(m, k, p));
}
// The 16x16 operand B (rows k, columns n), stored [n][k] or (trans) [k][n]:
// r[0], r[1] are the first 8 columns', r[2], r[3] the others'.
template <bool kTrans, int RB>
__device__ __forceinline__ void load_b(uint32_t (&r)[4], const Tile<RB> &t, int k, int n, int p) {
  if (kTrans) ldsm_t(r, t.template part<false>(k, n, p));
  else ldsm(r, t.template part<true>(n, k, p));
}
// c0 and c1 += A times the two halves of B, for the planes' products that are
// not below the last plane of the finer operand (all of them for two planes,
// whose last product would be the largest one left out).  The matrix unit cuts
// its sums off instead of rounding them, by about half a unit each time and all
// to one side, so that long chains of sums drift: with kApart all but the
// largest of the products have sums of their own, l0 and l1, which are small.
template <bool kApart, int NA, int NB>
__device__ __forceinline__ void product(float (&c0)[4], float (&c1)[4], float (&l0)[4], float (&l1)[4],
                                        const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
  constexpr int most = NA == 2 && NB == 2 ? 3 : NA > NB ? NA : NB;
  // (small ones first)
#pragma unroll
  for (int sum = most - 1; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == sum) {
          mma(kApart && sum ? l0 : c0, a[i], b[j][0], b[j][1]);
          mma(kApart && sum ? l1 : c1, a[i], b[j][2], b[j][3]);
        }
}
template <int M>
__device__ __forceinline__ void join(float (&c)[M][4], const float (&l)[M][4]) {
#pragma unroll
  for (int j = 0; j < M; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[j][e] += l[j][e];
}
template <bool kTrans, int N, int RB>
__device__ __forceinline__ void load_a(uint32_t (&r)[N][4], const Tile<RB> &t, int m, int k) {
#pragma unroll
  for (int p = 0; p < N; ++p) load_a<kTrans>(r[p], t, m, k, p);
}
template <bool kTrans, int N, int RB>
__device__ __forceinline__ void load_b(uint32_t (&r)[N][4], const Tile<RB> &t, int k, int n) {
#pragma unroll
  for (int p = 0; p < N; ++p) load_b<kTrans>(r[p], t, k, n, p);
}

// A chunk's scores: the 16x16 blocks on and below the diagonal, in P planes.  Of 64 tokens, rows of 1 to 4 blocks,
// two planes lie in 80 rows of 128 bytes instead of 128 (with these a fourth block of an SM would not fit for 128 keys:
// 16384 tokens of 16 heads of 128 432 us instead of 337): a plane's rows of one and of three blocks side by side, its
// four-block rows below them, and at last the two-block rows of both planes side by side.
template <int C, int P>
struct Scores {
  static constexpr bool kPacked = C == 64 && P == 2;
  static constexpr int kBytes = kPacked ? 80 * 128 : P * C * 2 * C;
  Tile<2 * C> t;
  __device__ __forceinline__ explicit Scores(uint32_t at) : t(at, C * 2 * C) {}
  // where the block (row, col) of plane p is: a block of `t`, in its plane 0 if packed
  static __device__ __forceinline__ void place(int row, int col, int p, int &r, int &c) {
    r = !kPacked ? row : row == 1 ? 4 : 2 * p + (row == 3);
    c = !kPacked ? col : row == 1 ? 2 * p + col : col + (row == 2);
  }
  __device__ __forceinline__ uint32_t piece(int row, int col8, int p) const {
    int r, c;
    place(row >> 4, col8 >> 1, p, r, c);
    return t.piece(r * 16 + (row & 15), c * 2 + (col8 & 1), kPacked ? 0 : p);
  }
  // the operand B of tokens s as its rows k and tokens `at` as its columns n, both as blocks
  __device__ __forceinline__ void load(uint32_t (&b)[P][4], int s, int at) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      int r, c;
      place(at, s, p, r, c);
      load_b<false>(b[p], t, c * 16, r * 16, kPacked ? 0 : p);
    }
  }
};

// Scores beyond the causal border are zeros that a product multiplies, which an
// infinity or NaN on the other side would turn into NaN for tokens that it does
// not reach.  Only the 16x16 blocks on the border hold such zeros: where A has
// a value that is not finite, these are summed one by one instead.
__device__ __forceinline__ bool any_not_finite(const uint32_t (&a)[4]) {
  // (infinities and NaN times zero are NaN, all others +0 after the sums)
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  __nv_bfloat162 x = zero;
#pragma unroll
  for (int i = 0; i < 4; ++i) x = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&a[i]), zero, x);
  return __any_sync(0xffffffffu, *reinterpret_cast<const uint32_t *>(&x) != 0u);
}
template <int N, typename Matrix>
__device__ __forceinline__ float number(const Matrix &t, int row, int col) {
  float x = 0.f;
#pragma unroll
  for (int p = N - 1; p >= 0; --p) {
    unsigned short u;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(t.piece(row, col / 8, p) + (col & 7) * 2));
    x += __uint_as_float((unsigned)u << 16);
  }
  return x;
}
// c0, c1 += x[rows m ..][tokens at ..] times the border's scores: of a token
// and those up to it (kUpTo), or of a token and those from it on.
// (Inline and not unrolled: a call would keep c0 and c1 in memory.)
template <int N, int M, bool kUpTo, int RB, typename Matrix>
__device__ __forceinline__ void border(float (&c0)[4], float (&c1)[4], const Tile<RB> &x, int m, const Matrix &scores,
                                       int at) {
  const int lane = threadIdx.x & 31, gr = lane >> 2, gc = lane & 3;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    const int row = m + gr + (e >> 1 & 1) * 8, mine = (e >> 2) * 8 + 2 * gc + (e & 1);
    float s = 0.f;
#pragma unroll 1
    for (int i = kUpTo ? 0 : mine; i < (kUpTo ? mine + 1 : 16); ++i)
      s += number<N>(x, row, at + i) *
           (kUpTo ? number<M>(scores, at + mine, at + i) : number<M>(scores, at + i, at + mine));
#pragma unroll
    for (int f = 0; f < 4; ++f) {  // (no register is indexed by a variable)
      c0[f] += e == f ? s : 0.f;
      c1[f] += e == f + 4 ? s : 0.f;
    }
  }
}

// ----------------------------------------------------------------- chunks

// Fills a tile [rows16][C] with tokens t0 .. t0+n-1 of an array [rows][length];
// zeros elsewhere.  bfloat16 on a vector's boundary comes by asynchronous
// copies.
template <typename T, int C>
__device__ __forceinline__ void fill(const Tile<2 * C> &t, const T *src, int rows, int rows16, int64_t length, int64_t t0, int n,
                                     bool vec) {
  constexpr int N = Planes<T>::in;
  if (N == 1 && vec && n == C) {  // whole chunks: few instructions a copy
    const int c8 = threadIdx.x % (C / 8), step = blockDim.x / (C / 8);
    const T *from = src + (threadIdx.x / (C / 8)) * length + t0 + c8 * 8;
    int row = threadIdx.x / (C / 8);
    for (; row < rows; row += step, from += step * length) copy16(t.piece(row, c8), from);
    for (; row < rows16; row += step)
      asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(t.piece(row, c8)), "r"(0) : "memory");
    return;
  }
  for (int i = threadIdx.x; i < rows16 * (C / 8); i += blockDim.x) {
    const int row = i / (C / 8), c8 = i % (C / 8), left = row < rows ? n - c8 * 8 : 0;
    const T *from = src + row * length + t0 + c8 * 8;
    if (N == 1 && vec && left >= 8) {
      copy16(t.piece(row, c8), from);
      continue;
    }
    Pack<T, 8> x;
    if (vec && left >= 8) {
      x.load(from);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = j < left ? from[j] : from_f<T>(0.f);
    }
    uint32_t p[4][N];
#pragma unroll
    for (int j = 0; j < 4; ++j) split<N>(x.f(2 * j), x.f(2 * j + 1), p[j]);
#pragma unroll
    for (int q = 0; q < N; ++q)
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(t.piece(row, c8, q)), "r"(p[0][q]), "r"(p[1][q]),
                   "r"(p[2][q]), "r"(p[3][q])
                   : "memory");
  }
}

// A number as the sum of two, the second below half a unit of the first.
__device__ __forceinline__ float2 two_sum(float a, float b) {
  const float s = a + b, t = s - a;
  return make_float2(s, (a - (s - t)) + (b - t));
}
__device__ __forceinline__ float2 two_sum(float2 a, float2 b) {
  const float2 s = two_sum(a.x, b.x);
  const float low = s.y + (a.y + b.y), hi = s.x + low;
  return make_float2(hi, low - (hi - s.x));
}
// 2^x of a pair, off by little more than half a unit: 2^n (1 + y + y^2 q(y)),
// y = ln 2 (x - n) at most 0.35, by the exponential's series, its last two sums
// with their roundings.  A state passes through this factor at every chunk.
__device__ __forceinline__ float exp2_pair(float2 x) {
  const float n = rintf(x.x), f = x.x - n;
  constexpr float ln2 = 0.693147182464599609f, ln2_low = -1.904654323148236e-9f;
  const float y = f * ln2, y_low = fmaf(f, ln2, -y) + fmaf(f, ln2_low, x.y * ln2);
  float q = 2.48015873e-5f;  // 1/8!
  q = fmaf(q, y, 1.98412698e-4f);
  q = fmaf(q, y, 1.38888889e-3f);
  q = fmaf(q, y, 8.33333333e-3f);
  q = fmaf(q, y, 4.16666667e-2f);
  q = fmaf(q, y, 1.66666667e-1f);
  q = fmaf(q, y, 0.5f);
  const float2 s = two_sum(y, fmaf(y * y, q, y_low));
  const float2 r = two_sum(1.f, s.x);
  return ldexpf(r.x + (r.y + s.y), (int)fminf(fmaxf(n, -1000.f), 1000.f));
}

// What a chunk's decays come to, in powers of two.
template <int C>
struct Decays {
  float2 at[C];               // b_t as a pair
  alignas(8) float begin[C];  // exp2(b_t)
  alignas(8) float end[C];    // exp2(b_C - b_t)
  float whole;         // exp2(b_C)
  float2 sum;          // b_C
  // log2 of exp(b_t - b_s)
  static __device__ __forceinline__ float between(float2 t, float2 s) { return (t.x - s.x) + (t.y - s.y); }
};
// A warp's share of the decays of tokens t0 .. t0+n-1, loaded ahead.
template <int C>
struct DecayLoad {
  float v[C / 32];
  __device__ __forceinline__ void load(const Args &a, int b, int h, int64_t t0, int n) {
    const float *g = a.g + b * a.g_batch + h * a.g_head;
#pragma unroll
    for (int i = 0; i < C / 32; ++i) {
      const int t = (threadIdx.x & 31) * (C / 32) + i;
      v[i] = t < n ? g[(t0 + t) * a.g_token] : 0.f;
    }
  }
  __device__ __forceinline__ void finish(Decays<C> &d) const {
    const int lane = threadIdx.x & 31;
    constexpr float log2e = 1.44269502162933349609f, log2e_low = 1.925963033500811e-8f;
    float2 b[C / 32], upto;
#pragma unroll
    for (int i = 0; i < C / 32; ++i) {
      const float x = v[i] * log2e;
      // (a NaN stays one)
      const float2 at = x < -kNothing ? make_float2(-kNothing, 0.f)
                                      : make_float2(x, fmaf(v[i], log2e_low, fmaf(v[i], log2e, -x)));
      b[i] = upto = i ? two_sum(upto, at) : at;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float2 x = make_float2(__shfl_up_sync(0xffffffffu, upto.x, o), __shfl_up_sync(0xffffffffu, upto.y, o));
      if (lane >= o) upto = two_sum(x, upto);
    }
    const float2 whole =
        make_float2(__shfl_sync(0xffffffffu, upto.x, 31), __shfl_sync(0xffffffffu, upto.y, 31));
    float2 before = make_float2(__shfl_up_sync(0xffffffffu, upto.x, 1), __shfl_up_sync(0xffffffffu, upto.y, 1));
    if (lane == 0) before = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < C / 32; ++i) {
      const int t = lane * (C / 32) + i;
      const float2 at = two_sum(before, b[i]);
      d.at[t] = at;
      d.begin[t] = exp2_pair(at);
      d.end[t] = exp2_pair(two_sum(whole, make_float2(-at.x, -at.y)));
    }
    if (lane == 0) {
      d.whole = exp2_pair(whole);
      d.sum = whole;
    }
  }
};

// The 16x16 blocks on and below the diagonal of a chunk's scores.
template <int C>
__device__ __forceinline__ void block_of(int i, int &row, int &col) {
  row = 0;
  while (i > row) i -= ++row;
  col = i;
}

__device__ __forceinline__ int tokens_of(const Args &a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length;
}

enum Mode { kOutput, kForwardState, kBackwardState };

// One slab of up to 64 values of one head: 16 of them a warp, with their
// transposed state in registers.  kOutput: the outputs of a segment of chunks
// (and the states before each, for the backward pass).  kForwardState: only
// the state that a segment adds.  kBackwardState: D, from the last chunk to
// the first, from queries and the outputs' gradients in the places of keys and
// values; with `dstates` those behind each chunk, else what a segment adds.
// The chain of dependent steps that a chunk takes is long, so what counts is
// the warps that an SM has to change between: the outputs go by 32 tokens at a
// time, their tiles have no second buffer, and registers are held to four blocks
// an SM (five for up to 64 keys).
template <typename T, int DK, Mode kMode>
__global__ void __launch_bounds__(128, sizeof(T) == 2 ? (DK == 64 ? 5 : 4) : 2) linattn_kernel(const Args a) {
  using Pl = Planes<T>;
  constexpr int C = Pl::chunk, N = Pl::in;
  constexpr bool kApart = N > 1;
  constexpr bool kOut = kMode == kOutput, kBack = kMode == kBackwardState;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Decays<C> decays[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, gc = lane & 3;
  int unit = blockIdx.x;
  const int slab = unit % a.slabs;
  unit /= a.slabs;
  const int seg = unit % a.segments;
  unit /= a.segments;
  const int h = unit % a.heads, b = unit / a.heads;
  const int share = h / (a.heads / a.groups);
  const int dk16 = (a.dk + 15) & ~15, rows = min(a.slab, a.dv - slab * a.slab), rows16 = (rows + 15) & ~15;
  const int len = tokens_of(a, b);
  const int64_t L = a.length;
  const T *q = (const T *)a.q + ((int64_t)b * a.groups + share) * a.dk * L;
  const T *k = kBack ? q : (const T *)a.k + ((int64_t)b * a.groups + share) * a.dk * L;
  const int64_t values = (((int64_t)b * a.heads + h) * a.dv + slab * a.slab) * L;
  const T *v = (const T *)(kBack ? a.grad : a.v) + values;
  const int64_t state_size = (int64_t)a.dk * a.dv, head = (int64_t)b * a.heads + h;
  const int first = seg * a.per_segment, last = min(first + a.per_segment, a.chunks);
  const int used = min(last, (len + C - 1) / C);  // chunks with tokens

  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  constexpr int kRow = 2 * C;
  const int kb = dk16 * kRow, vb = a.slab * kRow;
  // keys and values; behind them queries and scores, or (where the copies are asynchronous) the next chunk's
  constexpr bool kAhead = !kOut && N == 1;
  const int stage = N * (kb + vb);
  const Tile<kRow> tq(base + stage, kb);
  const Scores<C, Pl::out> scores(base + stage + N * kb);
  auto tile_k = [&](int s) { return Tile<kRow>(base + s * stage, kb); };
  auto tile_v = [&](int s) { return Tile<kRow>(base + s * stage + N * kb, vb); };
  auto bring = [&](int c, int s) {
    const int64_t t0 = (int64_t)c * C;
    const int n = min(C, (int)(len - t0));
    fill<T, C>(tile_k(s), k, a.dk, dk16, L, t0, n, a.vec);
    fill<T, C>(tile_v(s), v, rows, rows16, L, t0, n, a.vec);
  };
  auto bring_queries = [&](int c) {
    const int64_t t0 = (int64_t)c * C;
    fill<T, C>(tq, q, a.dk, dk16, L, t0, min(C, (int)(len - t0)), a.vec);
  };

  // S^T of this warp's 16 values: tile j holds keys 8j .. 8j+7
  float S[DK / 8][4];
  const int value0 = slab * a.slab + warp * 16;
  auto each_state = [&](auto &&f) {  // f(number in registers, key, value)
#pragma unroll
    for (int j = 0; j < DK / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 8 * j + 2 * gc + (i & 1), value = value0 + gr + (i >> 1) * 8;
        if (key < a.dk && warp * 16 + gr + (i >> 1) * 8 < rows) f(S[j][i], key, value);
      }
  };
#pragma unroll
  for (int j = 0; j < DK / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) S[j][i] = 0.f;
  // a whole row, or the second pass over its segments: from what comes in
  const bool alone = a.segments == 1;
  const bool whole_pass = kOut || (kBack && a.dstates);
  const float *start = alone ? (kBack ? a.last_grad : a.initial) : whole_pass ? a.starts : nullptr;
  if (start) {
    start += (alone ? head : head * a.segments + seg) * state_size;
    each_state([&](float &s, int key, int value) { s = start[(int64_t)key * a.dv + value]; });
  }

  // chunks in the order of the pass
  const int count = max(0, used - first);
  auto chunk_at = [&](int i) { return kBack ? first + count - 1 - i : first + i; };
  // The decays of as many chunks as there are warps are made at once, a warp each: one warp's chain of sums and
  // exponentials for every chunk is what the others would wait for.
  const int warps = blockDim.x >> 5;
  DecayLoad<C> ahead;
  auto load_decays = [&](int i) {
    if (i + warp < count) ahead.load(a, b, h, (int64_t)chunk_at(i + warp) * C, min(C, len - chunk_at(i + warp) * C));
  };
  float2 total = make_float2(0.f, 0.f);
  if (count) {
    bring(chunk_at(0), 0);
    if (kOut) bring_queries(chunk_at(0));
    load_decays(0);
  }
  for (int i = 0, turn = 0; i < count; ++i, turn = turn + 1 == warps ? 0 : turn + 1) {
    const int c = chunk_at(i);
    const int64_t t0 = (int64_t)c * C;
    const int n = min(C, (int)(len - t0));
    if (turn == 0) {
      if (i) __syncthreads();
      if (i + warp < count) ahead.finish(decays[warp]);
      load_decays(i + warps);
    }
    copies_done();
    __syncthreads();
    const Decays<C> &d = decays[turn];
    const int s = kAhead ? i & 1 : 0;
    const Tile<kRow> tk = tile_k(s), tv = tile_v(s);
    if (kAhead && i + 1 < count) bring(chunk_at(i + 1), s ^ 1);
    if (float *keep = kOut ? a.states : kBack ? a.dstates : nullptr)
      each_state([&](float &x, int key, int value) {
        keep[(head * a.chunks + c) * state_size + (int64_t)key * a.dv + value] = x;
      });
    if (kOut) {
      // the scores, a 16x16 block at a time
      for (int blk = warp; blk < (C / 16) * (C / 16 + 1) / 2; blk += blockDim.x >> 5) {
        int row, col;
        block_of<C>(blk, row, col);
        float x[2][4] = {}, xl[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          if (kk >= dk16) break;
          uint32_t A[N][4], B[N][4];
          load_a<true>(A, tq, row * 16, kk);
          load_b<true>(B, tk, kk, col * 16);
          product<kApart>(x[0], x[1], xl[0], xl[1], A, B);
        }
        if (kApart) join(x, xl);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int t = row * 16 + gr + (e >> 1) * 8, u = col * 16 + j * 8 + 2 * gc;
            const float x0 = u <= t ? x[j][e] * a.scale * exp2_fast(d.between(d.at[t], d.at[u])) : 0.f;
            const float x1 = u + 1 <= t ? x[j][e + 1] * a.scale * exp2_fast(d.between(d.at[t], d.at[u + 1])) : 0.f;
            uint32_t p[Pl::out];
            split<Pl::out>(x0, x1, p);
#pragma unroll
            for (int z = 0; z < Pl::out; ++z) {
              int br, bc;
              scores.place(row, col, z, br, bc);
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(scores.t.piece(br * 16 + gr + (e >> 1) * 8, bc * 2 + j,
                                                                          scores.kPacked ? 0 : z) + gc * 4),
                           "r"(p[z])
                           : "memory");
            }
          }
      }
      __syncthreads();
      if (warp * 16 < rows) {
#pragma unroll
        for (int part = 0; part < C / 32; ++part) {
          // what the state before the chunk gives 32 tokens
          float o[4][4] = {}, ol[4][4] = {};
#pragma unroll
          for (int kk = 0; kk < DK / 16; ++kk) {
            if (kk * 16 >= dk16) break;
            uint32_t A[Pl::out][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t p[Pl::out];
              split<Pl::out>(S[2 * kk + (e >> 1)][2 * (e & 1)], S[2 * kk + (e >> 1)][2 * (e & 1) + 1], p);
#pragma unroll
              for (int z = 0; z < Pl::out; ++z) A[z][e] = p[z];
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t B[N][4];
              load_b<true>(B, tq, kk * 16, part * 32 + j * 16);
              product<kApart>(o[2 * j], o[2 * j + 1], ol[2 * j], ol[2 * j + 1], A, B);
            }
          }
          if (kApart) join(o, ol);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] *= a.scale * d.begin[part * 32 + 8 * j + 2 * gc + (e & 1)];
          // and what the chunk's values give
#pragma unroll
          for (int ss = 0; ss < 2 * part + 2; ++ss) {
            uint32_t V[N][4];
            load_a<false>(V, tv, warp * 16, ss * 16);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int at = 2 * part + j;
              if (at < ss) continue;
              if (at == ss && any_not_finite(V[0])) {
                border<N, Pl::out, true>(o[2 * j], o[2 * j + 1], tv, warp * 16, scores, at * 16);
                continue;
              }
              uint32_t B[Pl::out][4];
              scores.load(B, ss, at);
              product<false>(o[2 * j], o[2 * j + 1], o[2 * j], o[2 * j + 1], V, B);
            }
          }
#pragma unroll
          for (int r8 = 0; r8 < 2; ++r8) {
            const int r = warp * 16 + gr + r8 * 8;
            if (r >= rows) continue;
            T *out = (T *)a.out + values + r * L + t0 + part * 32 + 2 * gc;
            if (a.vec && n == C) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                Pack<T, 2> p;
                p.set({o[j][2 * r8], o[j][2 * r8 + 1]});
                p.store(out + 8 * j);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (part * 32 + 8 * j + 2 * gc + e < n) out[8 * j + e] = from_f<T>(o[j][2 * r8 + e]);
            }
          }
        }
      }
    }
    if (kOut && i + 1 < count) {  // the queries are done with
      __syncthreads();
      bring_queries(chunk_at(i + 1));
    }
    // the state behind the chunk
    const float whole = d.whole;
    if (warp * 16 < rows) {
#pragma unroll
      for (int ss = 0; ss < C / 16; ++ss) {
        uint32_t V[N][4], W[Pl::update][4];
        load_a<false>(V, tv, warp * 16, ss * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = ss * 16 + (e >> 1) * 8 + 2 * gc;
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int z = N - 1; z >= 0; --z) {
            const float2 r = unpair(V[z][e]);
            x += r.x;
            y += r.y;
          }
          const float2 w = *reinterpret_cast<const float2 *>((kBack ? d.begin : d.end) + t);
          uint32_t p[Pl::update];
          split<Pl::update>(x * (kBack ? w.x * a.scale : w.x), y * (kBack ? w.y * a.scale : w.y), p);
#pragma unroll
          for (int z = 0; z < Pl::update; ++z) W[z][e] = p[z];
        }
#pragma unroll
        for (int j = 0; j < DK / 16; ++j) {
          if (j * 16 >= dk16) break;
          uint32_t B[N][4];
          load_b<false>(B, tk, ss * 16, j * 16);
          // (added in 32 bits, which rounds: a state is a sum over thousands of tokens)
          float u[2][4] = {};
          product<false>(u[0], u[1], u[0], u[1], W, B);
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              float *x = &S[2 * j + z][e];
              const float2 had = make_float2(x[0], x[1]), more = make_float2(u[z][e], u[z][e + 1]);
              const float2 now = ss == 0 ? __ffma2_rn(make_float2(whole, whole), had, more) : __fadd2_rn(had, more);
              x[0] = now.x;
              x[1] = now.y;
            }
        }
      }
    }
    total = two_sum(total, d.sum);
    if (!kAhead && i + 1 < count) {
      __syncthreads();
      bring(chunk_at(i + 1), 0);
    }
  }
  if (kOut) {  // zeros behind the last token
    const int64_t t0 = max((int64_t)first * C, (int64_t)len), behind = min((int64_t)last * C, L) - t0;
    if (behind > 0)
      for (int64_t i = threadIdx.x; i < behind * rows; i += blockDim.x)
        ((T *)a.out)[values + i / behind * L + t0 + i % behind] = from_f<T>(0.f);
  }
  if (!whole_pass) {
    each_state([&](float &s, int key, int value) {
      a.starts[(head * a.segments + seg) * state_size + (int64_t)key * a.dv + value] = s;
    });
    if (slab == 0 && threadIdx.x == 0) a.decays[head * a.segments + seg] = exp2_pair(total);
  } else if (alone && a.final_state) {
    each_state([&](float &s, int key, int value) { a.final_state[head * state_size + (int64_t)key * a.dv + value] = s; });
  }
}

// The states that the segments of each row start from, in place of what they
// add, and the one behind the last (backwards: before the first).
__global__ void __launch_bounds__(256) linattn_carry_kernel(const Args a, bool back) {
  const int64_t size = (int64_t)a.dk * a.dv, head = blockIdx.y + (int64_t)blockIdx.z * 65535;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size || head >= (int64_t)a.batch * a.heads) return;
  const float *from = back ? a.last_grad : a.initial;
  float s = from ? from[head * size + i] : 0.f;
  for (int j = 0; j < a.segments; j += 8) {  // eight reads in flight
    float added[8], decay[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (j + k < a.segments) {
        const int64_t seg = head * a.segments + (back ? a.segments - 1 - j - k : j + k);
        added[k] = a.starts[seg * size + i];
        decay[k] = a.decays[seg];
      }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (j + k < a.segments) {
        a.starts[(head * a.segments + (back ? a.segments - 1 - j - k : j + k)) * size + i] = s;
        s = fmaf(decay[k], s, added[k]);
      }
  }
  if (a.final_state) a.final_state[head * size + i] = s;
}

// ------------------------------------------------------------------ gradients

__device__ __forceinline__ float column_sum(float v) {  // over the eight rows of a fragment
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The gradients of one chunk of one head, from the states S before and D
// behind it.  With Z_ts = scale exp(b_t - b_s) for s <= t:
//   P = Z (q_t k_s),  E = Z (do_t v_s)
//   dq_t = sum_s E_ts k_s + scale exp(b_t) S do_t
//   dk_s = sum_t E_ts q_t + exp(b_C - b_s) D v_s
//   dv_s = sum_t P_ts do_t + exp(b_C - b_s) D^T k_s
// and the decays', dg_t, from the pairs W_us = P_us (do_u v_s), s < t <= u, the
// parts that S has in q dq from t on and D in k dk before t, and exp(b_C) <S, D>.
// The pairs of a 16x16 block on the diagonal are summed for each t: along its
// rows before t, then down its columns from t on.  Of the other blocks t has
// whole ones, rows from t on and columns before t.  So each sum has only what
// belongs to it: nothing is added and taken away again, and what is not finite
// stays on its side.
// A warp takes 16 of the dk or dv rows of a gradient and 32 tokens at a time.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) linattn_backward_kernel(const Args a) {
  using Pl = Planes<T>;
  constexpr int C = Pl::chunk, N = Pl::in, X = Pl::back, B16 = C / 16, kBlocks = B16 * (B16 + 1) / 2;
  constexpr bool kApart = N > 1;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Decays<C> d;
  __shared__ float row_sums[kBlocks][16], col_sums[kBlocks][16], all_sums[kBlocks], old_part[8][C], new_part[8][C], across_part[8];
  constexpr int warps = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, gc = lane & 3;
  int64_t unit = blockIdx.x;
  const int c = unit % a.chunks;
  const int64_t head = unit / a.chunks;
  const int h = head % a.heads, b = head / a.heads, share = h / (a.heads / a.groups);
  const int dk16 = (a.dk + 15) & ~15, dv16 = (a.dv + 15) & ~15, dv64 = (a.dv + 63) & ~63;
  const int64_t L = a.length, t0 = (int64_t)c * C;
  const int n = min(C, (int)(tokens_of(a, b) - t0)), kept = min(C, (int)(L - t0));
  const int64_t shared_at = ((int64_t)b * a.groups + share) * a.dk * L, values_at = head * a.dv * L;
  float *dg = a.dg + head * L + t0;
  // where the gradients of queries and keys go: the outputs, or a head's own in 32 bits
  auto put_shared = [&](T *out, float *heads, int row, int t, float x) {
    if (heads) heads[(head * a.dk + row) * L + t0 + t] = x;
    else out[shared_at + row * L + t0 + t] = from_f<T>(x);
  };
  if (n <= 0) {
    for (int i = threadIdx.x; i < kept * a.dk; i += blockDim.x) {
      put_shared((T *)a.dq, a.dq_heads, i / kept, i % kept, 0.f);
      put_shared((T *)a.dk_, a.dk_heads, i / kept, i % kept, 0.f);
    }
    for (int i = threadIdx.x; i < kept * a.dv; i += blockDim.x)
      ((T *)a.dv_)[values_at + i / kept * L + t0 + i % kept] = from_f<T>(0.f);
    for (int i = threadIdx.x; i < kept; i += blockDim.x) dg[i] = 0.f;
    return;
  }
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  constexpr int kRow = 2 * C;
  const int kb = dk16 * kRow, vb = dv16 * kRow;
  const Tile<kRow> tq(base, kb), tk(base + N * kb, kb), tv(base + 2 * N * kb, vb), to(base + 2 * N * kb + N * vb, vb);
  const uint32_t behind = base + 2 * N * (kb + vb);
  const Tile<kRow> tp(behind, C * kRow), te(behind + Pl::out * C * kRow, C * kRow);
  const Tile<0> ts(behind + 2 * Pl::out * C * kRow, dk16 * 2 * dv64, 2 * dv64);  // S, then D, [dk][dv]

  const int64_t state_size = (int64_t)a.dk * a.dv;
  const float *S = a.states + (head * a.chunks + c) * state_size, *D = a.dstates + (head * a.chunks + c) * state_size;
  // Brings a state into `ts`, four values of a key to a thread and eight of these in flight; also the sum of its
  // products with another one's values (or 0).
  const int quads = dv64 / 4;
  auto bring_state = [&](const float *from, const float *other) {
    float sum = 0.f;
    const bool wide = a.dv % 4 == 0;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < dk16 * quads; i0 += 256 * U) {
      float x[U][4] = {}, y[U][4] = {};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 256, row = i / quads, col = i % quads * 4;
        if (row < a.dk && col < a.dv) {
          const int64_t at = (int64_t)row * a.dv + col;
          if (wide) {
            *reinterpret_cast<float4 *>(x[u]) = *reinterpret_cast<const float4 *>(from + at);
            if (other) *reinterpret_cast<float4 *>(y[u]) = *reinterpret_cast<const float4 *>(other + at);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < a.dv) {
                x[u][e] = from[at + e];
                if (other) y[u][e] = other[at + e];
              }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 256, row = i / quads, col = i % quads * 4;
        if (row >= dk16) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fmaf(x[u][e], y[u][e], sum);
        uint32_t p[X], q[X];
        split<X>(x[u][0], x[u][1], p);
        split<X>(x[u][2], x[u][3], q);
#pragma unroll
        for (int z = 0; z < X; ++z)
          asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(ts.piece(row, col / 8, z) + (col & 7) * 2), "r"(p[z]), "r"(q[z])
                       : "memory");
      }
    }
    return sum;
  };
  fill<T, C>(tq, (const T *)a.q + shared_at, a.dk, dk16, L, t0, n, a.vec);
  fill<T, C>(tk, (const T *)a.k + shared_at, a.dk, dk16, L, t0, n, a.vec);
  fill<T, C>(tv, (const T *)a.v + values_at, a.dv, dv16, L, t0, n, a.vec);
  fill<T, C>(to, (const T *)a.grad + values_at, a.dv, dv16, L, t0, n, a.vec);
  {
    float x = bring_state(S, D);
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) across_part[warp] = x;
  }
  if (warp == 0) {
    DecayLoad<C> g;
    g.load(a, b, h, t0, n);
    g.finish(d);
  }
  copies_done();
  __syncthreads();

  for (int blk = warp; blk < kBlocks; blk += warps) {
    int row, col;
    block_of<C>(blk, row, col);
    float x[2][4] = {}, y[2][4] = {}, xl[2][4] = {}, yl[2][4] = {};
#pragma unroll 4
    for (int kk = 0; kk < dk16; kk += 16) {
      uint32_t A[N][4], B[N][4];
      load_a<true>(A, tq, row * 16, kk);
      load_b<true>(B, tk, kk, col * 16);
      product<kApart>(x[0], x[1], xl[0], xl[1], A, B);
    }
#pragma unroll 4
    for (int kk = 0; kk < dv16; kk += 16) {
      uint32_t A[N][4], B[N][4];
      load_a<true>(A, to, row * 16, kk);
      load_b<true>(B, tv, kk, col * 16);
      product<kApart>(y[0], y[1], yl[0], yl[1], A, B);
    }
    if (kApart) {
      join(x, xl);
      join(y, yl);
    }
    float w[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int t = row * 16 + gr + (e >> 1) * 8, u = col * 16 + j * 8 + 2 * gc;
        float p[2], q[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const float z = u + f <= t ? a.scale * exp2_fast(d.between(d.at[t], d.at[u + f])) : 0.f;
          p[f] = u + f <= t ? x[j][e + f] * z : 0.f;
          q[f] = u + f <= t ? y[j][e + f] * z : 0.f;
          w[j][e + f] = u + f < t ? p[f] * y[j][e + f] : 0.f;
        }
        uint32_t pp[Pl::out], pq[Pl::out];
        split<Pl::out>(p[0], p[1], pp);
        split<Pl::out>(q[0], q[1], pq);
#pragma unroll
        for (int z = 0; z < Pl::out; ++z) {
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(tp.piece(t, u / 8, z) + (u & 7) * 2), "r"(pp[z]) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(te.piece(t, u / 8, z) + (u & 7) * 2), "r"(pq[z]) : "memory");
        }
      }
    float cs[2][2];
    if (row == col) {
      // of each row u, the pairs before t = its columns 2 gc, 2 gc + 1 and 8 more, where t <= u
      cs[0][0] = cs[0][1] = cs[1][0] = cs[1][1] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float upto[2], left = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          upto[j] = w[j][2 * e] + w[j][2 * e + 1];
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            const float v = __shfl_up_sync(0xffffffffu, upto[j], o, 4);
            if (gc >= o) upto[j] += v;
          }
          float before = __shfl_up_sync(0xffffffffu, upto[j], 1, 4);
          before = gc == 0 ? left : left + before;
          left = __shfl_sync(0xffffffffu, upto[j], 3, 4);
          const int u = gr + e * 8, t = j * 8 + 2 * gc;
          cs[j][0] += t <= u ? before : 0.f;
          cs[j][1] += t + 1 <= u ? before + w[j][2 * e] : 0.f;
        }
      }
    } else {
      float rs[2], all;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        rs[e] = (w[0][2 * e] + w[0][2 * e + 1]) + (w[1][2 * e] + w[1][2 * e + 1]);
        rs[e] += __shfl_xor_sync(0xffffffffu, rs[e], 1);
        rs[e] += __shfl_xor_sync(0xffffffffu, rs[e], 2);
        if (gc == 0) row_sums[blk][gr + e * 8] = rs[e];
      }
      all = column_sum(rs[0] + rs[1]);
      if (lane == 0) all_sums[blk] = all;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int f = 0; f < 2; ++f) cs[j][f] = w[j][f] + w[j][2 + f];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        cs[j][f] = column_sum(cs[j][f]);
        if (gr == 0) col_sums[blk][j * 8 + 2 * gc + f] = cs[j][f];
      }
  }

  // A piece of a gradient: 16 of its rows (of keys or values) and 32 tokens.
  constexpr int kParts = C / 32;
  const int key_tiles = dk16 / 16, value_tiles = dv16 / 16;
  float acc[4][4];
  auto zero = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  };
  // acc += A[rows m ..][k] B[k][tokens], k over `depth`; A the state, transposed or not
  auto times = [&](auto trans, int m, const Tile<kRow> &B_, int depth, int part) {
    float low[4][4] = {};
#pragma unroll 2
    for (int kk = 0; kk < depth; kk += 16) {
      uint32_t A[X][4];
      load_a<decltype(trans)::value>(A, ts, m, kk);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t B[N][4];
        load_b<true>(B, B_, kk, part * 32 + j * 16);
        product<kApart>(acc[2 * j], acc[2 * j + 1], low[2 * j], low[2 * j + 1], A, B);
      }
    }
    if (kApart) join(acc, low);
  };
  auto factors = [&](const float *factor, float scale, int part) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] *= scale * factor[part * 32 + 8 * j + 2 * gc + (e & 1)];
  };
  // the sums of acc times x's rows, for each token
  auto share_of = [&](const Tile<kRow> &x, int m, int part, float *sums) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float s[2] = {};
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float f0 = 0.f, f1 = 0.f;
#pragma unroll
        for (int z = N - 1; z >= 0; --z) {
          uint32_t w;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(x.piece(m + gr + r * 8, part * 4 + j, z) + 4 * gc));
          const float2 v = unpair(w);
          f0 += v.x;
          f1 += v.y;
        }
        s[0] = fmaf(acc[j][2 * r], f0, s[0]);
        s[1] = fmaf(acc[j][2 * r + 1], f1, s[1]);
      }
      s[0] = column_sum(s[0]);
      s[1] = column_sum(s[1]);
      if (gr == 0) {
        sums[part * 32 + 8 * j + 2 * gc] = s[0];
        sums[part * 32 + 8 * j + 2 * gc + 1] = s[1];
      }
    }
  };
  // acc += x[rows m ..][tokens up to (or from) each one on] times the scores between them
  auto within = [&](auto up_to, const Tile<kRow> &x, int m, const Tile<kRow> &scores, int part) {
    constexpr bool kUpTo = decltype(up_to)::value;
#pragma unroll
    for (int s = 0; s < B16; ++s) {
      if (kUpTo ? s > 2 * part + 1 : s < 2 * part) continue;
      uint32_t A[N][4];
      load_a<false>(A, x, m, s * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = 2 * part + j;
        if (kUpTo ? s > at : s < at) continue;
        if (at == s && any_not_finite(A[0])) {
          border<N, Pl::out, kUpTo>(acc[2 * j], acc[2 * j + 1], x, m, scores, at * 16);
          continue;
        }
        uint32_t B[Pl::out][4];
        load_b<!kUpTo>(B, scores, s * 16, at * 16);
        product<false>(acc[2 * j], acc[2 * j + 1], acc[2 * j], acc[2 * j + 1], A, B);
      }
    }
  };
  const std::true_type yes;
  const std::false_type no;
  // Writes a piece to rows m .. of `out` (its row 0 at the chunk's first token).
  auto put = [&](auto *out, int m, int limit, int part) {
    using O = std::remove_pointer_t<decltype(out)>;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = m + gr + r * 8, t = part * 32 + 2 * gc;
      if (row >= limit) continue;
      O *at = out + row * L + t;
      if (a.vec && n == C) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Pack<O, 2> p;
          p.set({acc[j][2 * r], acc[j][2 * r + 1]});
          p.store(at + 8 * j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int u = t + 8 * j + e;
            if (u < kept) at[8 * j + e] = from_f<O>(u < n ? acc[j][2 * r + e] : 0.f);
          }
      }
    }
  };
  auto put_keys = [&](void *out, float *heads, int m, int part) {
    if (heads) put(heads + head * a.dk * L + t0, m, a.dk, part);
    else put((T *)out + shared_at + t0, m, a.dk, part);
  };
  // (the first pieces' states are multiplied before the barrier, while other warps still make scores)
  for (int it = warp; it < key_tiles * kParts; it += warps) {
    const int m = it / kParts * 16, part = it % kParts;
    zero();
    times(no, m, to, dv16, part);
    factors(d.begin, a.scale, part);
    share_of(tq, m, part, old_part[m / 16]);
    if (it == warp) __syncthreads();  // the scores are there
    within(yes, tk, m, te, part);
    put_keys(a.dq, a.dq_heads, m, part);
  }
  if (warp >= key_tiles * kParts) __syncthreads();
  __syncthreads();  // S is done with
  bring_state(D, nullptr);
  __syncthreads();
  for (int it = warp; it < (key_tiles + value_tiles) * kParts; it += warps) {
    const int tile = it / kParts, part = it % kParts;
    zero();
    if (tile < key_tiles) {
      const int m = tile * 16;
      times(no, m, tv, dv16, part);
      factors(d.end, 1.f, part);
      share_of(tk, m, part, new_part[tile]);
      within(no, tq, m, te, part);
      put_keys(a.dk_, a.dk_heads, m, part);
    } else {
      const int m = (tile - key_tiles) * 16;
      times(yes, m, tk, dk16, part);
      factors(d.end, 1.f, part);
      within(no, to, m, tp, part);
      put((T *)a.dv_ + values_at + t0, m, a.dv, part);
    }
  }
  __syncthreads();
  if (warp == 0) {
    // dg_t = sum_(u >= t) old_u + sum_(s < t) new_s + across + the pairs' share: the diagonal block's, whole blocks,
    // and in t's block of 16 tokens the sums of rows from t on and of columns before t
    constexpr int M = C / 32, W = 16 / M;  // tokens of a lane, lanes of a block
    const int tb = lane / W;
    float old[M], fresh[M], rows[M], cols[M], pairs[M], old_sum = 0.f, fresh_sum = 0.f, row_sum = 0.f, col_sum = 0.f;
    float whole = 0.f;
#pragma unroll
    for (int o = 0; o < B16; ++o)
#pragma unroll
      for (int u = o + 2; u < B16; ++u)
        if (o < tb && tb < u) whole += all_sums[u * (u + 1) / 2 + o];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int t = lane * M + i;
      float x = 0.f, y = 0.f;
      pairs[i] = col_sums[tb * (tb + 1) / 2 + tb][t % 16] + whole;
#pragma unroll
      for (int o = 0; o < B16; ++o) {
        if (o < tb) x += row_sums[tb * (tb + 1) / 2 + o][t % 16];
        if (o > tb) y += col_sums[o * (o + 1) / 2 + tb][t % 16];
      }
      rows[i] = x;
      cols[i] = y;
      row_sum += x;
      col_sum += y;
      x = y = 0.f;
      for (int w = 0; w < key_tiles; ++w) {
        x += old_part[w][t];
        y += new_part[w][t];
      }
      old[i] = x;
      fresh[i] = y;
      old_sum += x;
      fresh_sum += y;
    }
    // sums over the lanes behind this one and before it, of all or of its block
    auto behind = [&](float v, int width) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        if (o >= width) break;
        const float x = __shfl_down_sync(0xffffffffu, v, o, width);
        if (lane % width + o < width) v += x;
      }
      v = __shfl_down_sync(0xffffffffu, v, 1, width);
      return lane % width == width - 1 ? 0.f : v;
    };
    auto before = [&](float v, int width) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        if (o >= width) break;
        const float x = __shfl_up_sync(0xffffffffu, v, o, width);
        if (lane % width >= o) v += x;
      }
      v = __shfl_up_sync(0xffffffffu, v, 1, width);
      return lane % width == 0 ? 0.f : v;
    };
    float sum = behind(old_sum, 32) + before(fresh_sum, 32) + behind(row_sum, W) + before(col_sum, W);
    float across = 0.f;
    for (int w = 0; w < warps; ++w) across += across_part[w];
    sum += across * d.whole;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int t = lane * M + i;
      float x = sum + pairs[i];
#pragma unroll
      for (int j = 0; j < M; ++j) x += j < i ? fresh[j] + cols[j] : old[j] + rows[j];
      if (t < kept) dg[t] = t < n ? x : 0.f;
    }
  }
}

// Gradients of queries or keys that heads share: the sum over a group's heads.
template <typename T>
__global__ void __launch_bounds__(256) linattn_group_kernel(const float *heads, int64_t size, int per, int64_t count,
                                                            T *out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t group = i / size, at = i % size;
    float s = 0.f;
    for (int j = 0; j < per; ++j) s += heads[(group * per + j) * size + at];
    out[i] = from_f<T>(s);
  }
}

// The gradient of one decay for each head: the sum over rows and tokens.
__global__ void __launch_bounds__(256) linattn_decay_kernel(const float *dg, int batch, int heads, int64_t length,
                                                            float *out) {
  __shared__ double part[256];
  double s = 0.0;
  for (int b = 0; b < batch; ++b)
    for (int64_t t = threadIdx.x; t < length; t += 256) s += dg[((int64_t)b * heads + blockIdx.x) * length + t];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] = (float)part[0];
}

// -------------------------------------------------------------- single tokens

// One token of a row and head: the state is read and written once, V values of
// a key to a thread, the keys over the threads that are left.  Memory bounds it:
// 64 rows of 32 heads of 128x128 (268 MB) take 51 us, 5.2 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256) linattn_step_kernel(const T *q, const T *k, const T *v, const float *g,
                                                           int64_t g_batch, int64_t g_head, float *state,
                                                           const int *slots, int places, int heads, int groups, int dk,
                                                           int dv, float scale, T *out) {
  __shared__ float qs[kMaxDim], ks[kMaxDim], sums[256 * V];
  const int h = blockIdx.x % heads, b = blockIdx.x / heads, share = h / (heads / groups);
  StepKind kind;
  const int place = step_place(slots, b, places, &kind);
  const int twice = step_twice(slots, b, place, kind);
  const int cols = (dv + V - 1) / V, rows = 256 / cols, tx = threadIdx.x % cols, ty = threadIdx.x / cols;
  const int64_t at = ((int64_t)b * groups + share) * dk;
  for (int i = threadIdx.x; i < dk; i += 256) {
    qs[i] = to_f(q[at + i]) * scale;
    ks[i] = to_f(k[at + i]);
  }
  const float decay = expf(g[b * g_batch + h * g_head]);
  const int64_t values = ((int64_t)b * heads + h) * dv;
  const bool mine = ty < rows;
  float x[V] = {}, o[V] = {};
  if (mine) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f(v[values + tx * V + i]);
  }
  kind = step_served(twice, kind);  // (a barrier: the queries and keys are there)
  float *s = state + ((int64_t)place * heads + h) * dk * dv + tx * V;
  if (mine && kind == kStepServed) {
    constexpr int U = 8;
    for (int r0 = ty; r0 < dk; r0 += U * rows) {
      Pack<float, V> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 + u * rows < dk) {
          if constexpr (V == 4) *reinterpret_cast<float4 *>(p[u].v) = *reinterpret_cast<const float4 *>(s + (int64_t)(r0 + u * rows) * dv);
          else p[u].v[0] = s[(int64_t)(r0 + u * rows) * dv];
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * rows;
        if (r < dk) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            p[u].v[i] = fmaf(decay, p[u].v[i], ks[r] * x[i]);
            o[i] = fmaf(qs[r], p[u].v[i], o[i]);
          }
          p[u].store(s + (int64_t)r * dv);
        }
      }
    }
  }
  if (mine) {
#pragma unroll
    for (int i = 0; i < V; ++i) sums[(ty * cols + tx) * V + i] = o[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < dv; i += 256) {
    float y = step_nothing(kind);
    if (kind == kStepServed)
      for (int r = 0; r < rows; ++r) y += sums[r * cols * V + i];
    out[values + i] = from_f<T>(y);
  }
}

// ----------------------------------------------------------------------- host

struct Plan {
  int slabs, slab, segments, per_segment, chunks;
  size_t starts, decays;  // bytes, where there are segments
};

int chunk_of(int dtype) {
  return dtype == PC2D_DTYPE_F32   ? Planes<float>::chunk
         : dtype == PC2D_DTYPE_F16 ? Planes<__half>::chunk
                                   : Planes<__nv_bfloat16>::chunk;
}

// Slabs of up to 64 values, of equal numbers of 16; and, where heads and slabs
// leave the GPU without work, the sequence in segments (each at least 4 chunks).
Plan make_plan(int dtype, int batch, int heads, int length, int dk, int dv) {
  Plan p{};
  const int tiles = (dv + 15) / 16;
  p.slabs = (tiles + 3) / 4;
  p.slab = 16 * ((tiles + p.slabs - 1) / p.slabs);
  p.chunks = ceil_div(length, chunk_of(dtype));
  const int64_t units = (int64_t)batch * heads * p.slabs;
  auto segments = [&](int blocks) {  // for so many blocks an SM
    const int64_t wanted = (int64_t)device_sm_count() * blocks;
    return units * 2 <= wanted && p.chunks >= 8 ? (int)std::min<int64_t>(wanted / units, p.chunks / 4) : 1;
  };
  p.segments = segments(4);
  // Five fit with up to 64 keys: taken where their segments are shorter by as much as they share the SM more (70 heads
  // of 48x80 at 777 tokens in float16: 5 segments of 5 chunks 96 us, 4 of up to 7 112; 128 heads of 64 at 2048 tokens in
  // bfloat16, where they would be 5 of up to 7 chunks for 4 of 8: 154 us for 146, a training step 508 for 493; from a
  // cold cache, in turn).
  if (dk <= 64 && ceil_div(p.chunks, segments(5)) * 5 <= ceil_div(p.chunks, p.segments) * 4) p.segments = segments(5);
  p.per_segment = ceil_div(p.chunks, p.segments);
  p.segments = std::max(1, ceil_div(p.chunks, std::max(1, p.per_segment)));
  return p;
}
void sizes_of(Plan &p, int batch, int heads, int dk, int dv) {
  if (p.segments > 1) {
    p.starts = align_up((size_t)batch * heads * p.segments * dk * dv * 4, 256);
    p.decays = align_up((size_t)batch * heads * p.segments * 4, 256);
  }
}

template <typename T>
size_t forward_smem(const Args &a, bool out) {
  using Pl = Planes<T>;
  const int dk16 = (a.dk + 15) & ~15, bytes = 2 * Pl::chunk;
  const size_t stage = (size_t)Pl::in * (dk16 + a.slab) * bytes;
  return out ? stage + (size_t)Pl::in * dk16 * bytes + Scores<Pl::chunk, Pl::out>::kBytes : Pl::in == 1 ? 2 * stage : stage;
}
template <typename T>
size_t backward_smem(const Args &a) {
  using Pl = Planes<T>;
  const int dk16 = (a.dk + 15) & ~15, dv16 = (a.dv + 15) & ~15, dv64 = (a.dv + 63) & ~63, bytes = 2 * Pl::chunk;
  return (size_t)2 * Pl::in * (dk16 + dv16) * bytes + (size_t)2 * Pl::out * Pl::chunk * bytes +
         (size_t)Pl::back * dk16 * 2 * dv64;
}

template <typename K>
int allow_smem(K *kernel, PerContext<uint64_t> &allowed) {
  return once_per_context(allowed, 1, [&]() -> int {
    PC2D_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 8 * 1024));
    return PC2D_OK;
  });
}

template <typename T, int DK, Mode kMode>
int launch_pass(const Args &a, cudaStream_t stream) {
  auto *kernel = linattn_kernel<T, DK, kMode>;
  static PerContext<uint64_t> allowed;
  const int st = allow_smem(kernel, allowed);
  if (st != PC2D_OK) return st;
  const int64_t grid = (int64_t)a.batch * a.heads * a.slabs * a.segments;
  kernel<<<(unsigned)grid, a.slab * 2, forward_smem<T>(a, kMode == kOutput), stream>>>(a);
  PC2D_LAUNCH_CHECK("linattn_kernel");
  return PC2D_OK;
}

template <typename T, Mode kMode>
int launch_passes(const Args &a, cudaStream_t stream) {
  return a.dk <= 64 ? launch_pass<T, 64, kMode>(a, stream) : launch_pass<T, 128, kMode>(a, stream);
}

int launch_carry(const Args &a, bool back, cudaStream_t stream) {
  const int64_t heads = (int64_t)a.batch * a.heads;
  const dim3 grid((unsigned)ceil_div((int64_t)a.dk * a.dv, 256), (unsigned)std::min<int64_t>(heads, 65535),
                  (unsigned)ceil_div(heads, 65535));
  linattn_carry_kernel<<<grid, 256, 0, stream>>>(a, back);
  PC2D_LAUNCH_CHECK("linattn_carry_kernel");
  return PC2D_OK;
}

template <typename T>
int run_forward(const Args &a, cudaStream_t stream) {
  int st;
  if (a.segments > 1 && ((st = launch_passes<T, kForwardState>(a, stream)) != PC2D_OK ||
                         (st = launch_carry(a, false, stream)) != PC2D_OK))
    return st;
  // (of several segments the final state comes from the first pass)
  return launch_passes<T, kOutput>(a, stream);
}

template <typename T>
int run_backward(Args a, void *dq, void *dk, cudaStream_t stream) {
  int st;
  if (a.segments > 1) {
    Args first = a;
    first.dstates = nullptr;
    if ((st = launch_passes<T, kBackwardState>(first, stream)) != PC2D_OK || (st = launch_carry(a, true, stream)) != PC2D_OK)
      return st;
  }
  if ((st = launch_passes<T, kBackwardState>(a, stream)) != PC2D_OK) return st;
  auto *kernel = linattn_backward_kernel<T>;
  static PerContext<uint64_t> allowed;
  if ((st = allow_smem(kernel, allowed)) != PC2D_OK) return st;
  kernel<<<(unsigned)((int64_t)a.batch * a.heads * a.chunks), 256, backward_smem<T>(a),
           stream>>>(a);
  PC2D_LAUNCH_CHECK("linattn_backward_kernel");
  if (a.dq_heads) {
    const int64_t size = (int64_t)a.dk * a.length, count = size * a.batch * a.groups;
    const unsigned grid = (unsigned)std::min<int64_t>((count + 255) / 256, (int64_t)device_sm_count() * 8);
    linattn_group_kernel<T><<<grid, 256, 0, stream>>>(a.dq_heads, size, a.heads / a.groups, count, (T *)dq);
    linattn_group_kernel<T><<<grid, 256, 0, stream>>>(a.dk_heads, size, a.heads / a.groups, count, (T *)dk);
    PC2D_LAUNCH_CHECK("linattn_group_kernel");
  }
  return PC2D_OK;
}

int check_linattn(const char *what, int dtype, int batch, int heads, int groups, int length, int dk, int dv) {
  if (!seq_dtype(dtype)) {
    set_last_error("%s: unsupported dtype %d", what, dtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (batch < 0 || heads < 1 || groups < 1 || heads % groups || length < 0 || dk < 1 || dv < 1) {
    set_last_error("%s: invalid sizes (batch %d, heads %d, groups %d, length %d, dk %d, dv %d)", what, batch, heads,
                   groups, length, dk, dv);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (dk > kMaxDim || dv > kMaxDim || length > 1 << 30 || (int64_t)batch * heads > 1 << 20 ||
      (int64_t)batch * heads * ceil_div(length, chunk_of(dtype)) > 0x7fffffff) {
    set_last_error("%s: at most %d numbers a query, key or value, 2^30 tokens and 2^20 heads of rows", what, kMaxDim);
    return PC2D_ERR_UNSUPPORTED;
  }
  return PC2D_OK;
}

int check_states(const char *what, const float *states) {
  if (aligned16(states)) return PC2D_OK;
  set_last_error("%s: the kept states must be on a 16-byte boundary", what);
  return PC2D_ERR_INVALID_ARGUMENT;
}

int need_workspace(const char *what, const void *workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need || !aligned16(workspace))) {
    set_last_error("%s: workspace of %zu bytes on a 16-byte boundary needed", what, need);
    return PC2D_ERR_WORKSPACE;
  }
  return PC2D_OK;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" size_t pc2d_linear_attention_states_size(int dtype, int batch, int heads, int length, int dk, int dv) {
  if (check_linattn("pc2d_linear_attention_states_size", dtype, batch, heads, 1, length, dk, dv) != PC2D_OK) return 0;
  return (size_t)batch * heads * ceil_div(length, chunk_of(dtype)) * dk * dv * 4;
}

extern "C" size_t pc2d_linear_attention_workspace_size(int dtype, int batch, int heads, int groups, int length, int dk,
                                                       int dv, int backward) {
  if (check_linattn("pc2d_linear_attention_workspace_size", dtype, batch, heads, groups, length, dk, dv) != PC2D_OK)
    return 0;
  Plan p = make_plan(dtype, batch, heads, length, dk, dv);
  sizes_of(p, batch, heads, dk, dv);
  size_t bytes = p.starts + p.decays;
  if (backward) {
    bytes += align_up(pc2d_linear_attention_states_size(dtype, batch, heads, length, dk, dv), 256);
    bytes += align_up((size_t)batch * heads * length * 4, 256);
    if (groups != heads) bytes += 2 * align_up((size_t)batch * heads * dk * length * 4, 256);
  }
  return bytes;
}

extern "C" int pc2d_linear_attention_forward(int dtype, const void *q, const void *k, const void *v,
                                             const float *log_decay, int decay_per_token, const float *initial_state,
                                             const int *lengths, int batch, int heads, int groups, int length, int dk,
                                             int dv, double scale, void *output, float *final_state, float *states,
                                             void *workspace, size_t workspace_bytes, void *stream) {
  NvtxRange range("pc2d_linear_attention_forward");
  const char *what = "pc2d_linear_attention_forward";
  int st = check_linattn(what, dtype, batch, heads, groups, length, dk, dv);
  if (st != PC2D_OK) return st;
  if (!isfinite(scale)) {
    set_last_error("%s: scale must be finite", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (!batch) return PC2D_OK;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const size_t size = seq_dtype_size(dtype);
  if ((st = check_elements(what, 4, {log_decay, initial_state, lengths, final_state, states})) != PC2D_OK ||
      (st = pending_device_error()) != PC2D_OK)
    return st;
  if (!length) {
    if (final_state) {
      const size_t bytes = (size_t)batch * heads * dk * dv * 4;
      if (initial_state)
        PC2D_CUDA_CHECK(cudaMemcpyAsync(final_state, initial_state, bytes, cudaMemcpyDeviceToDevice, s));
      else
        PC2D_CUDA_CHECK(cudaMemsetAsync(final_state, 0, bytes, s));
    }
    return PC2D_OK;
  }
  if (!q || !k || !v || !log_decay || !output) {
    set_last_error("%s: null pointer (q, k, v, log_decay or output)", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_elements(what, size, {q, k, v, output})) != PC2D_OK || (st = check_states(what, states)) != PC2D_OK)
    return st;
  Plan p = make_plan(dtype, batch, heads, length, dk, dv);
  sizes_of(p, batch, heads, dk, dv);
  if ((st = need_workspace(what, workspace, workspace_bytes, p.starts + p.decays)) != PC2D_OK) return st;
  Args a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.g = log_decay;
  a.g_batch = decay_per_token ? (int64_t)heads * length : 0;
  a.g_head = decay_per_token ? length : 1;
  a.g_token = decay_per_token ? 1 : 0;
  a.initial = initial_state;
  a.lengths = lengths;
  a.out = output;
  a.final_state = final_state;
  a.states = states;
  a.starts = static_cast<float *>(workspace);
  a.decays = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.starts);
  a.batch = batch;
  a.heads = heads;
  a.groups = groups;
  a.length = length;
  a.dk = dk;
  a.dv = dv;
  a.chunks = p.chunks;
  a.slabs = p.slabs;
  a.slab = p.slab;
  a.segments = p.segments;
  a.per_segment = p.per_segment;
  a.scale = (float)scale;
  a.vec = length % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(output);
  switch (dtype) {
    case PC2D_DTYPE_F32: return run_forward<float>(a, s);
    case PC2D_DTYPE_F16: return run_forward<__half>(a, s);
    default: return run_forward<__nv_bfloat16>(a, s);
  }
}

extern "C" int pc2d_linear_attention_backward(int dtype, const void *grad, const float *grad_final, const void *q,
                                              const void *k, const void *v, const float *log_decay, int decay_per_token,
                                              const float *states, const int *lengths, int batch, int heads, int groups,
                                              int length, int dk, int dv, double scale, void *qgrad, void *kgrad,
                                              void *vgrad, float *decaygrad, float *initialgrad, void *workspace,
                                              size_t workspace_bytes, void *stream) {
  NvtxRange range("pc2d_linear_attention_backward");
  const char *what = "pc2d_linear_attention_backward";
  int st = check_linattn(what, dtype, batch, heads, groups, length, dk, dv);
  if (st != PC2D_OK) return st;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const size_t size = seq_dtype_size(dtype);
  if ((st = check_elements(what, 4, {log_decay, grad_final, lengths, states, decaygrad, initialgrad})) != PC2D_OK ||
      (st = pending_device_error()) != PC2D_OK)
    return st;
  if (!batch || !length) {
    if (decaygrad && !decay_per_token) PC2D_CUDA_CHECK(cudaMemsetAsync(decaygrad, 0, heads * sizeof(float), s));
    if (initialgrad && batch) {
      const size_t bytes = (size_t)batch * heads * dk * dv * 4;
      if (grad_final) PC2D_CUDA_CHECK(cudaMemcpyAsync(initialgrad, grad_final, bytes, cudaMemcpyDeviceToDevice, s));
      else PC2D_CUDA_CHECK(cudaMemsetAsync(initialgrad, 0, bytes, s));
    }
    return PC2D_OK;
  }
  if (!grad || !q || !k || !v || !log_decay || !states || !qgrad || !kgrad || !vgrad || !decaygrad) {
    set_last_error("%s: null pointer", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_elements(what, size, {grad, q, k, v, qgrad, kgrad, vgrad})) != PC2D_OK ||
      (st = check_states(what, states)) != PC2D_OK)
    return st;
  if ((st = need_workspace(what, workspace, workspace_bytes,
                           pc2d_linear_attention_workspace_size(dtype, batch, heads, groups, length, dk, dv, 1))) != PC2D_OK)
    return st;
  Plan p = make_plan(dtype, batch, heads, length, dk, dv);
  sizes_of(p, batch, heads, dk, dv);
  char *at = static_cast<char *>(workspace);
  auto take = [&](size_t bytes) {
    char *r = at;
    at += align_up(bytes, 256);
    return r;
  };
  Args a{};
  a.starts = reinterpret_cast<float *>(take(p.starts));
  a.decays = reinterpret_cast<float *>(take(p.decays));
  a.dstates =
      reinterpret_cast<float *>(take(pc2d_linear_attention_states_size(dtype, batch, heads, length, dk, dv)));
  float *per_token = reinterpret_cast<float *>(take((size_t)batch * heads * length * 4));
  if (groups != heads) {
    a.dq_heads = reinterpret_cast<float *>(take((size_t)batch * heads * dk * length * 4));
    a.dk_heads = reinterpret_cast<float *>(take((size_t)batch * heads * dk * length * 4));
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.grad = grad;
  a.g = log_decay;
  a.g_batch = decay_per_token ? (int64_t)heads * length : 0;
  a.g_head = decay_per_token ? length : 1;
  a.g_token = decay_per_token ? 1 : 0;
  a.last_grad = grad_final;
  a.lengths = lengths;
  a.final_state = initialgrad;
  a.states = const_cast<float *>(states);
  a.dq = qgrad;
  a.dk_ = kgrad;
  a.dv_ = vgrad;
  a.dg = decay_per_token ? decaygrad : per_token;
  a.batch = batch;
  a.heads = heads;
  a.groups = groups;
  a.length = length;
  a.dk = dk;
  a.dv = dv;
  a.chunks = p.chunks;
  a.slabs = p.slabs;
  a.slab = p.slab;
  a.segments = p.segments;
  a.per_segment = p.per_segment;
  a.scale = (float)scale;
  a.vec = length % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(grad) && aligned16(qgrad) &&
          aligned16(kgrad) && aligned16(vgrad);
  switch (dtype) {
    case PC2D_DTYPE_F32: st = run_backward<float>(a, qgrad, kgrad, s); break;
    case PC2D_DTYPE_F16: st = run_backward<__half>(a, qgrad, kgrad, s); break;
    default: st = run_backward<__nv_bfloat16>(a, qgrad, kgrad, s);
  }
  if (st != PC2D_OK || decay_per_token) return st;
  linattn_decay_kernel<<<heads, 256, 0, s>>>(per_token, batch, heads, length, decaygrad);
  PC2D_LAUNCH_CHECK("linattn_decay_kernel");
  return PC2D_OK;
}

extern "C" int pc2d_linear_attention_step(int dtype, const void *q, const void *k, const void *v, const float *log_decay,
                                          int decay_per_row, float *state, const int *slots, int batch, int places,
                                          int heads, int groups, int dk, int dv, double scale, void *output,
                                          void *stream) {
  NvtxRange range("pc2d_linear_attention_step");
  const char *what = "pc2d_linear_attention_step";
  int st = check_linattn(what, dtype, batch, heads, groups, 1, dk, dv);
  if (st != PC2D_OK) return st;
  if (!isfinite(scale) || places < 0 || (!slots && batch > places)) {
    set_last_error("%s: scale must be finite, and every row needs a place (batch %d, places %d)", what, batch, places);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (!batch) return PC2D_OK;
  if (!q || !k || !v || !log_decay || !output || (places && !state)) {
    set_last_error("%s: null pointer (q, k, v, log_decay, state or output)", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  const size_t size = seq_dtype_size(dtype);
  if ((st = check_elements(what, size, {q, k, v, output})) != PC2D_OK ||
      (st = check_elements(what, 4, {log_decay, slots})) != PC2D_OK)
    return st;
  if (!aligned16(state)) {
    set_last_error("%s: the state must be on a 16-byte boundary", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = pending_device_error()) != PC2D_OK) return st;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto type, auto width) -> int {
    using T = decltype(type);
    constexpr int V = decltype(width)::value;
    linattn_step_kernel<T, V><<<(unsigned)((int64_t)batch * heads), 256, 0, s>>>(
        (const T *)q, (const T *)k, (const T *)v, log_decay, decay_per_row ? heads : 0, 1, state, slots, places, heads,
        groups, dk, dv, (float)scale, (T *)output);
    PC2D_LAUNCH_CHECK("linattn_step_kernel");
    return PC2D_OK;
  };
  auto typed = [&](auto type) -> int {
    return dv % 4 == 0 ? run(type, std::integral_constant<int, 4>()) : run(type, std::integral_constant<int, 1>());
  };
  switch (dtype) {
    case PC2D_DTYPE_F32: return typed(float());
    case PC2D_DTYPE_F16: return typed(__half());
    default: return typed(__nv_bfloat16());
  }
}
