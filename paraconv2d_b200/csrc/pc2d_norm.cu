// Group norm with an optional SiLU, over maps in either order of dimensions:
// [batch][channels][length] ("rows" are channels of tokens) or channels last,
// [batch][length][channels] ("rows" are tokens of channels).
//
//   xhat = (x - mean) rstd over the tokens and channels of a (batch row, group)
//   pre = xhat w_c + b_c,  y = pre or pre sigmoid(pre)
//   h = dy (1 or the SiLU's slope at pre)
//   dw_c = sum h xhat,  db_c = sum h
//   dx = rstd (h w_c - mean(h w) - xhat mean(h w xhat))
//
// A slab, all that shares statistics (and, channels last, the neighbouring
// groups that fill a few sectors of a token), is one cluster of 1 to 8 thread
// blocks' work: they read it, exchange their partial sums through distributed
// shared memory, and read it again, from the L2 cache, which holds the slabs of
// all clusters at work.  Where there are too few slabs for the GPU, two launches
// share the same code and exchange the partial sums in device memory instead.
//
// Variance: each thread sums x - K and its square, K its own first value (of
// the channel, channels last), and the (count, mean, M2) of threads, warps and
// blocks are joined by M2 = sum M2_i + n_i (mean_i - mean)^2.  Neither a large
// mean nor a single outlier cancels: a thread's sums are off by 2^-24 of
// squares that the slab's M2 holds too, once per element of the thread.
// All joins go by fixed orders.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "pc2d_seq.cuh"
#include "pc2d_tc.cuh"

namespace cg = cooperative_groups;

namespace pc2d {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxSplit = 64;         // blocks of a slab that exchange through device memory
constexpr int kMaxChannels = 8192;    // of a slab: its sums are in shared memory

enum Phase { kFused, kSums, kApply };

struct NormArgs {
  const void *x, *dy, *w, *b;
  const int *lengths;
  void *out;            // y, or dx
  float *stats;         // [batch][groups][2]: mean and rstd
  float *part;          // kSums, kApply: [slab][split][numbers of a block]
  float *chan;          // backward: [batch][channels][2], sums of h and of h xhat
  int batch, C, P, G, cg;
  int slab_channels;    // channels of a slab: cg, or a multiple of it
  int slabs;            // slabs of a batch row
  int split;            // blocks of a slab
  int seg, segs;        // channels first: vectors and number of the pieces of a row
  int wf32;             // weight and bias in float32, else in x's type
  int silu;
  Phase phase;
  float eps;
};

template <typename T>
__device__ __forceinline__ float load_w(const void *p, int i, bool f32, float none) {
  if (!p) return none;
  return f32 ? static_cast<const float *>(p)[i] : to_f(static_cast<const T *>(p)[i]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Place {
  int rank, n, slab, len;  // block of its slab; batch row; slab of the row; tokens of the row
};
__device__ __forceinline__ Place place_of(const NormArgs &a) {
  Place p;
  p.rank = blockIdx.x % a.split;
  const int unit = blockIdx.x / a.split;
  p.n = unit / a.slabs;
  p.slab = unit % a.slabs;
  p.len = a.lengths ? min(max(a.lengths[p.n], 0), a.P) : a.P;
  return p;
}

// Calls take(numbers) with a function that gives number i of block r of this
// slab, once the `count` numbers that every block has in `mine` are known to
// all of its blocks.  False: this block is done.
template <typename Take>
__device__ __forceinline__ bool exchange(const NormArgs &a, const float *mine, int count, Take &&take) {
  const int rank = blockIdx.x % a.split;
  float *global = a.part + (size_t)(blockIdx.x / a.split) * a.split * count;
  __syncthreads();
  if (a.phase == kSums) {
    for (int i = threadIdx.x; i < count; i += kThreads) global[(size_t)rank * count + i] = mine[i];
    return false;
  }
  if (a.phase == kApply) {
    take([&](int r, int i) { return global[(size_t)r * count + i]; });
  } else if (a.split == 1) {
    take([&](int, int i) { return mine[i]; });
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    take([&](int r, int i) { return cluster.map_shared_rank(mine, r)[i]; });
    cluster.sync();  // nobody leaves while its numbers are read
  }
  __syncthreads();
  return true;
}

// (count, mean, M2) of `entries` entries by one warp, the mean and the M2 of
// entry i at v[at(i)] and v[at(i) + 1] and its count n(i).
template <typename At, typename Count>
__device__ __forceinline__ void join(const float *v, int entries, At &&at, Count &&n, float &total, float &mean,
                                     float &m2) {
  const int lane = threadIdx.x & 31;
  float c = 0.f, s = 0.f, q = 0.f;
  for (int i = lane; i < entries; i += 32) {
    c += n(i);
    s += n(i) * v[at(i)];
  }
  total = warp_sum(c);
  mean = total > 0.f ? warp_sum(s) / total : 0.f;
  for (int i = lane; i < entries; i += 32) {
    const float d = v[at(i)] - mean;
    q += n(i) > 0.f ? v[at(i) + 1] + n(i) * d * d : 0.f;
  }
  m2 = warp_sum(q);
}

// Pairs of numbers, one instruction for two.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 sigmoid2(float2 v) {  // as sigmoid_f
  float2 e = mul2(v, both(-1.4426950408889634f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
  e = add2(e, both(1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
  return e;
}
// The SiLU's slope at `pre`, whose sigmoid is s.
__device__ __forceinline__ float2 silu_slope(float2 pre, float2 s) {
  return mul2(s, fma2(pre, fma2(s, both(-1.f), both(1.f)), both(1.f)));
}

template <typename T, int V>
struct Norm {
  using Vec = Pack<T, V>;
  static constexpr int P = (V + 1) / 2;  // pairs of a vector (of one element: half of one)

  // vectors in flight
  static constexpr int kFlight = 4;

  static __device__ __forceinline__ float2 get(const Vec &v, int i) {
    if constexpr (V == 1) {
      return make_float2(v.f(0), 0.f);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const unsigned w = reinterpret_cast<const unsigned *>(v.v)[i];
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else if constexpr (std::is_same<T, __half>::value) {
      return __half22float2(reinterpret_cast<const __half2 *>(v.v)[i]);
    } else {
      return make_float2(v.v[2 * i], v.v[2 * i + 1]);
    }
  }
  static __device__ __forceinline__ void write(T *p, const float2 (&v)[P]) {
    Vec o;
    if constexpr (V > 1) {
      float x[V];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        x[2 * i] = v[i].x;
        x[2 * i + 1] = v[i].y;
      }
      o.set(x);
    } else {
      o.v[0] = from_f<T>(v[0].x);
    }
    o.store(p);
  }
  // number i of a vector's pairs
  static __device__ __forceinline__ float &at(float2 (&v)[P], int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }

  // ------------------------------------------------------------ channels last
  // Threads: `cols` vectors of channels by `rows` tokens; a slab of more
  // vectors than threads is gone through by columns of `cols`.
  struct Last {
    int sc, sv, cols, rows, r0, r1;
    int64_t base;  // of the slab's first channel at token 0
    __device__ Last(const NormArgs &a, const Place &p) {
      sc = min(a.slab_channels, a.C - p.slab * a.slab_channels);
      sv = sc / V;
      cols = min(sv, kThreads);
      rows = kThreads / cols;
      r0 = (int)((int64_t)p.len * p.rank / a.split);
      r1 = (int)((int64_t)p.len * (p.rank + 1) / a.split);
      base = (int64_t)p.n * a.P * a.C + (int64_t)p.slab * a.slab_channels;
    }
    __device__ float count(int ty) const { return (float)((r1 - r0 - ty + rows - 1) / rows); }
  };

  // Tokens behind the row's last: zeros.
  static __device__ void clear_last(const NormArgs &a, const Place &p, const Last &l) {
    const float2 zero[P] = {};
    const int behind = a.P - p.len, first = p.len + (int)((int64_t)behind * p.rank / a.split),
              last = p.len + (int)((int64_t)behind * (p.rank + 1) / a.split);
    for (int64_t i = threadIdx.x; i < (int64_t)(last - first) * l.sv; i += kThreads)
      write((T *)a.out + l.base + (first + i / l.sv) * a.C + i % l.sv * V, zero);
  }

  static __device__ void forward_last(const NormArgs &a, float *smem) {
    const Place p = place_of(a);
    const Last l(a, p);
    const T *x = (const T *)a.x;
    const int groups = l.sc / a.cg, tx = threadIdx.x % l.cols, ty = threadIdx.x / l.cols;
    float *red = smem;                                    // [rows][sc][2]
    float *mine = red + (size_t)2 * l.rows * l.sc;        // [groups][3]
    float *all = mine + 3 * groups, *stat = all + (size_t)a.split * 3 * groups;  // [split][groups][3], [groups][2]
    if (a.phase != kApply) {
      for (int c0 = 0; c0 < l.sv; c0 += l.cols) {
        const int col = c0 + tx;
        if (ty < l.rows && col < l.sv) {
          const T *at = x + l.base + col * V;
          float2 k[P] = {}, s[P] = {}, q[P] = {};
          const int first = l.r0 + ty;
          auto one = [&](const Vec &v) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 d = add2(get(v, i), k[i]);
              s[i] = add2(s[i], d);
              q[i] = fma2(d, d, q[i]);
            }
          };
          if (first < l.r1) {
            Vec v;
            v.load(at + (int64_t)first * a.C);
#pragma unroll
            for (int i = 0; i < P; ++i) k[i] = mul2(get(v, i), both(-1.f));
            int r = first + l.rows;
            for (; r + (kFlight - 1) * l.rows < l.r1; r += kFlight * l.rows) {
              Vec u[kFlight];
#pragma unroll
              for (int j = 0; j < kFlight; ++j) u[j].load(at + (int64_t)(r + j * l.rows) * a.C);
#pragma unroll
              for (int j = 0; j < kFlight; ++j) one(u[j]);
            }
            for (; r < l.r1; r += l.rows) {
              v.load(at + (int64_t)r * a.C);
              one(v);
            }
          }
          const float n = l.count(ty), inv = n > 0.f ? 1.f / n : 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float m = Norm::at(s, i) * inv;
            float *e = red + 2 * ((size_t)ty * l.sc + col * V + i);
            e[0] = n > 0.f ? m - Norm::at(k, i) : 0.f;
            e[1] = Norm::at(q, i) - Norm::at(s, i) * m;
          }
        }
      }
      __syncthreads();
      for (int g = threadIdx.x >> 5; g < groups; g += kWarps) {
        float n, mean, m2;
        join(red, l.rows * a.cg, [&](int i) { return 2 * ((i / a.cg) * l.sc + g * a.cg + i % a.cg); },
             [&](int i) { return l.count(i / a.cg); }, n, mean, m2);
        if ((threadIdx.x & 31) == 0) {
          mine[3 * g] = n;
          mine[3 * g + 1] = mean;
          mine[3 * g + 2] = m2;
        }
      }
    }
    if (!exchange(a, mine, 3 * groups, [&](auto &&number) {
          for (int i = threadIdx.x; i < a.split * 3 * groups; i += kThreads)
            all[i] = number(i / (3 * groups), i % (3 * groups));
        }))
      return;
    finish_stats(a, p, all, stat, groups, p.slab * a.slab_channels / a.cg);
    for (int c0 = 0; c0 < l.sv; c0 += l.cols) {
      const int col = c0 + tx;
      if (ty < l.rows && col < l.sv) {
        float2 mean[P] = {}, scale[P] = {}, shift[P] = {};  // (the mean's negative)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = col * V + i, g = c / a.cg, ch = p.slab * a.slab_channels + c;
          Norm::at(mean, i) = -stat[2 * g];
          Norm::at(scale, i) = stat[2 * g + 1] * load_w<T>(a.w, ch, a.wf32, 1.f);
          Norm::at(shift, i) = load_w<T>(a.b, ch, a.wf32, 0.f);
        }
        const int64_t at = l.base + col * V;
        auto one = [&](const Vec &v, int64_t e) {
          float2 y[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 pre = fma2(add2(get(v, i), mean[i]), scale[i], shift[i]);
            y[i] = a.silu ? mul2(pre, sigmoid2(pre)) : pre;
          }
          write((T *)a.out + e, y);
        };
        int r = l.r0 + ty;
        for (; r + (kFlight - 1) * l.rows < l.r1; r += kFlight * l.rows) {
          Vec u[kFlight];
#pragma unroll
          for (int j = 0; j < kFlight; ++j) u[j].load(x + at + (int64_t)(r + j * l.rows) * a.C);
#pragma unroll
          for (int j = 0; j < kFlight; ++j) one(u[j], at + (int64_t)(r + j * l.rows) * a.C);
        }
        for (; r < l.r1; r += l.rows) {
          Vec v;
          v.load(x + at + (int64_t)r * a.C);
          one(v, at + (int64_t)r * a.C);
        }
      }
    }
    clear_last(a, p, l);
  }

  // Joins the blocks' (count, mean, M2) of each group to (mean, rstd).
  static __device__ void finish_stats(const NormArgs &a, const Place &p, const float *all, float *stat, int groups,
                                      int first) {
    for (int g = threadIdx.x >> 5; g < groups; g += kWarps) {
      float n, mean, m2;
      join(all, a.split, [&](int i) { return 3 * (i * groups + g) + 1; }, [&](int i) { return all[3 * (i * groups + g)]; },
           n, mean, m2);
      const float rstd = n > 0.f ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
      if ((threadIdx.x & 31) == 0) {
        stat[2 * g] = mean;
        stat[2 * g + 1] = rstd;
        if (p.rank == 0 && a.stats) {
          float *s = a.stats + 2 * ((size_t)p.n * a.G + first + g);
          s[0] = mean;
          s[1] = rstd;
        }
      }
    }
    __syncthreads();
  }

  static __device__ void backward_last(const NormArgs &a, float *smem) {
    const Place p = place_of(a);
    const Last l(a, p);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    const int groups = l.sc / a.cg, tx = threadIdx.x % l.cols, ty = threadIdx.x / l.cols;
    float *red = smem;                                 // [rows][sc][2]
    float *mine = red + (size_t)2 * l.rows * l.sc;     // [sc][2]: sums of h and of h xhat
    float *chan = mine + 2 * l.sc, *sums = chan + 2 * l.sc;  // [sc][2]; [groups][2]: means of h w and of h w xhat
    const float *stats = a.stats + 2 * ((size_t)p.n * a.G + p.slab * a.slab_channels / a.cg);
    float2 mean[P] = {}, rstd[P] = {}, w[P] = {}, b[P] = {};  // (the mean's negative)
    auto channel = [&](int col) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = col * V + i, g = c / a.cg, ch = p.slab * a.slab_channels + c;
        Norm::at(mean, i) = -stats[2 * g];
        Norm::at(rstd, i) = stats[2 * g + 1];
        Norm::at(w, i) = load_w<T>(a.w, ch, a.wf32, 1.f);
        Norm::at(b, i) = load_w<T>(a.b, ch, a.wf32, 0.f);
      }
    };
    auto slope = [&](const Vec &vx, const Vec &vd, int i, float2 &xhat) {
      xhat = mul2(add2(get(vx, i), mean[i]), rstd[i]);
      const float2 h = get(vd, i);
      if (!a.silu) return h;
      const float2 pre = fma2(xhat, w[i], b[i]);
      return mul2(h, silu_slope(pre, sigmoid2(pre)));
    };
    if (a.phase != kApply) {
      for (int c0 = 0; c0 < l.sv; c0 += l.cols) {
        const int col = c0 + tx;
        if (ty < l.rows && col < l.sv) {
          channel(col);
          const int64_t at = l.base + col * V;
          float2 s[P] = {}, q[P] = {};
          auto one = [&](const Vec &vx, const Vec &vd) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              float2 xhat;
              const float2 h = slope(vx, vd, i, xhat);
              s[i] = add2(s[i], h);
              q[i] = fma2(h, xhat, q[i]);
            }
          };
          int r = l.r0 + ty;
          for (; r + l.rows < l.r1; r += 2 * l.rows) {
            Vec u[2], d[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              u[j].load(x + at + (int64_t)(r + j * l.rows) * a.C);
              d[j].load(dy + at + (int64_t)(r + j * l.rows) * a.C);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) one(u[j], d[j]);
          }
          for (; r < l.r1; r += l.rows) {
            Vec u, d;
            u.load(x + at + (int64_t)r * a.C);
            d.load(dy + at + (int64_t)r * a.C);
            one(u, d);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float *e = red + 2 * ((size_t)ty * l.sc + col * V + i);
            e[0] = Norm::at(s, i);
            e[1] = Norm::at(q, i);
          }
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * l.sc; i += kThreads) {
        float s = 0.f;
        for (int r = 0; r < l.rows; ++r) s += red[(size_t)2 * r * l.sc + i];
        mine[i] = s;
      }
    }
    if (!exchange(a, mine, 2 * l.sc, [&](auto &&number) { join_sums(a, chan, l.sc, number); })) return;
    finish_sums(a, p, sums, chan, l.sc, groups, p.slab * a.slab_channels);
    for (int c0 = 0; c0 < l.sv; c0 += l.cols) {
      const int col = c0 + tx;
      if (ty < l.rows && col < l.sv) {
        channel(col);
        float2 hw[P] = {}, hx[P] = {};  // (their negatives)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          Norm::at(hw, i) = -sums[2 * ((col * V + i) / a.cg)];
          Norm::at(hx, i) = -sums[2 * ((col * V + i) / a.cg) + 1];
        }
        const int64_t at = l.base + col * V;
        auto one = [&](const Vec &vx, const Vec &vd, int64_t e) {
          float2 o[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            float2 xhat;
            const float2 h = slope(vx, vd, i, xhat);
            o[i] = mul2(rstd[i], fma2(xhat, hx[i], fma2(h, w[i], hw[i])));
          }
          write((T *)a.out + e, o);
        };
        int r = l.r0 + ty;
        for (; r + l.rows < l.r1; r += 2 * l.rows) {
          Vec u[2], d[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            u[j].load(x + at + (int64_t)(r + j * l.rows) * a.C);
            d[j].load(dy + at + (int64_t)(r + j * l.rows) * a.C);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) one(u[j], d[j], at + (int64_t)(r + j * l.rows) * a.C);
        }
        for (; r < l.r1; r += l.rows) {
          Vec u, d;
          u.load(x + at + (int64_t)r * a.C);
          d.load(dy + at + (int64_t)r * a.C);
          one(u, d, at + (int64_t)r * a.C);
        }
      }
    }
    clear_last(a, p, l);
  }

  // Joins the blocks' sums of a slab's channels.
  template <typename Number>
  static __device__ __forceinline__ void join_sums(const NormArgs &a, float *chan, int sc, Number &&number) {
    for (int i = threadIdx.x; i < 2 * sc; i += kThreads) {
      float s = 0.f;
      for (int r = 0; r < a.split; ++r) s += number(r, i);
      chan[i] = s;
    }
  }

  // Keeps them for dw and db; the means over each group.
  static __device__ void finish_sums(const NormArgs &a, const Place &p, float *sums, const float *chan, int sc,
                                     int groups, int first) {
    if (p.rank == 0 && a.chan)
      for (int i = threadIdx.x; i < 2 * sc; i += kThreads) a.chan[2 * ((size_t)p.n * a.C + first) + i] = chan[i];
    const float inv = p.len > 0 ? 1.f / ((float)p.len * a.cg) : 0.f;
    for (int g = threadIdx.x >> 5; g < groups; g += kWarps) {
      float s = 0.f, q = 0.f;
      for (int i = threadIdx.x & 31; i < a.cg; i += 32) {
        const int c = g * a.cg + i;
        const float w = load_w<T>(a.w, first + c, a.wf32, 1.f);
        s += w * chan[2 * c];
        q += w * chan[2 * c + 1];
      }
      s = warp_sum(s);
      q = warp_sum(q);
      if ((threadIdx.x & 31) == 0) {
        sums[2 * g] = s * inv;
        sums[2 * g + 1] = q * inv;
      }
    }
    __syncthreads();
  }

  // ----------------------------------------------------------- channels first
  // A slab is one group.  Each row (channel) is cut into `segs` pieces of `seg`
  // vectors; 2^k neighbouring lanes take a piece, and a block a run of pieces.
  struct First {
    int lanes, lane, who, takers, begin, end;
    int64_t base;
    __device__ First(const NormArgs &a, const Place &p) {
      lanes = 32;
      while (lanes > 1 && lanes / 2 >= a.seg) lanes >>= 1;
      lane = threadIdx.x % lanes;
      who = threadIdx.x / lanes;
      takers = kThreads / lanes;
      const int64_t pieces = (int64_t)a.cg * a.segs;
      begin = (int)(pieces * p.rank / a.split);
      end = (int)(pieces * (p.rank + 1) / a.split);
      base = ((int64_t)p.n * a.C + (int64_t)p.slab * a.cg) * a.P;
    }
  };

  // Calls body(row, first token, last token) for this thread's pieces, the
  // tokens cut at `len`.
  template <typename Body>
  static __device__ __forceinline__ void pieces(const NormArgs &a, const First &f, int len, Body &&body) {
    for (int i = f.begin + f.who; i < f.end; i += f.takers) {
      const int row = i / a.segs, t0 = (i - row * a.segs) * a.seg * V;
      body(i, row, t0, min(t0 + a.seg * V, len));
    }
  }

  static __device__ void clear_first(const NormArgs &a, const Place &p, const First &f) {
    if (p.len == a.P) return;
    const float2 zero[P] = {};
    pieces(a, f, a.P, [&](int, int row, int t0, int t1) {
      T *out = (T *)a.out + f.base + (int64_t)row * a.P;
      // (a vector that the row's last token is in has been written)
      for (int t = t0 + f.lane * V; t < t1; t += f.lanes * V)
        if (t >= p.len) write(out + t, zero);
    });
  }

  static __device__ void forward_first(const NormArgs &a, float *smem) {
    const Place p = place_of(a);
    const First f(a, p);
    const T *x = (const T *)a.x;
    float *red = smem, *mine = red + 3 * kThreads, *all = mine + 3, *stat = all + 3 * a.split;
    if (a.phase != kApply) {
      float k = 0.f;
      float2 s2 = {}, q2 = {};
      int n = 0;
      pieces(a, f, p.len, [&](int, int row, int t0, int t1) {
        const T *at = x + f.base + (int64_t)row * a.P;
        // a vector of `left` tokens, all of them or (at a row's last) some
        auto one = [&](const Vec &v, int left) {
          left = min(left, V);
          if (n == 0) k = v.f(0);
          n += left;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            float2 d = add2(get(v, i), both(-k));
            if (left < V || V == 1) d = make_float2(2 * i < left ? d.x : 0.f, 2 * i + 1 < left ? d.y : 0.f);
            s2 = add2(s2, d);
            q2 = fma2(d, d, q2);
          }
        };
        int t = t0 + f.lane * V;
        for (; t + ((kFlight - 1) * f.lanes + 1) * V <= t1; t += kFlight * f.lanes * V) {
          Vec u[kFlight];
#pragma unroll
          for (int j = 0; j < kFlight; ++j) u[j].load(at + t + j * f.lanes * V);
#pragma unroll
          for (int j = 0; j < kFlight; ++j) one(u[j], V);
        }
        for (; t < t1; t += f.lanes * V) {
          Vec v;
          v.load(at + t);
          one(v, t1 - t);
        }
      });
      const float s = s2.x + s2.y, q = q2.x + q2.y;
      const float m = n ? s / n : 0.f;
      float *e = red + 3 * threadIdx.x;
      e[0] = (float)n;
      e[1] = n ? k + m : 0.f;
      e[2] = q - s * m;
      __syncthreads();
      if (threadIdx.x < 32) {
        float total, mean, m2;
        join(red, kThreads, [](int i) { return 3 * i + 1; }, [&](int i) { return red[3 * i]; }, total, mean, m2);
        if (threadIdx.x == 0) {
          mine[0] = total;
          mine[1] = mean;
          mine[2] = m2;
        }
      }
    }
    if (!exchange(a, mine, 3, [&](auto &&number) {
          for (int i = threadIdx.x; i < a.split * 3; i += kThreads) all[i] = number(i / 3, i % 3);
        }))
      return;
    finish_stats(a, p, all, stat, 1, p.slab);
    const float mean = stat[0], rstd = stat[1];
    pieces(a, f, p.len, [&](int, int row, int t0, int t1) {
      const int64_t at = f.base + (int64_t)row * a.P;
      const int ch = p.slab * a.cg + row;
      const float2 scale = both(rstd * load_w<T>(a.w, ch, a.wf32, 1.f)), shift = both(load_w<T>(a.b, ch, a.wf32, 0.f));
      auto one = [&](const Vec &v, int t) {
        float2 y[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 pre = fma2(add2(get(v, i), both(-mean)), scale, shift);
          y[i] = a.silu ? mul2(pre, sigmoid2(pre)) : pre;
          if (t + V > t1) y[i] = make_float2(t + 2 * i < t1 ? y[i].x : 0.f, t + 2 * i + 1 < t1 ? y[i].y : 0.f);
        }
        write((T *)a.out + at + t, y);
      };
      int t = t0 + f.lane * V;
      for (; t + ((kFlight - 1) * f.lanes + 1) * V <= t1; t += kFlight * f.lanes * V) {
        Vec u[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) u[j].load(x + at + t + j * f.lanes * V);
#pragma unroll
        for (int j = 0; j < kFlight; ++j) one(u[j], t + j * f.lanes * V);
      }
      for (; t < t1; t += f.lanes * V) {
        Vec v;
        v.load(x + at + t);
        one(v, t);
      }
    });
    clear_first(a, p, f);
  }

  static __device__ void backward_first(const NormArgs &a, float *smem) {
    const Place p = place_of(a);
    const First f(a, p);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    const int most = (int)(((int64_t)a.cg * a.segs + a.split - 1) / a.split) + 1;  // pieces of a block
    float *red = smem;                                   // [pieces][2]
    float *mine = red + (size_t)2 * most;                // [cg][2]
    float *chan = mine + 2 * a.cg, *sums = chan + 2 * a.cg;
    const float *stats = a.stats + 2 * ((size_t)p.n * a.G + p.slab);
    const float mean = stats[0], rstd = stats[1];
    float w = 0.f, b = 0.f;
    auto slope = [&](const Vec &vx, const Vec &vd, int i, float2 &xhat) {
      xhat = mul2(add2(get(vx, i), both(-mean)), both(rstd));
      const float2 h = get(vd, i);
      if (!a.silu) return h;
      const float2 pre = fma2(xhat, both(w), both(b));
      return mul2(h, silu_slope(pre, sigmoid2(pre)));
    };
    // pair i of a vector that has `left` tokens, with zeros behind them
    auto held = [&](float2 v, int i, int left) {
      left = min(left, V);
      return left == V && V > 1 ? v : make_float2(2 * i < left ? v.x : 0.f, 2 * i + 1 < left ? v.y : 0.f);
    };
    auto channel = [&](int row) {
      w = load_w<T>(a.w, p.slab * a.cg + row, a.wf32, 1.f);
      b = load_w<T>(a.b, p.slab * a.cg + row, a.wf32, 0.f);
    };
    // body(x, dy, token) for this thread's vectors of a piece, two in flight
    auto vectors = [&](int64_t at, int t0, int t1, auto &&body) {
      int t = t0 + f.lane * V;
      for (; t + f.lanes * V < t1; t += 2 * f.lanes * V) {
        Vec u[2], d[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u[j].load(x + at + t + j * f.lanes * V);
          d[j].load(dy + at + t + j * f.lanes * V);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) body(u[j], d[j], t + j * f.lanes * V);
      }
      if (t < t1) {
        Vec u, d;
        u.load(x + at + t);
        d.load(dy + at + t);
        body(u, d, t);
      }
    };
    if (a.phase != kApply) {
      // (all lanes of a warp go through the same number of pieces)
      for (int i0 = f.begin; i0 < f.end; i0 += f.takers) {
        const int i = i0 + f.who;
        float2 s2 = {}, q2 = {};
        if (i < f.end) {
          const int row = i / a.segs, t0 = (i - row * a.segs) * a.seg * V, t1 = min(t0 + a.seg * V, p.len);
          channel(row);
          vectors(f.base + (int64_t)row * a.P, t0, t1, [&](const Vec &u, const Vec &d, int t) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
              float2 xhat;
              const float2 h = held(slope(u, d, j, xhat), j, t1 - t);
              s2 = add2(s2, h);
              q2 = add2(q2, held(mul2(h, xhat), j, t1 - t));
            }
          });
        }
        float s = s2.x + s2.y, q = q2.x + q2.y;
        for (int o = f.lanes >> 1; o; o >>= 1) {
          s += __shfl_xor_sync(0xffffffffu, s, o);
          q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (i < f.end && f.lane == 0) {
          red[2 * (i - f.begin)] = s;
          red[2 * (i - f.begin) + 1] = q;
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * a.cg; i += kThreads) {
        const int row = i >> 1;
        float s = 0.f;
        for (int j = max(f.begin, row * a.segs); j < min(f.end, (row + 1) * a.segs); ++j)
          s += red[2 * (j - f.begin) + (i & 1)];
        mine[i] = s;
      }
    }
    if (!exchange(a, mine, 2 * a.cg, [&](auto &&number) { join_sums(a, chan, a.cg, number); })) return;
    finish_sums(a, p, sums, chan, a.cg, 1, p.slab * a.cg);
    const float hw = sums[0], hx = sums[1];
    pieces(a, f, p.len, [&](int, int row, int t0, int t1) {
      channel(row);
      const int64_t at = f.base + (int64_t)row * a.P;
      vectors(at, t0, t1, [&](const Vec &u, const Vec &d, int t) {
        float2 o[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          float2 xhat;
          const float2 h = slope(u, d, j, xhat);
          o[j] = held(mul2(both(rstd), fma2(xhat, both(-hx), fma2(h, both(w), both(-hw)))), j, t1 - t);
        }
        write((T *)a.out + at + t, o);
      });
    });
    clear_first(a, p, f);
  }
};

template <typename T, int V, bool kLast, bool kBackward>
__global__ void __launch_bounds__(kThreads, 3) norm_kernel(const NormArgs a) {
  extern __shared__ float smem[];
  if constexpr (kLast && kBackward) Norm<T, V>::backward_last(a, smem);
  else if constexpr (kLast) Norm<T, V>::forward_last(a, smem);
  else if constexpr (kBackward) Norm<T, V>::backward_first(a, smem);
  else Norm<T, V>::forward_first(a, smem);
}

// dw and db: the batch rows' sums of a channel, in 64 bits.
template <typename W>
__global__ void __launch_bounds__(kThreads) norm_weight_kernel(const float *chan, int batch, int C, W *dw, W *db) {
  // a warp takes 32 numbers of neighbouring channels, the block's warps share the batch
  __shared__ double red[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  double s = 0.0;
  if (i < 2 * (int64_t)C)
    for (int n = warp; n < batch; n += kWarps) s += chan[(size_t)n * 2 * C + i];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < 2 * (int64_t)C) {
    for (int k = 1; k < kWarps; ++k) s += red[k][lane];
    W *out = i & 1 ? dw : db;
    if (out) out[i >> 1] = from_f<W>((float)s);
  }
}

// The launch of a problem: how its slabs are cut and shared.
struct Plan {
  int V, slab_channels, slabs, split, seg, segs;
  bool fused;
  size_t numbers;  // of a block's part
  size_t smem, part_bytes;
};

Plan make_plan(int size, bool last, bool backward, int batch, int C, int P, int G, bool vectors) {
  Plan p{};
  const int cg = C / G;
  const int widest = 16 / size, line = last ? C : P;
  // the widest vectors (16 bytes, or two elements, or one) that rows keep to
  for (int v : {widest, 2, 1}) {
    if (v > 1 && (!vectors || line % v || (v == 2 && size == 4))) continue;
    p.V = v;
    p.slab_channels = cg;
    if (!last) break;
    // whole groups, whole vectors and 128 bytes of a token (the L2 cache's line) where the channels allow it
    while (p.slab_channels < C && (p.slab_channels % v || p.slab_channels * size < 128)) p.slab_channels += cg;
    if (p.slab_channels <= kMaxChannels) break;
  }
  p.slabs = ceil_div(C, p.slab_channels);
  const int64_t units = (int64_t)batch * p.slabs, elements = (int64_t)p.slab_channels * P;
  // A block of 256 threads wants a few vectors a thread; the GPU wants some blocks for each SM.
  const int64_t useful = std::max<int64_t>(1, elements / (kThreads * widest * 2));
  const int64_t wanted = (int64_t)device_sm_count() * 4;
  int64_t split = 1;
  while (split < kMaxSplit && split * 2 <= useful && units * split < wanted) split *= 2;
  // Clusters of up to 8 blocks; more blocks share a slab by two launches, where the clusters would leave most of
  // the GPU without work.
  p.fused = true;
  if (split > kMaxCluster) {
    if (units * kMaxCluster >= device_sm_count()) split = kMaxCluster;
    else p.fused = false;
  }
  p.split = (int)split;
  if (!last) {
    // pieces of a row: as many as give every taker of every block one
    const int vectors_of_row = ceil_div(P, p.V);
    const int64_t takers = (int64_t)kWarps * split;
    p.segs = (int)std::min<int64_t>(std::max<int64_t>(1, (takers + cg - 1) / cg), std::max(1, vectors_of_row / 32));
    p.seg = ceil_div(vectors_of_row, p.segs);
    p.segs = std::max(1, ceil_div(vectors_of_row, std::max(1, p.seg)));
    p.seg = std::max(1, p.seg);
  }
  const int sc = p.slab_channels, groups = sc / cg;
  p.numbers = backward ? 2 * (size_t)sc : 3 * (size_t)groups;
  size_t red;
  if (last) red = 2 * (size_t)std::max(kThreads * p.V, sc);
  else if (backward) red = 2 * ((size_t)ceil_div((int64_t)cg * p.segs, p.split) + 1);
  else red = 3 * kThreads;
  p.smem = 4 * (red + p.numbers * (backward ? 2 : 1 + p.split) + 2 * (size_t)groups);
  p.part_bytes = p.fused ? 0 : (size_t)units * p.split * p.numbers * 4;
  return p;
}

template <typename T, int V, bool kLast, bool kBackward>
int launch_norm(const Plan &p, NormArgs a, cudaStream_t stream) {
  auto *kernel = norm_kernel<T, V, kLast, kBackward>;
  static PerContext<uint64_t> allowed;
  int st = once_per_context(allowed, 1, [&]() -> int {
    PC2D_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    return PC2D_OK;
  });
  if (st != PC2D_OK) return st;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)((int64_t)a.batch * a.slabs * a.split));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = p.smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)a.split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  if (p.fused) {
    a.phase = kFused;
    if (a.split > 1) {
      config.attrs = &cluster;
      config.numAttrs = 1;
    }
    PC2D_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a));
    return PC2D_OK;
  }
  a.phase = kSums;
  PC2D_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a));
  a.phase = kApply;
  PC2D_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a));
  return PC2D_OK;
}

template <typename T, bool kBackward>
int launch_type(const Plan &p, bool last, const NormArgs &a, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(T);
  if (p.V == W)
    return last ? launch_norm<T, W, true, kBackward>(p, a, stream) : launch_norm<T, W, false, kBackward>(p, a, stream);
  if constexpr (sizeof(T) == 2)
    if (p.V == 2)
      return last ? launch_norm<T, 2, true, kBackward>(p, a, stream)
                  : launch_norm<T, 2, false, kBackward>(p, a, stream);
  return last ? launch_norm<T, 1, true, kBackward>(p, a, stream) : launch_norm<T, 1, false, kBackward>(p, a, stream);
}

int check_norm(const char *what, int dtype, int wdtype, int batch, int channels, int length, int groups) {
  if (!seq_dtype(dtype) || (wdtype != dtype && wdtype != PC2D_DTYPE_F32)) {
    set_last_error("%s: unsupported dtypes %d and %d", what, dtype, wdtype);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (batch < 0 || channels < 1 || length < 0 || groups < 1 || channels % groups) {
    set_last_error("%s: invalid sizes (batch %d, channels %d, length %d, groups %d)", what, batch, channels, length,
                   groups);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (length > 1 << 30 || channels / groups > kMaxChannels || (int64_t)batch * groups > 1 << 24) {
    set_last_error("%s: at most 2^30 positions, %d channels a group and 2^24 groups in all", what, kMaxChannels);
    return PC2D_ERR_UNSUPPORTED;
  }
  return PC2D_OK;
}

}  // namespace
}  // namespace pc2d

using namespace pc2d;

extern "C" size_t pc2d_group_norm_workspace_size(int dtype, int channels_last, int batch, int channels, int length,
                                                 int groups, int backward) {
  if (check_norm("pc2d_group_norm_workspace_size", dtype, dtype, batch, channels, length, groups) != PC2D_OK) return 0;
  // (whether vectors can be used is not known yet: the larger of the two needs)
  size_t most = 0;
  for (bool vectors : {false, true})
    most = std::max(most, make_plan((int)seq_dtype_size(dtype), channels_last || length == 1, backward, batch, channels,
                                    length, groups, vectors)
                              .part_bytes);
  return align_up(most, 256) + (backward ? (size_t)batch * channels * 8 : 0);
}

extern "C" int pc2d_group_norm_forward(int dtype, int wdtype, int channels_last, const void *input, const void *weight,
                                       const void *bias, const int *lengths, int batch, int channels, int length,
                                       int groups, double eps, int silu, void *output, float *stats, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  NvtxRange range("pc2d_group_norm_forward");
  const char *what = "pc2d_group_norm_forward";
  int st = check_norm(what, dtype, wdtype, batch, channels, length, groups);
  if (st != PC2D_OK) return st;
  if (!(eps >= 0.0)) {
    set_last_error("%s: eps must be non-negative", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if (!batch || !length) return PC2D_OK;
  const size_t size = seq_dtype_size(dtype);
  if (!input || !output) {
    set_last_error("%s: null pointer (input or output)", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_elements(what, size, {input, output})) != PC2D_OK ||
      (st = check_elements(what, seq_dtype_size(wdtype), {weight, bias})) != PC2D_OK ||
      (st = check_elements(what, 4, {lengths, stats})) != PC2D_OK || (st = pending_device_error()) != PC2D_OK)
    return st;
  const bool last = channels_last || length == 1;
  const Plan p = make_plan((int)size, last, false, batch, channels, length, groups,
                           aligned16(input) && aligned16(output));
  if (p.part_bytes && (!workspace || workspace_bytes < p.part_bytes || !aligned16(workspace))) {
    set_last_error("%s: workspace of %zu bytes on a 16-byte boundary needed", what, p.part_bytes);
    return PC2D_ERR_WORKSPACE;
  }
  NormArgs a{};
  a.x = input;
  a.w = weight;
  a.b = bias;
  a.lengths = lengths;
  a.out = output;
  a.stats = stats;
  a.part = static_cast<float *>(workspace);
  a.batch = batch;
  a.C = channels;
  a.P = length;
  a.G = groups;
  a.cg = channels / groups;
  a.slab_channels = p.slab_channels;
  a.slabs = p.slabs;
  a.split = p.split;
  a.seg = p.seg;
  a.segs = p.segs;
  a.wf32 = wdtype == PC2D_DTYPE_F32;
  a.silu = silu;
  a.eps = (float)eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PC2D_DTYPE_F32: return launch_type<float, false>(p, last, a, s);
    case PC2D_DTYPE_F16: return launch_type<__half, false>(p, last, a, s);
    default: return launch_type<__nv_bfloat16, false>(p, last, a, s);
  }
}

extern "C" int pc2d_group_norm_backward(int dtype, int wdtype, int channels_last, const void *grad, const void *input,
                                        const void *weight, const void *bias, const int *lengths, const float *stats,
                                        int batch, int channels, int length, int groups, int silu, void *inputgrad,
                                        void *weightgrad, void *biasgrad, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  NvtxRange range("pc2d_group_norm_backward");
  const char *what = "pc2d_group_norm_backward";
  int st = check_norm(what, dtype, wdtype, batch, channels, length, groups);
  if (st != PC2D_OK) return st;
  const size_t size = seq_dtype_size(dtype), wsize = seq_dtype_size(wdtype);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!batch || !length) {
    if ((st = pending_device_error()) != PC2D_OK) return st;
    for (void *p : {weightgrad, biasgrad})
      if (p) PC2D_CUDA_CHECK(cudaMemsetAsync(p, 0, channels * wsize, s));
    return PC2D_OK;
  }
  if (!grad || !input || !stats || !inputgrad) {
    set_last_error("%s: null pointer (grad, input, stats or inputgrad)", what);
    return PC2D_ERR_INVALID_ARGUMENT;
  }
  if ((st = check_elements(what, size, {grad, input, inputgrad})) != PC2D_OK ||
      (st = check_elements(what, wsize, {weight, bias, weightgrad, biasgrad})) != PC2D_OK ||
      (st = check_elements(what, 4, {lengths, stats})) != PC2D_OK || (st = pending_device_error()) != PC2D_OK)
    return st;
  const bool last = channels_last || length == 1;
  const Plan p = make_plan((int)size, last, true, batch, channels, length, groups,
                           aligned16(input) && aligned16(grad) && aligned16(inputgrad));
  const size_t part = align_up(p.part_bytes, 256), need = part + (size_t)batch * channels * 8;
  if (!workspace || workspace_bytes < need || !aligned16(workspace)) {
    set_last_error("%s: workspace of %zu bytes on a 16-byte boundary needed", what, need);
    return PC2D_ERR_WORKSPACE;
  }
  NormArgs a{};
  a.x = input;
  a.dy = grad;
  a.w = weight;
  a.b = bias;
  a.lengths = lengths;
  a.out = inputgrad;
  a.stats = const_cast<float *>(stats);
  a.part = static_cast<float *>(workspace);
  a.chan = reinterpret_cast<float *>(static_cast<char *>(workspace) + part);
  a.batch = batch;
  a.C = channels;
  a.P = length;
  a.G = groups;
  a.cg = channels / groups;
  a.slab_channels = p.slab_channels;
  a.slabs = p.slabs;
  a.split = p.split;
  a.seg = p.seg;
  a.segs = p.segs;
  a.wf32 = wdtype == PC2D_DTYPE_F32;
  a.silu = silu;
  if (!weightgrad && !biasgrad) a.chan = nullptr;
  switch (dtype) {
    case PC2D_DTYPE_F32: st = launch_type<float, true>(p, last, a, s); break;
    case PC2D_DTYPE_F16: st = launch_type<__half, true>(p, last, a, s); break;
    default: st = launch_type<__nv_bfloat16, true>(p, last, a, s);
  }
  if (st != PC2D_OK || !a.chan) return st;
  const unsigned grid = (unsigned)ceil_div(2 * (int64_t)channels, 32);
  if (wdtype == PC2D_DTYPE_F32)
    norm_weight_kernel<<<grid, kThreads, 0, s>>>(a.chan, batch, channels, (float *)weightgrad, (float *)biasgrad);
  else if (wdtype == PC2D_DTYPE_F16)
    norm_weight_kernel<<<grid, kThreads, 0, s>>>(a.chan, batch, channels, (__half *)weightgrad, (__half *)biasgrad);
  else
    norm_weight_kernel<<<grid, kThreads, 0, s>>>(a.chan, batch, channels, (__nv_bfloat16 *)weightgrad,
                                                 (__nv_bfloat16 *)biasgrad);
  PC2D_LAUNCH_CHECK("norm_weight_kernel");
  return PC2D_OK;
}
