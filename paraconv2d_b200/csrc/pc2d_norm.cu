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
// blocks' work.  They bring it into shared memory by asynchronous copies, all
// under way at once, sum, exchange their sums through distributed shared memory,
// and go over it again there; what does not fit is read again, from the L2
// cache as a rule.  Each thread reads only what it has copied.
// Measured (one B200; of a training step, forwards / backwards): 64x128x56x56
// float32 43 / 71 us, 4.8 and 4.3 TB/s of the two or three passes over the map
// that have to be; 16x512x64x64 bfloat16 channels last 51 / 87 us, 2.6 and 2.3
// TB/s.  The first is near the memory's time; the second is bound by the
// exponentials and reciprocals of the sigmoid (two an element forwards, four
// backwards: at least 15 and 30 us) and by the chain load, sum, exchange, go
// over it again, which few blocks of an SM hide.  A small call (2x320x17x31
// float16) is that chain alone: 10.5 us.  Where there are too few slabs for the GPU, two launches
// share the same code and exchange the partial sums in device memory instead.
//
// Variance: each thread sums x - K and its square, K its own first value (of
// the channel, channels last), and the (count, mean, M2) of threads, warps and
// blocks are joined by M2 = sum M2_i + n_i (mean_i - mean)^2.  Neither a large
// mean nor a single outlier cancels: a thread's sums are off by 2^-24 of
// squares that the slab's M2 holds too, once per element of a run of the thread.
// Runs are at most kRun vectors: a sum over tens of thousands of squares rounds
// the small ones among them away, all to one side (65,536 a thread: 7e-5 of the
// variance).  All joins go by fixed orders.
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
constexpr int kRun = 256;             // vectors of a thread that are summed before they are joined with those before
constexpr int kMaxSplit = 64;         // blocks of a slab that exchange through device memory
constexpr int kMaxChannels = 8192;    // of a slab: its sums are in shared memory
constexpr int kCacheBytes = 64 * 1024;  // of a slab's share that a block keeps, x and dy together

enum Phase { kFused, kSums, kApply };

struct NormArgs {
  const void *x, *dy, *w, *b;
  const int *lengths;
  void *out;            // y, or dx
  float *stats;         // [batch][groups][2]: mean and rstd
  float *part;          // kSums, kApply: [slab][split][numbers of a block]
  int numbers;          // of a block of a whole slab: what the blocks' parts lie apart (the last slab may have fewer)
  float *chan;          // backward: [batch][channels][2], sums of h and of h xhat
  int batch, C, P, G, cg;
  int slab_channels;    // channels of a slab: cg, or a multiple of it
  int slabs;            // slabs of a batch row
  int split, split_log;  // blocks of a slab, a power of two
  int cols_log;         // channels last: 2^cols_log threads for the vectors of a slab's token
  int seg, segs;        // channels first: vectors and number of the pieces of a row
  int red;              // channels last: numbers of the block's partial sums
  int cache;            // vectors of an array that a thread keeps in shared memory
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

// (Integer divisions are chains of tens of dependent instructions, which is what
// a small block's time would go to: powers of two where that can be arranged,
// and numbers that the host has divided.)

// Where part i of 2^log equal parts of n begins.
__device__ __forceinline__ int part_of(int n, int i, int log) {
  const int each = n >> log;
  return i * each + min(i, n - (each << log));
}

struct Place {
  int rank, n, slab, len;  // block of its slab; batch row; slab of the row; tokens of the row
};
__device__ __forceinline__ Place place_of(const NormArgs &a) {
  Place p;
  p.rank = blockIdx.x & (a.split - 1);
  const int unit = blockIdx.x >> a.split_log;
  p.n = a.slabs == 1 ? unit : unit / a.slabs;
  p.slab = unit - p.n * a.slabs;
  p.len = a.lengths ? min(max(a.lengths[p.n], 0), a.P) : a.P;
  return p;
}

// Calls take(numbers) with a function that gives number i of block r of this
// slab, once the `count` numbers that every block has in `mine` are known to
// all of its blocks.  False: this block is done.
template <typename Take>
__device__ __forceinline__ bool exchange(const NormArgs &a, const float *mine, int count, Take &&take) {
  const int rank = blockIdx.x & (a.split - 1);
  float *global = a.part + (size_t)(blockIdx.x - rank) * a.numbers;
  __syncthreads();
  if (a.phase == kSums) {
    for (int i = threadIdx.x; i < count; i += kThreads) global[(size_t)rank * a.numbers + i] = mine[i];
    return false;
  }
  if (a.phase == kApply) {
    take([&](int r, int i) { return global[(size_t)r * a.numbers + i]; });
  } else if (a.split == 1) {
    take([&](int, int i) { return mine[i]; });
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    take([&](int r, int i) { return cluster.map_shared_rank(mine, r)[i]; });
    cluster.barrier_arrive();  // (and leave() at the end)
  }
  __syncthreads();
  return true;
}
// Nobody leaves while others may still read its numbers.
__device__ __forceinline__ void leave(const NormArgs &a) {
  if (a.phase == kFused && a.split > 1) cg::this_cluster().barrier_wait();
}

// (count, mean, M2) of rows x cols entries by one warp, the mean and the M2 of
// entry (r, c) at v[at(r, c)] and v[at(r, c) + 1] and its count n(r).
template <typename At, typename Count>
__device__ __forceinline__ void join(const float *v, int rows, int cols, At &&at, Count &&n, float &total, float &mean,
                                     float &m2) {
  // lanes: 2^k columns by 32 / 2^k rows (no division, whose chain would be longer than all of this)
  const int lane = threadIdx.x & 31, shift = cols >= 32 ? 5 : 31 - __clz(cols);
  auto each = [&](auto &&f) {
    for (int r = lane >> shift; r < rows; r += 32 >> shift) {
      const float k = n(r);
      for (int c = lane & ((1 << shift) - 1); c < cols; c += 1 << shift) f(at(r, c), k);
    }
  };
  float c = 0.f, s = 0.f, q = 0.f;
  each([&](int i, float k) {
    c += k;
    s += k * v[i];
  });
  total = warp_sum(c);
  mean = total > 0.f ? warp_sum(s) / total : 0.f;
  // (the differences from it, whose sum corrects its rounding)
  s = 0.f;
  each([&](int i, float k) {
    const float d = k > 0.f ? v[i] - mean : 0.f;
    s = fmaf(k, d, s);
    q += k > 0.f ? v[i + 1] + k * d * d : 0.f;
  });
  s = total > 0.f ? warp_sum(s) / total : 0.f;
  m2 = warp_sum(q) - total * s * s;
  mean += s;
}

// Pairs of numbers, one instruction for two.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
// A product that no sum takes in (the intrinsics' products may become part of a fused one).
__device__ __forceinline__ float2 mul2_rounded(float2 a, float2 b) {
  return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y));
}
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
  static_assert(kThreads == 256, "Last");
  static constexpr int P = (V + 1) / 2;  // pairs of a vector (of one element: half of one)

  struct Two {
    Vec x, d;
  };

  // vectors in flight
  static constexpr int kFlight = 2;
  // pairs of vectors in the backward pass, where half of a large slab has no room in shared memory: four take the
  // registers of two blocks an SM, which 16-bit types gain from (16x512x64x64 bfloat16, both passes: 148 to 139 us)
  // and float32 loses by (64x128x56x56: 118 to 127 us)
  static constexpr int kFlightTwo = sizeof(T) == 2 ? 4 : 2;

  // The weights of channels ch .. ch+V-1, or `none`.
  static __device__ __forceinline__ void weights(float2 (&v)[P], const void *p, int ch, bool f32, float none) {
    if (!p) {
#pragma unroll
      for (int i = 0; i < V; ++i) at(v, i) = none;
    } else if (f32) {
#pragma unroll
      for (int i = 0; i < V; ++i) at(v, i) = static_cast<const float *>(p)[ch + i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) at(v, i) = to_f(static_cast<const T *>(p)[ch + i]);
    }
  }
  // f(i, group of channel c + i) for the V channels from c on of a slab
  template <typename F>
  static __device__ __forceinline__ void with_groups(int c, int cg, F &&f) {
    int g = c / cg, left = cg - (c - g * cg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f(i, g);
      if (--left == 0) left = cg, ++g;
    }
  }

  static constexpr bool kKeeps = V * sizeof(T) == 16;
  // Vector `slot` of this thread, from `p`: copied ahead, and taken from the copy where there is one.
  static __device__ __forceinline__ void ahead(const NormArgs &a, unsigned char *kept, int slot, const T *p) {
    if constexpr (kKeeps) {
      const unsigned to = (unsigned)__cvta_generic_to_shared(kept + ((size_t)slot * kThreads + threadIdx.x) * 16);
      if (slot < a.cache) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
    }
  }
  static __device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_all;" ::: "memory"); }
  static __device__ __forceinline__ Vec copied(const unsigned char *kept, int slot) {
    Vec v;
    *reinterpret_cast<uint4 *>(v.v) =
        *reinterpret_cast<const uint4 *>(kept + ((size_t)slot * kThreads + threadIdx.x) * 16);
    return v;
  }
  // use(vector i, i) for the thread's n vectors from `p` on, `stride` apart, the first one's slot given.
  template <int U, typename Use>
  static __device__ __forceinline__ void each(const NormArgs &a, const unsigned char *kept, int slot, const T *p,
                                              int64_t stride, int n, Use &&use) {
    int i = 0;
    if constexpr (kKeeps) {
      const int here = min(n, a.cache - slot);
      if (here > 0) {
        batches<1>(here, [&](int j) { return copied(kept, slot + j); }, use);
        i = here;
      }
    }
    batches<U>(
        n - i,
        [&](int j) {
          Vec v;
          v.load(p + (i + j) * stride);
          return v;
        },
        [&](const Vec &v, int j) { use(v, i + j); });
  }
  template <int U, typename Use>
  static __device__ __forceinline__ void each_two(const NormArgs &a, const unsigned char *kept, int slot, const T *p,
                                                  const T *d, int64_t stride, int n, Use &&use) {
    int i = 0;
    if constexpr (kKeeps) {
      const int here = min(n, a.cache - slot);
      if (here > 0) {
        batches<1>(here, [&](int j) { return Two{copied(kept, slot + j), copied(kept, a.cache + slot + j)}; }, use);
        i = here;
      }
    }
    batches<U>(
        n - i,
        [&](int j) {
          Two v;
          v.x.load(p + (i + j) * stride);
          v.d.load(d + (i + j) * stride);
          return v;
        },
        [&](const Two &v, int j) { use(v, i + j); });
  }
  // Calls f with SiLU as a constant.
  template <typename F>
  static __device__ __forceinline__ void by_silu(const NormArgs &a, F &&f) {
    if (a.silu) f(std::true_type());
    else f(std::false_type());
  }

  // use(get(i), i) for i < count, U of them in flight
  template <int U, typename Get, typename Use>
  static __device__ __forceinline__ void batches(int count, Get &&get, Use &&use) {
    int i = 0;
    if constexpr (U > 1) for (; i + U <= count; i += U) {
      decltype(get(0)) u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = get(i + j);
#pragma unroll
      for (int j = 0; j < U; ++j) use(u[j], i + j);
    }
    for (; i < count; ++i) use(get(i), i);
  }
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
  // Threads: `cols` vectors of channels (a power of two: some lanes may have
  // none) by `rows` tokens; a slab of more vectors than threads is gone through
  // by columns of `cols`.
  struct Last {
    int sc, sv, cols, rows, r0, r1, each, more;  // `each` tokens a thread, and one more for the first `more` rows
    int64_t base;  // of the slab's first channel at token 0
    int tx, ty, log;
    __device__ Last(const NormArgs &a, const Place &p) {
      sc = min(a.slab_channels, a.C - p.slab * a.slab_channels);
      sv = sc / V;
      log = a.cols_log;
      cols = 1 << log;
      rows = kThreads >> log;
      ty = threadIdx.x >> log;
      tx = threadIdx.x & (cols - 1);
      r0 = part_of(p.len, p.rank, a.split_log);
      r1 = part_of(p.len, p.rank + 1, a.split_log);
      each = (r1 - r0) >> (8 - log);  // (2^8 threads)
      more = (r1 - r0) & (rows - 1);
      base = (int64_t)p.n * a.P * a.C + (int64_t)p.slab * a.slab_channels;
    }
    // Where a warp has whole rows of a slab, their sums are joined by shuffles: one row of sums for a warp.
    __device__ bool folds() const { return log <= 5; }
    __device__ int sum_rows() const { return folds() ? kWarps : rows; }
    __device__ int sum_row(int ty) const { return folds() ? threadIdx.x >> 5 : ty; }
    __device__ bool sums_here() const { return !folds() || (int)(threadIdx.x & 31) < cols; }
    __device__ int warp_count(int warp) const {  // tokens of a warp's rows
      const int per = 32 >> log, first = warp * per;
      return per * each + min(max(more - first, 0), per);
    }
    __device__ int slots() const { return each + (more > 0); }
    __device__ int count(int ty) const { return each + (ty < more); }
  };

  // Tokens behind the row's last: zeros.
  static __device__ void clear_last(const NormArgs &a, const Place &p, const Last &l) {
    if (p.len == a.P) return;
    const float2 zero[P] = {};
    const int behind = a.P - p.len, first = p.len + part_of(behind, p.rank, a.split_log),
              last = p.len + part_of(behind, p.rank + 1, a.split_log);
    for (int64_t i = threadIdx.x; i < (int64_t)(last - first) * l.sv; i += kThreads)
      write((T *)a.out + l.base + (first + i / l.sv) * a.C + i % l.sv * V, zero);
  }

  static __device__ void forward_last(const NormArgs &a, unsigned char *kept) {
    const Place p = place_of(a);
    const Last l(a, p);
    const T *x = (const T *)a.x;
    const int groups = l.sc / a.cg, tx = l.tx, ty = l.ty;
    float *red = reinterpret_cast<float *>(kept + (size_t)a.cache * kThreads * 16);  // [rows][sc][2]
    float *mine = red + a.red;                                                        // [groups][3]
    float *all = mine + 3 * groups, *stat = all + 3 * kWarps;  // the block's parts [8][3]; [groups][2]
    // f(column, its first slot, this thread's tokens) for the thread's columns
    auto columns = [&](auto &&f) {
      int slot = 0;
      for (int c0 = 0; c0 < l.sv; c0 += l.cols, slot += l.slots()) f(c0 + tx, slot, c0 + tx < l.sv ? l.count(ty) : 0);
    };
    const int64_t stride = (int64_t)l.rows * a.C;
    auto place = [&](int col) { return l.base + col * V + (int64_t)(l.r0 + ty) * a.C; };
    if (a.phase != kApply) {
      if (a.cache) {
        columns([&](int col, int slot, int n) {
          const T *at = x + place(col);
          for (int i = 0; i < min(n, a.cache - slot); ++i) ahead(a, kept, slot + i, at + i * stride);
        });
        arrived();
      }
      columns([&](int col, int slot, int all_mine) {
        for (int run = 0; run == 0 || run < l.slots(); run += kRun) {
          const int n = min(max(all_mine - run, 0), kRun);
          float2 k[P] = {}, s[P] = {}, q[P] = {};
          each<kFlight>(a, kept, slot + run, x + place(col) + run * stride, stride, n, [&](const Vec &v, int j) {
            if (j == 0)
#pragma unroll
              for (int i = 0; i < P; ++i) k[i] = mul2(get(v, i), both(-1.f));
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 d = add2(get(v, i), k[i]);
              s[i] = add2(s[i], d);
              q[i] = fma2(d, d, q[i]);
            }
          });
          const float inv = n > 0 ? 1.f / n : 0.f;
#pragma unroll
          for (int i = 0; i < P; ++i) {  // s: the mean, q: M2
            const float2 m = mul2(s[i], both(inv));
            q[i] = fma2(s[i], mul2(m, both(-1.f)), q[i]);
            s[i] = n > 0 ? fma2(k[i], both(-1.f), m) : both(0.f);
          }
          float count = n;
          if (l.folds()) {
            for (int o = l.cols; o < 32; o <<= 1) {
              const float other = __shfl_xor_sync(0xffffffffu, count, o), sum = count + other;
              const float share = sum > 0.f ? other / sum : 0.f;
#pragma unroll
              for (int i = 0; i < P; ++i) {
                const float2 m = make_float2(__shfl_xor_sync(0xffffffffu, s[i].x, o), __shfl_xor_sync(0xffffffffu, s[i].y, o));
                const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, q[i].x, o), __shfl_xor_sync(0xffffffffu, q[i].y, o));
                const float2 d = fma2(s[i], both(-1.f), m);
                s[i] = fma2(d, both(share), s[i]);
                q[i] = add2(add2(q[i], v), mul2(mul2(d, d), both(count * share)));
              }
              count = sum;
            }
          }
          if (l.sums_here() && col < l.sv)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float *e = red + 2 * ((size_t)l.sum_row(ty) * l.sc + col * V + i);
              if (run == 0) {
                e[0] = Norm::at(s, i);
                e[1] = Norm::at(q, i);
              } else {  // (all rows of threads had the tokens of the runs before)
                const float had = (float)run * (l.folds() ? 32 >> l.log : 1), share = count / (had + count);
                const float d = Norm::at(s, i) - e[0];
                e[0] = fmaf(d, share, e[0]);
                e[1] += Norm::at(q, i) + d * d * (had * share);
              }
            }
        }
      });
      __syncthreads();
      // few groups of many sums: several warps share one's rows
      const int warp = threadIdx.x >> 5, share = l.sum_rows() * a.cg > 2048 && groups < kWarps ? kWarps / groups : 1;
      for (int i = warp; i < groups * share; i += kWarps) {
        const int g = share == 1 ? i : i / share, part = i - g * share, r0 = share == 1 ? 0 : l.sum_rows() * part / share,
                  r1 = share == 1 ? l.sum_rows() : l.sum_rows() * (part + 1) / share;
        float n, mean, m2;
        join(red, r1 - r0, a.cg, [&](int r, int c) { return 2 * ((r0 + r) * l.sc + g * a.cg + c); },
             [&](int r) { return (float)(l.folds() ? l.warp_count(r0 + r) : l.count(r0 + r)); }, n, mean, m2);
        if ((threadIdx.x & 31) == 0) {
          float *out = share == 1 ? mine + 3 * g : all + 3 * i;
          out[0] = n;
          out[1] = mean;
          out[2] = m2;
        }
      }
      if (share > 1) {
        __syncthreads();
        if (warp < groups) {
          float n, mean, m2;
          join(all + 3 * warp * share, share, 1, [](int r, int) { return 3 * r + 1; },
               [&](int r) { return all[3 * (warp * share + r)]; }, n, mean, m2);
          if ((threadIdx.x & 31) == 0) {
            mine[3 * warp] = n;
            mine[3 * warp + 1] = mean;
            mine[3 * warp + 2] = m2;
          }
        }
      }
    }
    const int first = p.slab * (a.slab_channels / a.cg);
    if (!exchange(a, mine, 3 * groups, [&](auto &&number) { finish_stats(a, p, number, stat, groups, first); })) return;
    columns([&](int col, int slot, int n) {
      if (!n) return;
      float2 mean[P] = {}, scale[P] = {}, shift[P] = {};  // (the mean's negative)
      const int ch = p.slab * a.slab_channels + col * V;
      weights(scale, a.w, ch, a.wf32, 1.f);
      weights(shift, a.b, ch, a.wf32, 0.f);
      with_groups(col * V, a.cg, [&](int i, int g) {
        Norm::at(mean, i) = -stat[2 * g];
        Norm::at(scale, i) *= stat[2 * g + 1];
      });
      T *out = (T *)a.out + place(col);
      by_silu(a, [&](auto silu) {
        each<kFlight>(a, kept, slot, x + place(col), stride, n, [&](const Vec &v, int j) {
          float2 y[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 pre = fma2(add2(get(v, i), mean[i]), scale[i], shift[i]);
            y[i] = decltype(silu)::value ? mul2(pre, sigmoid2(pre)) : pre;
          }
          write(out + j * stride, y);
        });
      });
    });
    clear_last(a, p, l);
    leave(a);
  }

  // Joins the blocks' (count, mean, M2) of each group to (mean, rstd); a thread a group.
  template <typename Number>
  static __device__ __forceinline__ void finish_stats(const NormArgs &a, const Place &p, Number &&number, float *stat,
                                                      int groups, int first) {
    for (int g = threadIdx.x; g < groups; g += kThreads) {
      float n = 0.f, s = 0.f, m2 = 0.f, off = 0.f;
#pragma unroll 4
      for (int r = 0; r < a.split; ++r) {
        n += number(r, 3 * g);
        s += number(r, 3 * g) * number(r, 3 * g + 1);
        m2 += number(r, 3 * g + 2);
      }
      const float inv = n > 0.f ? 1.f / n : 0.f;
      float mean = s * inv;
#pragma unroll 4
      for (int r = 0; r < a.split; ++r) {  // (as in join)
        const float k = number(r, 3 * g), d = k > 0.f ? number(r, 3 * g + 1) - mean : 0.f;
        off = fmaf(k, d, off);
        m2 += k * d * d;
      }
      off *= inv;
      m2 -= n * off * off;
      mean += off;
      const float rstd = n > 0.f ? 1.f / sqrtf((m2 < 0.f ? 0.f : m2) * inv + a.eps) : 0.f;
      stat[2 * g] = mean;
      stat[2 * g + 1] = rstd;
      if (p.rank == 0 && a.stats) {
        float *out = a.stats + 2 * ((size_t)p.n * a.G + first + g);
        out[0] = mean;
        out[1] = rstd;
      }
    }
  }

  static __device__ void backward_last(const NormArgs &a, unsigned char *kept) {
    const Place p = place_of(a);
    const Last l(a, p);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    const int groups = l.sc / a.cg, tx = l.tx, ty = l.ty;
    unsigned char *kept_d = kept + (size_t)a.cache * kThreads * 16;
    float *red = reinterpret_cast<float *>(kept_d + (size_t)a.cache * kThreads * 16);  // [rows][sc][2]
    float *mine = red + a.red;                                                          // [sc][2]: sums of h and of h xhat
    float *chan = mine + 2 * l.sc, *sums = chan + 2 * l.sc;  // [sc][2]; [groups][2]: means of h w and of h w xhat
    const float *stats = a.stats + 2 * ((size_t)p.n * a.G + p.slab * a.slab_channels / a.cg);
    auto columns = [&](auto &&f) {
      int slot = 0;
      for (int c0 = 0; c0 < l.sv; c0 += l.cols, slot += l.slots()) f(c0 + tx, slot, c0 + tx < l.sv ? l.count(ty) : 0);
    };
    const int64_t stride = (int64_t)l.rows * a.C;
    auto place = [&](int col) { return l.base + col * V + (int64_t)(l.r0 + ty) * a.C; };
    float2 mean[P] = {}, rstd[P] = {}, w[P] = {}, b[P] = {};  // (the mean's negative)
    auto channel = [&](int col) {
      const int ch = p.slab * a.slab_channels + col * V;
      weights(w, a.w, ch, a.wf32, 1.f);
      weights(b, a.b, ch, a.wf32, 0.f);
      with_groups(col * V, a.cg, [&](int i, int g) {
        Norm::at(mean, i) = -stats[2 * g];
        Norm::at(rstd, i) = stats[2 * g + 1];
      });
    };
    auto slope = [&](auto silu, const Two &v, int i, float2 &xhat) {
      xhat = mul2(add2(get(v.x, i), mean[i]), rstd[i]);
      const float2 h = get(v.d, i);
      if constexpr (!decltype(silu)::value) return h;
      const float2 pre = fma2(xhat, w[i], b[i]);
      return mul2(h, silu_slope(pre, sigmoid2(pre)));
    };
    if (a.phase != kApply) {
      if (a.cache)
        columns([&](int col, int slot, int n) {
          const int64_t at = place(col);
          for (int i = 0; i < min(n, a.cache - slot); ++i) {
            ahead(a, kept, slot + i, x + at + i * stride);
            ahead(a, kept_d, slot + i, dy + at + i * stride);
          }
        });
      columns([&](int col, int slot, int n) {
        if (n) channel(col);
        if (slot == 0) arrived();
        for (int run = 0; run == 0 || run < l.slots(); run += kRun) {
          float2 s[P] = {}, q[P] = {};
          by_silu(a, [&](auto silu) {
            const int64_t from = place(col) + run * stride;
            const int here = min(max(n - run, 0), kRun);
            each_two<kFlightTwo>(a, kept, slot + run, x + from, dy + from, stride, here, [&](const Two &v, int) {
#pragma unroll
              for (int i = 0; i < P; ++i) {
                float2 xhat;
                const float2 h = slope(silu, v, i, xhat);
                s[i] = add2(s[i], h);
                q[i] = fma2(h, xhat, q[i]);
              }
            });
          });
          if (l.folds())
            for (int o = l.cols; o < 32; o <<= 1)
#pragma unroll
              for (int i = 0; i < P; ++i) {
                s[i] = add2(s[i], make_float2(__shfl_xor_sync(0xffffffffu, s[i].x, o), __shfl_xor_sync(0xffffffffu, s[i].y, o)));
                q[i] = add2(q[i], make_float2(__shfl_xor_sync(0xffffffffu, q[i].x, o), __shfl_xor_sync(0xffffffffu, q[i].y, o)));
              }
          if (l.sums_here() && col < l.sv)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float *e = red + 2 * ((size_t)l.sum_row(ty) * l.sc + col * V + i);
              e[0] = run == 0 ? Norm::at(s, i) : e[0] + Norm::at(s, i);
              e[1] = run == 0 ? Norm::at(q, i) : e[1] + Norm::at(q, i);
            }
        }
      });
      __syncthreads();
      // a number's rows over up to 32 lanes
      int lanes = 1;
      const int rows = l.sum_rows();
      while (lanes < 32 && lanes * 2 <= rows && lanes * 4 * l.sc <= kThreads) lanes *= 2;
      for (int i0 = 0; i0 < 2 * l.sc; i0 += kThreads / lanes) {
        const int i = i0 + threadIdx.x / lanes;
        float s = 0.f;
        if (i < 2 * l.sc)
          for (int r = threadIdx.x % lanes; r < rows; r += lanes) s += red[(size_t)2 * r * l.sc + i];
        for (int o = lanes >> 1; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (i < 2 * l.sc && threadIdx.x % lanes == 0) mine[i] = s;
      }
    }
    if (!exchange(a, mine, 2 * l.sc, [&](auto &&number) { join_sums(a, chan, l.sc, number); })) return;
    finish_sums(a, p, sums, chan, l.sc, groups, p.slab * a.slab_channels);
    columns([&](int col, int slot, int n) {
      if (!n) return;
      channel(col);
      float2 hw[P] = {}, hx[P] = {};  // (their negatives)
      with_groups(col * V, a.cg, [&](int i, int g) {
        Norm::at(hw, i) = -sums[2 * g];
        Norm::at(hx, i) = -sums[2 * g + 1];
      });
      T *out = (T *)a.out + place(col);
      by_silu(a, [&](auto silu) {
        each_two<kFlightTwo>(a, kept, slot, x + place(col), dy + place(col), stride, n, [&](const Two &v, int j) {
          float2 o[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {  // (h w rounded as in its mean: a group of one value has no gradient)
            float2 xhat;
            const float2 h = slope(silu, v, i, xhat);
            o[i] = mul2(rstd[i], fma2(xhat, hx[i], add2(mul2_rounded(h, w[i]), hw[i])));
          }
          write(out + j * stride, o);
        });
      });
    });
    clear_last(a, p, l);
    leave(a);
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
        s += __fmul_rn(w, chan[2 * c]);
        q += __fmul_rn(w, chan[2 * c + 1]);
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
      begin = part_of(a.cg * a.segs, p.rank, a.split_log);
      end = part_of(a.cg * a.segs, p.rank + 1, a.split_log);
      base = ((int64_t)p.n * a.C + (int64_t)p.slab * a.cg) * a.P;
    }
  };

  // Calls body(row, first token, end, first slot, vectors) for this thread's
  // pieces, the tokens cut at `len`: the thread's own are every f.lanes-th vector
  // from the first token on.
  template <typename Body>
  static __device__ __forceinline__ void pieces(const NormArgs &a, const First &f, int len, Body &&body) {
    int slot = 0;
    for (int i = f.begin + f.who; i < f.end; i += f.takers) {
      const int row = i / a.segs, t0 = (i - row * a.segs) * a.seg * V, t1 = min(t0 + a.seg * V, len);
      const int left = t1 - t0 - f.lane * V, n = left > 0 ? (left - 1) / (f.lanes * V) + 1 : 0;
      body(row, t0 + f.lane * V, t1, slot, n);
      slot += n;
    }
  }

  static __device__ void clear_first(const NormArgs &a, const Place &p, const First &f) {
    if (p.len == a.P) return;
    const float2 zero[P] = {};
    pieces(a, f, a.P, [&](int row, int t, int t1, int, int) {
      T *out = (T *)a.out + f.base + (int64_t)row * a.P;
      // (a vector that the row's last token is in has been written)
      for (; t < t1; t += f.lanes * V)
        if (t >= p.len) write(out + t, zero);
    });
  }

  static __device__ void forward_first(const NormArgs &a, unsigned char *kept) {
    const Place p = place_of(a);
    const First f(a, p);
    const T *x = (const T *)a.x;
    float *red = reinterpret_cast<float *>(kept + (size_t)a.cache * kThreads * 16);
    float *mine = red + 3 * kThreads, *stat = mine + 3;
    const int step = f.lanes * V;
    if (a.phase != kApply) {
      if (a.cache) {
        pieces(a, f, p.len, [&](int row, int t0, int, int slot, int n) {
          const T *at = x + f.base + (int64_t)row * a.P + t0;
          for (int i = 0; i < n && slot + i < a.cache; ++i) ahead(a, kept, slot + i, at + i * step);
        });
        arrived();
      }
      float k = 0.f;
      float2 s2 = {}, q2 = {};
      int count = 0;
      pieces(a, f, p.len, [&](int row, int t0, int t1, int slot, int n) {
        const T *at = x + f.base + (int64_t)row * a.P + t0;
        for (int run = 0; run < n; run += kRun) {
          const int here = min(n - run, kRun);
          float2 s1 = {}, q1 = {};
          each<kFlight>(a, kept, slot + run, at + (int64_t)run * step, step, here, [&](const Vec &v, int j) {
            // all of a vector's tokens, or (at a row's last) some
            const int left = min(t1 - t0 - (run + j) * step, V);
            if (count == 0) k = v.f(0);
            count += left;
#pragma unroll
            for (int i = 0; i < P; ++i) {
              float2 d = add2(get(v, i), both(-k));
              if (left < V || V == 1) d = make_float2(2 * i < left ? d.x : 0.f, 2 * i + 1 < left ? d.y : 0.f);
              s1 = add2(s1, d);
              q1 = fma2(d, d, q1);
            }
          });
          s2 = add2(s2, s1);
          q2 = add2(q2, q1);
        }
      });
      const float s = s2.x + s2.y, q = q2.x + q2.y, m = count ? s / count : 0.f;
      float *e = red + 3 * threadIdx.x;
      e[0] = (float)count;
      e[1] = count ? k + m : 0.f;
      e[2] = q - s * m;
      __syncthreads();
      if (threadIdx.x < 32) {
        float total, mean, m2;
        join(red, kThreads, 1, [](int r, int) { return 3 * r + 1; }, [&](int r) { return red[3 * r]; }, total, mean, m2);
        if (threadIdx.x == 0) {
          mine[0] = total;
          mine[1] = mean;
          mine[2] = m2;
        }
      }
    }
    if (!exchange(a, mine, 3, [&](auto &&number) { finish_stats(a, p, number, stat, 1, p.slab); })) return;
    const float2 mean = both(-stat[0]);
    const float rstd = stat[1];
    pieces(a, f, p.len, [&](int row, int t0, int t1, int slot, int n) {
      const int64_t at = f.base + (int64_t)row * a.P + t0;
      const int ch = p.slab * a.cg + row;
      const float2 scale = both(rstd * load_w<T>(a.w, ch, a.wf32, 1.f)), shift = both(load_w<T>(a.b, ch, a.wf32, 0.f));
      by_silu(a, [&](auto silu) {
        each<kFlight>(a, kept, slot, x + at, step, n, [&](const Vec &v, int j) {
          const int left = t1 - t0 - j * step;
          float2 y[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 pre = fma2(add2(get(v, i), mean), scale, shift);
            y[i] = decltype(silu)::value ? mul2(pre, sigmoid2(pre)) : pre;
            if (left < V) y[i] = make_float2(2 * i < left ? y[i].x : 0.f, 2 * i + 1 < left ? y[i].y : 0.f);
          }
          write((T *)a.out + at + j * step, y);
        });
      });
    });
    clear_first(a, p, f);
    leave(a);
  }

  static __device__ void backward_first(const NormArgs &a, unsigned char *kept) {
    const Place p = place_of(a);
    const First f(a, p);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    unsigned char *kept_d = kept + (size_t)a.cache * kThreads * 16;
    const int most = (int)(((int64_t)a.cg * a.segs + a.split - 1) / a.split) + 1;  // pieces of a block
    float *red = reinterpret_cast<float *>(kept_d + (size_t)a.cache * kThreads * 16);  // [pieces][2]
    float *mine = red + (size_t)2 * most;                                               // [cg][2]
    float *chan = mine + 2 * a.cg, *sums = chan + 2 * a.cg;
    const float *stats = a.stats + 2 * ((size_t)p.n * a.G + p.slab);
    const float2 mean = both(-stats[0]), rstd = both(stats[1]);
    const int step = f.lanes * V;
    constexpr bool kReuse = kKeeps && sizeof(T) == 4;
    float2 w = {}, b = {};
    auto slope = [&](auto silu, const Two &v, int i, float2 &xhat) {
      xhat = mul2(add2(get(v.x, i), mean), rstd);
      const float2 h = get(v.d, i);
      if constexpr (!decltype(silu)::value) return h;
      const float2 pre = fma2(xhat, w, b);
      return mul2(h, silu_slope(pre, sigmoid2(pre)));
    };
    // pair i of a vector that has `left` tokens, with zeros behind them
    auto held = [&](float2 v, int i, int left) {
      left = min(left, V);
      return left == V && V > 1 ? v : make_float2(2 * i < left ? v.x : 0.f, 2 * i + 1 < left ? v.y : 0.f);
    };
    auto channel = [&](int row) {
      w = both(load_w<T>(a.w, p.slab * a.cg + row, a.wf32, 1.f));
      b = both(load_w<T>(a.b, p.slab * a.cg + row, a.wf32, 0.f));
    };
    if (a.phase != kApply) {
      if (a.cache) {
        pieces(a, f, p.len, [&](int row, int t0, int, int slot, int n) {
          const int64_t at = f.base + (int64_t)row * a.P + t0;
          for (int i = 0; i < n && slot + i < a.cache; ++i) {
            ahead(a, kept, slot + i, x + at + i * step);
            ahead(a, kept_d, slot + i, dy + at + i * step);
          }
        });
        arrived();
      }
      // (all lanes of a warp go through the same number of pieces)
      int slot = 0;
      for (int i0 = f.begin; i0 < f.end; i0 += f.takers) {
        const int i = i0 + f.who;
        float2 s2 = {}, q2 = {};
        if (i < f.end) {
          const int row = i / a.segs, start = (i - row * a.segs) * a.seg * V, t1 = min(start + a.seg * V, p.len);
          const int t0 = start + f.lane * V, n = t1 > t0 ? (t1 - t0 - 1) / step + 1 : 0;
          channel(row);
          const int64_t at = f.base + (int64_t)row * a.P + t0;
          by_silu(a, [&](auto silu) {
            for (int run = 0; run < n; run += kRun) {
              const int64_t from = at + (int64_t)run * step;
              const int here = min(n - run, kRun);
              float2 s1 = {}, q1 = {};
              each_two<kFlightTwo>(a, kept, slot + run, x + from, dy + from, step, here, [&](const Two &v, int j) {
                float2 h[P];
#pragma unroll
                for (int e = 0; e < P; ++e) {
                  float2 xhat;
                  h[e] = held(slope(silu, v, e, xhat), e, t1 - t0 - (run + j) * step);
                  s1 = add2(s1, h[e]);
                  q1 = add2(q1, held(mul2(h[e], xhat), e, t1 - t0 - (run + j) * step));
                }
                // (in 32 bits, what the second pass needs of dy is kept in its place)
                if (kReuse && slot + run + j < a.cache)
                  write(reinterpret_cast<T *>(kept_d + ((size_t)(slot + run + j) * kThreads + threadIdx.x) * 16), h);
              });
              s2 = add2(s2, s1);
              q2 = add2(q2, q1);
            }
          });
          slot += n;
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
    const float2 hw = both(-sums[0]), hx = both(-sums[1]);
    pieces(a, f, p.len, [&](int row, int t0, int t1, int slot, int n) {
      channel(row);
      const int64_t at = f.base + (int64_t)row * a.P + t0;
      auto last_pass = [&](auto silu, int slot, int64_t at, int t0, int n) {
        each_two<kFlightTwo>(a, kept, slot, x + at, dy + at, step, n, [&](const Two &v, int j) {
          float2 o[P];
#pragma unroll
          for (int e = 0; e < P; ++e) {
            float2 xhat;
            const float2 h = slope(silu, v, e, xhat);
            o[e] = held(mul2(rstd, fma2(xhat, hx, add2(mul2_rounded(h, w), hw))), e, t1 - t0 - j * step);
          }
          write((T *)a.out + at + j * step, o);
        });
      };
      const int here = kReuse ? min(n, max(0, a.cache - slot)) : 0;  // dy's places hold h
      if (here) last_pass(std::false_type(), slot, at, t0, here);
      if (here < n)
        by_silu(a, [&](auto silu) { last_pass(silu, slot + here, at + here * step, t0 + here * step, n - here); });
    });
    clear_first(a, p, f);
    leave(a);
  }
};

template <typename T, int V, bool kLast, bool kBackward>
__global__ void __launch_bounds__(kThreads, kBackward && sizeof(T) == 2 ? 2 : 3) norm_kernel(const NormArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
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
  int V, slab_channels, slabs, split, seg, segs, cache, red, cols_log;
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
    // whole groups, whole vectors and 64 bytes of a token where the channels allow it (with 128 a block's share of
    // 16 maps of 512x64x64 bf16 has no room in shared memory)
    while (p.slab_channels < C && (p.slab_channels % v || p.slab_channels * size < 64)) p.slab_channels += cg;
    if (p.slab_channels <= kMaxChannels) break;
  }
  p.slabs = ceil_div(C, p.slab_channels);
  const int64_t units = (int64_t)batch * p.slabs, elements = (int64_t)p.slab_channels * P;
  // A block of 256 threads wants a few vectors a thread (with 4, 8 or 16 instead of 2 at least a small call of
  // 2x320x17x31 float16 took 12.6 us instead of 10.5); the GPU wants some blocks for each SM (16x512x64x64 bfloat16,
  // both passes: at least 2 an SM 197 us, 4 149, 8 164).
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
  if (last) {
    // (as Last::sum_rows(): a row of sums for a warp, or for each row of threads)
    while (p.cols_log < 8 && 1 << p.cols_log < sc / p.V) ++p.cols_log;
    red = 2 * (size_t)sc * (p.cols_log <= 5 ? kWarps : kThreads >> p.cols_log);
    p.red = (int)red;
  }
  else if (backward) red = 2 * ((size_t)ceil_div((int64_t)cg * p.segs, p.split) + 1);
  else red = 3 * kThreads;
  // what a block keeps: as many of its vectors as there is room for
  const int arrays = backward ? 2 : 1;
  const size_t sums = 4 * (red + p.numbers * (backward ? 2 : 1) + 2 * (size_t)groups + 3 * kWarps);
  const size_t space = std::min<size_t>(kCacheBytes, 224 * 1024 - sums);
  const int room = (int)(space / (kThreads * 16 * arrays));
  int64_t need;
  if (last) {
    need = (int64_t)ceil_div(ceil_div(P, p.split), kThreads >> p.cols_log) * ceil_div(sc / p.V, 1 << p.cols_log);
  } else {
    int lanes = 32;
    while (lanes > 1 && lanes / 2 >= p.seg) lanes >>= 1;
    need = (int64_t)ceil_div(ceil_div((int64_t)cg * p.segs, p.split), kThreads / lanes) * ceil_div(p.seg, lanes);
  }
  p.cache = p.fused && p.V == widest ? (int)std::min<int64_t>(need, room) : 0;
  p.smem = (size_t)p.cache * arrays * kThreads * 16 + sums;
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
  a.split_log = 31 - __builtin_clz(p.split);
  a.cols_log = p.cols_log;
  a.seg = p.seg;
  a.cache = p.cache;
  a.red = p.red;
  a.segs = p.segs;
  a.numbers = (int)p.numbers;
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
  a.split_log = 31 - __builtin_clz(p.split);
  a.cols_log = p.cols_log;
  a.seg = p.seg;
  a.cache = p.cache;
  a.red = p.red;
  a.segs = p.segs;
  a.numbers = (int)p.numbers;
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
