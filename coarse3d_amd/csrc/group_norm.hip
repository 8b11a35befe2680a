// GroupNorm with an activation over channels-last images, forward and backward (gfx950; HBM-bound).
//
// For sample n and group g (D = C / G channels, HW pixels, M = HW * D values):
//     xhat = (x - mean) * rstd,  z = xhat * gamma[c] + beta[c],  y = act(z)
// and, with dz = dy * act'(z), t = dz * gamma:
//     dbeta = sum dz,  dgamma = sum dz * xhat  (over samples and pixels),  dx = rstd * (t - mean(t) - xhat * mean(t * xhat)).
//
// A thread owns V consecutive channels (16 bytes where alignment allows) and walks pixels, so that every load is a whole vector of
// a pixel's row whatever D is.  Two forms:
//   small: one workgroup holds all values of a (sample, group) in registers -- one launch, one read, no workspace;
//   large: a pass for the statistics, a pass that applies them.  The second walks the tensor backwards, so that it begins with what
//          the first has left in the caches, and its workgroups fold the partial statistics of their sample by themselves.
// One pass over x would need all workgroups of a sample to wait for one another; two passes cost a second read, most of it from the
// infinity cache.  8x64x2048x32 fp32 forward: 26 us (5.1 TB/s) + 40 us (6.7 TB/s, read and written); 2x32x1024x704 bf16: forward 21 + 5 + 34,
// backward 36 + 5 + 46.  A (sample, group) of 4096 bf16 values: 4 us, of 16384 fp32 ones 6 forward and 9 backward, latency all of it.
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include "common.h"
#include "../../include/coarse3d_hip.h"

namespace {

enum { ACT_NONE = 0, ACT_LRELU = 1, ACT_SILU = 2 };

template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ void ldv(const T* p, float (&r)[V]) {
  const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int q = 0; q < V; ++q) r[q] = (float)t.v[q];
}
// NT: past the caches
template <class T, int V, bool NT = false>
__device__ __forceinline__ void stv(T* p, const float (&r)[V]) {
  Vec<T, V> t;
#pragma unroll
  for (int q = 0; q < V; ++q) t.v[q] = (T)r[q];
  if constexpr (NT && sizeof(t) == 16) {
    typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, t), reinterpret_cast<u32x4_t*>(p));
    return;
  }
  *reinterpret_cast<Vec<T, V>*>(p) = t;
}

// 1 / (1 + e^-z) from the hardware's exp2 and reciprocal: off by a few units in the last place, and by |z| of them for z far below
// zero, where the result itself vanishes
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
template <int ACT>
__device__ __forceinline__ float act_fwd(float z, float slope) {
  if (ACT == ACT_LRELU) return z > 0.f ? z : z * slope;
  if (ACT == ACT_SILU) return z * sigmoid(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_bwd(float z, float slope) {
  if (ACT == ACT_LRELU) return z > 0.f ? 1.f : slope;
  if (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

struct Img {
  int64_t ns, ps;           // elements from sample to sample and from pixel to pixel
};

// ---------------------------------------------------------------- small: a (sample, group) in one workgroup

template <int V>
constexpr int kSmallThreads = V == 8 ? 512 : 1024;
template <int V>
constexpr int kSmallVecs = V == 8 ? 4 : 16 / V;        // vectors a thread holds
// thread t: vector t % dv of the group's D / V, pixels t / dv + r * pl

// K sums over the workgroup, the same bits in every thread; red: K times 16 floats that the last sums did not use
template <int K>
__device__ __forceinline__ void block_sums(float (&v)[K], float* red) {
#define C3D_SUM_STEP(ctrl, rows) v[k] += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v[k]), ctrl, rows, 0xf, false))
#pragma unroll
  for (int k = 0; k < K; ++k) {
    C3D_SUM_STEP(0x111, 0xf);    // row_shr:1, 2, 4, 8: lane 15 of a row of sixteen has the row's
    C3D_SUM_STEP(0x112, 0xf);
    C3D_SUM_STEP(0x114, 0xf);
    C3D_SUM_STEP(0x118, 0xf);
    C3D_SUM_STEP(0x142, 0xa);    // row_bcast:15 into rows 1 and 3, row_bcast:31 into 2 and 3: lane 63 has all
    C3D_SUM_STEP(0x143, 0xc);
  }
#undef C3D_SUM_STEP
  const int nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 63)
#pragma unroll
    for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int i = 0; i < nw; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += red[i * K + k];
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads<V>) void gn_small_kernel(const T* __restrict__ x, Img xi, int HW, int C, int G, int dv, int pl,
                                                                  const float* __restrict__ gamma, const float* __restrict__ beta, float eps,
                                                                  float slope, T* __restrict__ y, float* __restrict__ mean,
                                                                  float* __restrict__ rstd) {
  constexpr int R = kSmallVecs<V>;
  __shared__ float red[48];
  const int n = blockIdx.x / G, g = blockIdx.x % G, l = threadIdx.x / dv, c = g * (C / G) + (threadIdx.x % dv) * V;
  const T* xs = x + n * xi.ns + c;
  Vec<T, V> raw[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l < pl && l + r * pl < HW) raw[r] = *reinterpret_cast<const Vec<T, V>*>(xs + (int64_t)(l + r * pl) * xi.ps);
  float ga[V], be[V];                                    // (c is a channel of the group for idle threads too)
#pragma unroll
  for (int e = 0; e < V; ++e) {
    ga[e] = gamma ? gamma[c + e] : 1.f;
    be[e] = beta ? beta[c + e] : 0.f;
  }
  const float count = (float)HW * (float)(C / G);
  float first[1] = {0.f};
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l < pl && l + r * pl < HW)
#pragma unroll
      for (int e = 0; e < V; ++e) first[0] += (float)raw[r].v[e];
  block_sums(first, red);
  // about this mean, off by the rounding of its sum: what is left of the mean (a sum of small numbers) and the variance
  const float mu = first[0] / count;
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l < pl && l + r * pl < HW)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (float)raw[r].v[e] - mu;
        s[0] += d;
        s[1] = fmaf(d, d, s[1]);
      }
  block_sums(s, red + 16);
  const float left = s[0] / count, var = s[1] / count - left * left, rs = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps), off = -left * rs;
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = mu + left;
    rstd[blockIdx.x] = rs;
  }
  if (l >= pl) return;
  T* ys = y + (int64_t)n * HW * C + c;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l + r * pl < HW) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = act_fwd<ACT>(fmaf(fmaf((float)raw[r].v[e] - mu, rs, off), ga[e], be[e]), slope);
      stv<T, V>(ys + (int64_t)(l + r * pl) * C, o);
    }
}

// chan: [N][C] pairs (sum dz, sum dz xhat) of a sample, or with N == 1 straight into dbeta, dgamma
template <class T, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads<V>) void gn_small_bwd_kernel(const T* __restrict__ dy, Img di, const T* __restrict__ x, Img xi, int HW, int C,
                                                                      int G, int dv, int pl, const float* __restrict__ mean,
                                                                      const float* __restrict__ rstd, const float* __restrict__ gamma,
                                                                      const float* __restrict__ beta, float slope, T* __restrict__ dx, int wanted,
                                                                      float2* __restrict__ chan, float* __restrict__ dgamma,
                                                                      float* __restrict__ dbeta) {
  constexpr int R = kSmallVecs<V>;
  extern __shared__ float2 rows[];                       // [pl][D], then [pl / 8][D]
  __shared__ float red[32];                              // 16 waves, two sums
  const int n = blockIdx.x / G, g = blockIdx.x % G, D = C / G, l = threadIdx.x / dv, q = threadIdx.x % dv, c = g * D + q * V;
  const T* xs = x + n * xi.ns + c;
  const T* ds = dy + n * di.ns + c;
  Vec<T, V> xr[R], dr[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l < pl && l + r * pl < HW) {
      xr[r] = *reinterpret_cast<const Vec<T, V>*>(xs + (int64_t)(l + r * pl) * xi.ps);
      dr[r] = *reinterpret_cast<const Vec<T, V>*>(ds + (int64_t)(l + r * pl) * di.ps);
    }
  const float mu = mean[blockIdx.x], rs = rstd[blockIdx.x];
  float ga[V], be[V], a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    ga[e] = l < pl && gamma ? gamma[c + e] : 1.f;
    be[e] = l < pl && beta ? beta[c + e] : 0.f;
    a[e] = b[e] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (l < pl && l + r * pl < HW)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = ((float)xr[r].v[e] - mu) * rs;
        const float dz = (float)dr[r].v[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope);
        a[e] += dz;
        b[e] = fmaf(dz, xh, b[e]);
      }
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s[0] = fmaf(a[e], ga[e], s[0]);
    s[1] = fmaf(b[e], ga[e], s[1]);
  }
  block_sums(s, red);
  const float count = (float)HW * (float)D, c1 = s[0] / count, c2 = s[1] / count;
  if (l < pl) {
    T* os = dx + (int64_t)n * HW * C + c;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (l + r * pl < HW) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = ((float)xr[r].v[e] - mu) * rs;
          const float t = (float)dr[r].v[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope) * ga[e];
          o[e] = rs * (t - c1 - xh * c2);
        }
        stv<T, V>(os + (int64_t)(l + r * pl) * C, o);
      }
  }
  if (!wanted) return;
  // the channels' sums: eight rows to one until one is left
  if (l < pl)
#pragma unroll
    for (int e = 0; e < V; ++e) rows[l * D + q * V + e] = make_float2(a[e], b[e]);
  float2* from = rows;
  float2* to = rows + pl * D;
  for (int k = pl; k > 1; k = (k + 7) / 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < (k + 7) / 8 * D; i += blockDim.x) {
      const int row = i / D, ch = i % D;
      float2 v = make_float2(0.f, 0.f);
      for (int j = row * 8; j < row * 8 + 8 && j < k; ++j) {
        v.x += from[j * D + ch].x;
        v.y += from[j * D + ch].y;
      }
      to[i] = v;
    }
    float2* t = from;
    from = to;
    to = t;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += blockDim.x) {
    if (gridDim.x == (unsigned)G) {
      if (dbeta) dbeta[g * D + i] = from[i].x;
      if (dgamma) dgamma[g * D + i] = from[i].y;
    } else {
      chan[(int64_t)n * C + g * D + i] = from[i];
    }
  }
}

// ---------------------------------------------------------------- large: two passes

// How an image is cut.  A tile of channels is `gpt` whole groups (split == 1), or one of `split` parts of a group too wide for a
// workgroup; qt vectors wide, `pl` pixels side by side.  A sample's pixels are cut into runs of DEEP * pl, and of nb workgroups the
// b-th takes runs b, b + nb, ...: at any time the workgroups read one window of memory together, and the second pass, which begins
// with the last runs, finds the latest of it in the caches (8x64x2048x32 fp32: with a chunk of its own each, both passes take 5 % longer).
struct Plan {
  int D, qt, pl, threads, tiles, gpt, split, nb;
  int64_t each;             // every workgroup takes this many runs, and the first `more` one more
  int more;
  int run, last, missing;   // pixels of a run; the workgroup that has the last one, and how many pixels that one lacks
};
__device__ __forceinline__ int64_t runs_of(const Plan& p, int b) { return p.each + (b < p.more ? 1 : 0); }
__device__ __forceinline__ int64_t pixels_of(const Plan& p, int b) { return runs_of(p, b) * p.run - (b == p.last ? p.missing : 0); }
struct Tile {
  int c0, nq, g0, ng, part;      // first channel, vectors, first group, groups, part of the group
};
template <int V>
__device__ __forceinline__ Tile tile_of(const Plan& p, int t, int G) {
  Tile r;
  if (p.split == 1) {
    r.g0 = t * p.gpt;
    r.ng = min(p.gpt, G - r.g0);
    r.c0 = r.g0 * p.D;
    r.nq = r.ng * p.D / V;
    r.part = 0;
  } else {
    r.g0 = t / p.split;
    r.ng = 1;
    r.part = t % p.split;
    r.c0 = r.g0 * p.D + r.part * p.qt * V;
    r.nq = min(p.qt, p.D / V - r.part * p.qt);
  }
  return r;
}
// the second pass begins where the first ended, workgroup by workgroup on the same XCD (block b runs on XCD b % 8)
__device__ __forceinline__ int backwards(int b, int n) {
  const int whole = n & ~7;
  return b < whole ? whole - 8 - (b & ~7) + (b & 7) : b;
}

// sums of a pair over `lanes` (a power of two) neighbouring lanes, in 64 bits
__device__ __forceinline__ void sum_lanes(double& a, double& b, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
}
// Lanes that work on a group together, such that all of a tile's groups are worked on at once where the workgroup has the threads;
// `body(group, lane)` is called by whole waves, with groups past the last too
template <class F>
__device__ __forceinline__ void for_groups(int ng, F body) {
  int lanes = 64;
  while (lanes > 16 && ng * lanes > (int)blockDim.x) lanes >>= 1;
  const int per = 64 / lanes;
  for (int g = threadIdx.x / lanes; g < (ng + per - 1) / per * per; g += blockDim.x / lanes) body(g, (int)(threadIdx.x & (lanes - 1)), lanes);
}

// Partial results: [N][G][nb][split] pairs, part_at() the first of a chunk
__device__ __forceinline__ int64_t part_at(const Plan& p, int G, int n, int g) { return ((int64_t)n * G + g) * p.nb * p.split; }

// A thread's pixels of its workgroup's runs, all loads of a run in flight together; BACK: from the last run to the first.  (Fetching the
// next run ahead as well costs the registers of a wave and loses 1-7 %.)
template <bool BACK, int DEEP, class F>
struct Walk {
  using R = std::invoke_result_t<F, int64_t>;
  const Plan& p;
  int64_t HW;
  int b, l;
  F load;
  R ahead[DEEP];
  // first pixel of the k-th run in the walk's order
  __device__ __forceinline__ int64_t at(int64_t k) const { return ((BACK ? runs_of(p, b) - 1 - k : k) * p.nb + b) * p.run + l; }
  __device__ __forceinline__ void fetch(int64_t i) {
    if (i + (DEEP - 1) * p.pl < HW) {
#pragma unroll
      for (int u = 0; u < DEEP; ++u) ahead[u] = load(i + u * p.pl);
    } else {
#pragma unroll
      for (int u = 0; u < DEEP; ++u)
        if (i + u * p.pl < HW) ahead[u] = load(i + u * p.pl);
    }
  }
  // issues the first run's loads: what else has to be waited for ahead of `each` is waited for together with them
  __device__ __forceinline__ void begin() { fetch(at(0)); }
  template <class H>
  __device__ __forceinline__ void each(H use) {
    const int64_t runs = runs_of(p, b);
    for (int64_t k = 0; k < runs; ++k) {
      const int64_t i = at(k);
      if (k) fetch(i);
      if (i + (DEEP - 1) * p.pl < HW) {
#pragma unroll
        for (int u = 0; u < DEEP; ++u) use(i + u * p.pl, ahead[u]);
      } else {
#pragma unroll
        for (int u = 0; u < DEEP; ++u)
          if (i + u * p.pl < HW) use(i + u * p.pl, ahead[u]);
      }
    }
  }
};
template <bool BACK, int DEEP, class F>
__device__ __forceinline__ Walk<BACK, DEEP, F> walk(const Plan& p, int64_t HW, int b, int l, F load) {
  return {p, HW, b, l, load};
}

// sums of s1, s2 [V] over the workgroup's `pl` pixel lanes: -> shared sum[ch] of the tile's channels
template <int V>
__device__ __forceinline__ void join_lanes(const Plan& p, const Tile& t, bool on, int l, int q, const float (&s1)[V], const float (&s2)[V], float2* sum) {
  const int W = p.qt * V, wt = t.nq * V;
  if (on)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[l * W + q * V + e] = make_float2(s1[e], s2[e]);
  // halves onto halves: a few barriers instead of one thread's walk over all lanes
  for (int k = p.pl; k > 1;) {
    const int h = (k + 1) / 2;
    __syncthreads();
    for (int i = threadIdx.x; i < (k - h) * W; i += blockDim.x) {
      if (i % W < wt) {
        const float2 o = sum[h * W + i];
        sum[i].x += o.x;
        sum[i].y += o.y;
      }
    }
    k = h;
  }
  __syncthreads();
}

// First pass: mean and sum of squared deviations of every group over the workgroup's pixels.  Values are shifted by its first pixel, so that a mean
// far from zero costs nothing.
template <class T, int V, int DEEP>
__global__ __launch_bounds__(512) void gn_stats_kernel(const T* __restrict__ x, Img xi, Plan p, int64_t HW, int G, float2* __restrict__ part) {
  extern __shared__ float2 sum[];
  const Tile t = tile_of<V>(p, blockIdx.x % p.tiles, G);
  const int b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = threadIdx.x % p.qt;
  const bool on = l < p.pl && q < t.nq;
  float shift[V], s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) shift[e] = s1[e] = s2[e] = 0.f;
  if (on) {
    const T* xs = x + n * xi.ns + t.c0 + q * V;
    auto w = walk<false, DEEP>(p, HW, b, l, [&](int64_t i) { return *reinterpret_cast<const Vec<T, V>*>(xs + i * xi.ps); });
    w.begin();
    ldv<T, V>(xs + (int64_t)b * p.run * xi.ps, shift);
    w.each([&](int64_t, const Vec<T, V>& r) {
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float d = (float)r.v[e] - shift[e];
                s1[e] += d;
                s2[e] = fmaf(d, d, s2[e]);
              }
            });
  }
  join_lanes<V>(p, t, on, l, q, s1, s2, sum);
  const double cnt = (double)pixels_of(p, b);
  float2* shifts = sum + p.qt * V;                        // (row 1: free again)
  if (on && l == 0)
#pragma unroll
    for (int e = 0; e < V; ++e) shifts[q * V + e].x = shift[e];
  __syncthreads();
  const int chans = p.split == 1 ? p.D : t.nq * V;
  for_groups(t.ng, [&](int g, int lane, int lanes) {
    double m = 0.0, m2 = 0.0;
    if (g < t.ng)
      for (int k = lane; k < chans; k += lanes) {
        const float2 v = sum[g * p.D + k];
        const double d = (double)v.x / cnt, mu = (double)shifts[g * p.D + k].x + d;
        m += mu;
        m2 += ((double)v.y - (double)v.x * d) + cnt * mu * mu;
      }
    sum_lanes(m, m2, lanes);
    if (g < t.ng && lane == 0) {
      const double mu = m / chans;
      part[part_at(p, G, n, t.g0 + g) + b * p.split + t.part] = make_float2((float)mu, (float)fmax(m2 - cnt * chans * mu * mu, 0.0));
    }
  });
}

// mean and rstd of (n, g) from its partial results, by `lanes` lanes; every lane gets them
__device__ __forceinline__ float2 fold_stats(const float2* __restrict__ part, const Plan& p, int V, int64_t HW, int G, int n, int g, float eps, int lane,
                                             int lanes) {
  const float2* a = part + part_at(p, G, n, g);
  double s = 0.0, s2 = 0.0;
#pragma unroll 4
  for (int i = lane; i < p.nb * p.split; i += lanes) {
    const int b = p.split == 1 ? i : i / p.split, k = i - b * p.split;
    const double cnt = (double)pixels_of(p, b) * (p.split == 1 ? p.D : min(p.qt * V, p.D - k * p.qt * V));
    const float2 v = a[i];
    s += cnt * v.x;
    s2 += (double)v.y + cnt * ((double)v.x * v.x);
  }
  sum_lanes(s, s2, lanes);
  const double M = (double)HW * p.D, mu = s / M, var = s2 / M - mu * mu;
  return make_float2((float)mu, (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)eps)));
}

// a wave each, for tiles of many groups
template <int V>
__global__ __launch_bounds__(64) void gn_fold_kernel(const float2* __restrict__ part, Plan p, int64_t HW, int G, float eps, float* __restrict__ mean,
                                                    float* __restrict__ rstd) {
  const float2 r = fold_stats(part, p, V, HW, G, blockIdx.x / G, blockIdx.x % G, eps, threadIdx.x, 64);
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = r.x;
    rstd[blockIdx.x] = r.y;
  }
}

// Second pass.  part != NULL: the statistics are still in pieces; every workgroup folds those of its groups
template <class T, int V, int ACT, bool NT, int DEEP>
__global__ __launch_bounds__(512) void gn_apply_kernel(const T* __restrict__ x, Img xi, Plan p, int64_t HW, int C, int G, const float2* __restrict__ part,
                                                      float eps, float* __restrict__ mean, float* __restrict__ rstd,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta, float slope,
                                                      T* __restrict__ y) {
  extern __shared__ float2 stat[];                       // [gpt]
  const int block = backwards(blockIdx.x, gridDim.x);
  const Tile t = tile_of<V>(p, block % p.tiles, G);
  const int b = (block / p.tiles) % p.nb, n = block / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = threadIdx.x % p.qt;
  const bool on = l < p.pl && q < t.nq;
  const T* xs = x + n * xi.ns + t.c0 + q * V;
  T* ys = y + (int64_t)n * HW * C + t.c0 + q * V;
  auto w = walk<true, DEEP>(p, HW, b, l, [&](int64_t i) { return *reinterpret_cast<const Vec<T, V>*>(xs + i * xi.ps); });
  if (on) w.begin();
  for_groups(t.ng, [&](int g, int lane, int lanes) {
    const int k = n * G + t.g0 + min(g, t.ng - 1);
    const float2 r = part ? fold_stats(part, p, V, HW, G, n, k - n * G, eps, lane, lanes) : make_float2(mean[k], rstd[k]);
    if (g < t.ng && lane == 0) {
      stat[g] = r;
      if (part && b == 0 && t.part == 0) {
        mean[k] = r.x;
        rstd[k] = r.y;
      }
    }
  });
  __syncthreads();
  if (!on) return;
  float mu[V], rs[V], ga[V], be[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = t.c0 + q * V + e;
    const float2 v = stat[p.split == 1 ? (q * V + e) / p.D : 0];
    mu[e] = v.x;
    rs[e] = v.y;
    ga[e] = gamma ? gamma[c] : 1.f;
    be[e] = beta ? beta[c] : 0.f;
  }
  w.each([&](int64_t i, const Vec<T, V>& r) {
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = act_fwd<ACT>(fmaf(((float)r.v[e] - mu[e]) * rs[e], ga[e], be[e]), slope);
    stv<T, V, NT>(ys + i * C, o);
  });
}

template <class T, int V>
struct Two {
  Vec<T, V> x, d;
};

// Backward, first pass: per chunk and group (sum t, sum t xhat) -> part, and per channel (sum dz, sum dz xhat) -> chan [N][nb][C]
template <class T, int V, int ACT, int DEEP>
__global__ __launch_bounds__(512) void gn_bwd_stats_kernel(const T* __restrict__ dy, Img di, const T* __restrict__ x, Img xi, Plan p, int64_t HW, int C,
                                                          int G, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta, float slope,
                                                          float2* __restrict__ part, float2* __restrict__ chan) {
  extern __shared__ float2 sum[];
  const Tile t = tile_of<V>(p, blockIdx.x % p.tiles, G);
  const int b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = threadIdx.x % p.qt;
  const bool on = l < p.pl && q < t.nq;
  float s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
  if (on) {
    const T* xs = x + n * xi.ns + t.c0 + q * V;
    const T* ds = dy + n * di.ns + t.c0 + q * V;
    auto w = walk<false, DEEP>(p, HW, b, l, [&](int64_t i) {
      return Two<T, V>{*reinterpret_cast<const Vec<T, V>*>(xs + i * xi.ps), *reinterpret_cast<const Vec<T, V>*>(ds + i * di.ps)};
    });
    w.begin();
    float mu[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = t.c0 + q * V + e, k = n * G + t.g0 + (p.split == 1 ? (q * V + e) / p.D : 0);
      mu[e] = mean[k];
      rs[e] = rstd[k];
      ga[e] = gamma ? gamma[c] : 1.f;
      be[e] = beta ? beta[c] : 0.f;
    }
    w.each([&](int64_t, const Two<T, V>& r) {
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float xh = ((float)r.x.v[e] - mu[e]) * rs[e];
                const float dz = (float)r.d.v[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope);
                s1[e] += dz;
                s2[e] = fmaf(dz, xh, s2[e]);
              }
            });
  }
  join_lanes<V>(p, t, on, l, q, s1, s2, sum);
  if (chan)
    for (int i = threadIdx.x; i < t.nq * V; i += blockDim.x) chan[((int64_t)n * p.nb + b) * C + t.c0 + i] = sum[i];
  const int chans = p.split == 1 ? p.D : t.nq * V;
  for_groups(t.ng, [&](int g, int lane, int lanes) {
    double a = 0.0, c = 0.0;
    if (g < t.ng)
      for (int k = lane; k < chans; k += lanes) {
        const float2 v = sum[g * p.D + k];
        const double ga = gamma ? (double)gamma[t.c0 + g * p.D + k] : 1.0;
        a += ga * v.x;
        c += ga * v.y;
      }
    sum_lanes(a, c, lanes);
    if (g < t.ng && lane == 0) part[part_at(p, G, n, t.g0 + g) + b * p.split + t.part] = make_float2((float)a, (float)c);
  });
}

// the means of t and t xhat over (n, g), by `lanes` lanes
__device__ __forceinline__ float2 fold_means(const float2* __restrict__ part, const Plan& p, int64_t HW, int G, int n, int g, int lane, int lanes) {
  const float2* a = part + part_at(p, G, n, g);
  double s = 0.0, s2 = 0.0;
#pragma unroll 4
  for (int i = lane; i < p.nb * p.split; i += lanes) {
    s += (double)a[i].x;
    s2 += (double)a[i].y;
  }
  sum_lanes(s, s2, lanes);
  const double M = (double)HW * p.D;
  return make_float2((float)(s / M), (float)(s2 / M));
}
__global__ __launch_bounds__(64) void gn_bwd_fold_kernel(const float2* __restrict__ part, Plan p, int64_t HW, int G, float2* __restrict__ coef) {
  const float2 r = fold_means(part, p, HW, G, blockIdx.x / G, blockIdx.x % G, threadIdx.x, 64);
  if (threadIdx.x == 0) coef[blockIdx.x] = r;
}

// dgamma, dbeta of 8 channels: the rows of chan [rows][C], in 64 bits and a fixed order.  Latency is all of it, and where the second pass
// is short these workgroups are its end: many lanes a channel and many loads in flight (8x32x1024x64 fp32, both calls: 94 -> 92 us from 16
// channels and 4 loads)
constexpr int kFoldChannels = 8;
__device__ __forceinline__ void fold_channels(const float2* __restrict__ chan, int64_t rows, int C, int c0, float* __restrict__ dgamma,
                                              float* __restrict__ dbeta, double2* red) {
  const int k = threadIdx.x % kFoldChannels, c = c0 + k, lanes = blockDim.x / kFoldChannels;
  double a = 0.0, b = 0.0;
  if (c < C)
#pragma unroll 8
    for (int64_t r = threadIdx.x / kFoldChannels; r < rows; r += lanes) {
      const float2 v = chan[r * C + c];
      a += (double)v.x;
      b += (double)v.y;
    }
#pragma unroll
  for (int o = kFoldChannels; o < 64; o *= 2) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if ((threadIdx.x & 63) < kFoldChannels) red[(threadIdx.x >> 6) * kFoldChannels + k] = make_double2(a, b);
  __syncthreads();
  if (threadIdx.x < kFoldChannels && c < C) {
    a = b = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
      a += red[w * kFoldChannels + k].x;
      b += red[w * kFoldChannels + k].y;
    }
    if (dbeta) dbeta[c] = (float)a;
    if (dgamma) dgamma[c] = (float)b;
  }
}
__global__ __launch_bounds__(256) void gn_channels_kernel(const float2* __restrict__ chan, int64_t rows, int C, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta) {
  __shared__ double2 red[4 * kFoldChannels];
  fold_channels(chan, rows, C, blockIdx.x * kFoldChannels, dgamma, dbeta, red);
}

// Backward, second pass.  The first `extra` workgroups fold dgamma and dbeta; folded: part holds [N][G] means already
template <class T, int V, int ACT, bool NT, int DEEP>
__global__ __launch_bounds__(512) void gn_bwd_apply_kernel(const T* __restrict__ dy, Img di, const T* __restrict__ x, Img xi, Plan p, int64_t HW, int N,
                                                          int C, int G, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta, float slope,
                                                          const float2* __restrict__ part, int folded, const float2* __restrict__ chan, int extra,
                                                          float* __restrict__ dgamma, float* __restrict__ dbeta, T* __restrict__ dx) {
  extern __shared__ float2 stat[];
  if ((int)blockIdx.x < extra) {
    fold_channels(chan, (int64_t)N * p.nb, C, blockIdx.x * kFoldChannels, dgamma, dbeta, reinterpret_cast<double2*>(stat));
    return;
  }
  const int block = backwards(blockIdx.x - extra, gridDim.x - extra);
  const Tile t = tile_of<V>(p, block % p.tiles, G);
  const int b = (block / p.tiles) % p.nb, n = block / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = threadIdx.x % p.qt;
  const bool on = l < p.pl && q < t.nq;
  const T* xs = x + n * xi.ns + t.c0 + q * V;
  const T* ds = dy + n * di.ns + t.c0 + q * V;
  T* os = dx + (int64_t)n * HW * C + t.c0 + q * V;
  auto w = walk<true, DEEP>(p, HW, b, l, [&](int64_t i) {
    return Two<T, V>{*reinterpret_cast<const Vec<T, V>*>(xs + i * xi.ps), *reinterpret_cast<const Vec<T, V>*>(ds + i * di.ps)};
  });
  if (on) w.begin();
  for_groups(t.ng, [&](int g, int lane, int lanes) {
    const int k = t.g0 + min(g, t.ng - 1);
    const float2 r = folded ? part[n * G + k] : fold_means(part, p, HW, G, n, k, lane, lanes);
    if (g < t.ng && lane == 0) stat[g] = r;
  });
  __syncthreads();
  if (!on) return;
  float mu[V], rs[V], ga[V], be[V], c1[V], c2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = t.c0 + q * V + e, g = p.split == 1 ? (q * V + e) / p.D : 0, k = n * G + t.g0 + g;
    mu[e] = mean[k];
    rs[e] = rstd[k];
    ga[e] = gamma ? gamma[c] : 1.f;
    be[e] = beta ? beta[c] : 0.f;
    c1[e] = stat[g].x;
    c2[e] = stat[g].y;
  }
  w.each([&](int64_t i, const Two<T, V>& r) {
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float xh = ((float)r.x.v[e] - mu[e]) * rs[e];
      const float t1 = (float)r.d.v[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope) * ga[e];
      o[e] = rs[e] * (t1 - c1[e] - xh * c2[e]);
    }
    stv<T, V, NT>(os + i * C, o);
  });
}

// ---------------------------------------------------------------- host side

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kMostVectors = 512;      // of a tile: its threads
constexpr int64_t kMostThreads = (int64_t)1 << 32;   // of a launch
// Partial results that a workgroup of the second pass folds by itself: 3760 of them beat a launch for it (2x30000x128 bf16, 16 groups, forward:
// 21.2 us to 21.9), 12000 do not (1x9000x704 bf16, 32 groups: 31.6 to 22.3)
constexpr int kFoldMost = 4096;

// widest vector that the channels, the strides and every pointer allow
inline int vector_width(int esize, int C, int G, bool small, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  for (int v = 16 / esize; v > 1; v /= 2) {
    bool ok = C % v == 0;
    for (const void* p : ptrs) ok = ok && (reinterpret_cast<uintptr_t>(p) % (v * esize)) == 0;
    for (int64_t s : strides) ok = ok && s % v == 0;
    // small: a group is whole vectors.  Large: a tile is whole groups that begin on the vector grid, or part of a group that does
    const int D = C / G, u = v / gcd(D, v);
    ok = ok && (small ? D % v == 0 : C / v <= kMostVectors || (int64_t)u * D / v <= kMostVectors || D % v == 0);
    if (ok) return v;
  }
  return 1;
}

// Loads a thread has in flight together: 4, or more where they are narrow and memory would wait for requests.  Forward, odd channel
// counts: 33 channels fp32 50 -> 40 us (bf16 46 -> 31), 301 37 -> 35 (33 -> 28); 2-byte loads 16 deep up to 128 vectors (33: 35 -> 31, 701:
// 46 -> 50).  Backward with its two inputs: 33 channels 74 -> 60 (52 -> 47), 101 the same, 201 68 -> 72 (41 -> 46): up to 64 vectors only.
// bytes: a load's; vectors: a pixel's
struct DeepForward {
  constexpr int operator()(int bytes, int vectors) const { return bytes >= 8 ? 4 : bytes == 2 && vectors <= 128 ? 16 : 8; }
};
struct DeepBackward {
  constexpr int operator()(int bytes, int vectors) const { return bytes >= 8 || vectors > 64 ? 4 : 8; }
};
// f(depth, as a constant)
template <int BYTES, class R, class F>
int with_depth(R rule, int vectors, F f) {
  constexpr int kNarrow = R()(BYTES, 1), kWide = R()(BYTES, 1 << 20);
  if constexpr (kNarrow != kWide)
    if (rule(BYTES, vectors) == kNarrow) return f(std::integral_constant<int, kNarrow>());
  return f(std::integral_constant<int, kWide>());
}

inline Plan make_plan(int N, int64_t HW, int C, int G, int V, int deep, bool narrow) {
  Plan p;
  p.D = C / G;
  const int Q = C / V, u = V / gcd(p.D, V);
  p.split = 1;
  if (Q <= kMostVectors) {
    p.gpt = G;
    p.qt = Q;
    p.tiles = 1;
  } else if ((int64_t)u * p.D / V <= kMostVectors) {
    const int run = u * p.D / V;
    p.gpt = u * (kMostVectors / run);
    p.qt = p.gpt * p.D / V;
    p.tiles = (G + p.gpt - 1) / p.gpt;
  } else {
    const int w = p.D / V;
    p.gpt = 1;
    p.split = (w + kMostVectors - 1) / kMostVectors;
    p.qt = (w + p.split - 1) / p.split;
    p.split = (w + p.qt - 1) / p.qt;
    p.tiles = G * p.split;
  }
  const int most = p.qt > 128 ? 512 : 256;
  p.pl = most / p.qt > 1 ? most / p.qt : 1;
  p.threads = (p.qt * p.pl + 63) / 64 * 64;
  // Workgroups: two of 256 threads a CU saturate HBM with loads of 8 and 16 bytes, and what a workgroup costs beside them (its partial
  // results, and folding everybody's) counts double with twice as many (13x1777x320 bf16, 32 groups: 26 us forward and 42 backward with four a
  // CU, 21 and 27 with two); narrow loads want four (2x12000x701 bf16: 29 and 41 us, 37 and 57 with two).  All take equally many runs but for the
  // last, if need be with an eighth more workgroups: the slowest decides (11x20000x40 bf16: 23 and 37 us as even as the numbers come, 20 and 26 so)
  p.run = deep * p.pl;
  const int64_t runs = (HW + p.run - 1) / p.run;
  int64_t want = (narrow ? 262144 : 131072) / p.threads / ((int64_t)N * p.tiles);
  want = want < 1 ? 1 : want > 512 ? 512 : want;
  // (no fp32 sum of a thread has more than 256 terms)
  const int64_t most_runs = 256 / deep, least = (runs + most_runs - 1) / most_runs;
  want = want < least ? least : want;
  int64_t each = (runs - want / 8 + want - 1) / want;
  each = each < 1 ? 1 : each;
  p.nb = (int)((runs + each - 1) / each);
  p.each = runs / p.nb;
  p.more = (int)(runs % p.nb);
  p.last = (int)((runs - 1) % p.nb);
  p.missing = (int)(runs * p.run - HW);
  return p;
}

// The small form takes what fits the registers of one workgroup whatever the vector width: 16 values a thread of 1024 (512 with 32)
inline bool is_small(int64_t HW, int D) { return D <= 1024 && HW <= 16 * (1024 / D); }
struct Small {
  int dv, pl, threads;
};
template <int V>
inline Small make_small(int64_t HW, int D) {
  Small s;
  s.dv = D / V;
  const int64_t most = kSmallThreads<V> / s.dv;
  s.pl = (int)(HW < most ? HW : most);
  s.threads = (s.dv * s.pl + 63) / 64 * 64;
  return s;
}

// A result larger than the eight L2 caches goes past them and the infinity cache: its reader would not find it there, and what it does
// not push out is the input that this pass still has to read (8x64x2048x32 fp32: 80 -> 67 us, its step in bf16 with 704 channels 164 -> 148)
inline bool past_caches(int N, int64_t HW, int C, int esize) { return (int64_t)N * HW * C * esize > (32 << 20); }

template <class F>
int with_vector(int v, F f) {
  switch (v) {
    case 8: return f(std::integral_constant<int, 8>());
    case 4: return f(std::integral_constant<int, 4>());
    case 2: return f(std::integral_constant<int, 2>());
    default: return f(std::integral_constant<int, 1>());
  }
}
template <class F>
int with_act(int act, F f) {
  switch (act) {
    case ACT_LRELU: return f(std::integral_constant<int, ACT_LRELU>());
    case ACT_SILU: return f(std::integral_constant<int, ACT_SILU>());
    default: return f(std::integral_constant<int, ACT_NONE>());
  }
}

template <class T>
int forward(const T* x, Img xi, int N, int64_t HW, int C, int G, const float* gamma, const float* beta, float eps, int act, float slope, T* y,
            float* mean, float* rstd, float* ws, hipStream_t s) {
  const bool small = is_small(HW, C / G);
  return with_vector(vector_width(sizeof(T), C, G, small, {x, y}, {xi.ns, xi.ps}), [&](auto vv) {
    constexpr int V = decltype(vv)::value;
    if constexpr (V * sizeof(T) <= 16) {
      return with_act(act, [&](auto aa) {
        constexpr int A = decltype(aa)::value;
        if (small) {
          const Small m = make_small<V>(HW, C / G);
          C3D_REQUIRE((int64_t)N * G * m.threads < kMostThreads, "group_norm: too many samples and groups");
          hipLaunchKernelGGL((gn_small_kernel<T, V, A>), dim3(N * G), dim3(m.threads), 0, s, x, xi, (int)HW, C, G, m.dv, m.pl, gamma, beta, eps, slope, y,
                             mean, rstd);
          C3D_CHECK_LAUNCH();
          return 0;
        }
        return with_depth<V * sizeof(T)>(DeepForward(), C / V, [&](auto dd) {
          constexpr int DEEP = decltype(dd)::value;
          const Plan p = make_plan(N, HW, C, G, V, DEEP, V * sizeof(T) < 8);
          C3D_REQUIRE((int64_t)p.tiles * p.nb * N * p.threads < kMostThreads, "group_norm: too many samples and channels");
          const dim3 grid((unsigned)(p.tiles * p.nb * N));
          float2* part = reinterpret_cast<float2*>(ws);
          const size_t lds = (size_t)(p.pl > 2 ? p.pl : 2) * p.qt * V * sizeof(float2);
          hipLaunchKernelGGL((gn_stats_kernel<T, V, DEEP>), grid, dim3(p.threads), lds, s, x, xi, p, HW, G, part);
          C3D_CHECK_LAUNCH();
          const bool fold = p.gpt * p.nb * p.split > kFoldMost;
          if (fold) {
            hipLaunchKernelGGL(gn_fold_kernel<V>, dim3(N * G), dim3(64), 0, s, part, p, HW, G, eps, mean, rstd);
            C3D_CHECK_LAUNCH();
          }
          // (only whole vectors of 16 bytes have the form that goes past the caches)
          const auto apply = V * sizeof(T) == 16 && past_caches(N, HW, C, sizeof(T)) ? gn_apply_kernel<T, V, A, V * sizeof(T) == 16, DEEP> : gn_apply_kernel<T, V, A, false, DEEP>;
          hipLaunchKernelGGL(apply, grid, dim3(p.threads), p.gpt * sizeof(float2), s, x, xi, p, HW, C, G, fold ? nullptr : part, eps,
                             mean, rstd, gamma, beta, slope, y);
          C3D_CHECK_LAUNCH();
          return 0;
        });
      });
    }
    return 2;
  });
}

template <class T>
int backward(const T* dy, Img di, const T* x, Img xi, int N, int64_t HW, int C, int G, const float* mean, const float* rstd, const float* gamma,
             const float* beta, int act, float slope, T* dx, float* dgamma, float* dbeta, float* ws, hipStream_t s) {
  const bool small = is_small(HW, C / G);
  return with_vector(vector_width(sizeof(T), C, G, small, {x, dy, dx}, {xi.ns, xi.ps, di.ns, di.ps}), [&](auto vv) {
    constexpr int V = decltype(vv)::value;
    if constexpr (V * sizeof(T) <= 16) {
      const bool wanted = dgamma || dbeta;
      const int extra = wanted ? ((C + kFoldChannels - 1) / kFoldChannels + 7) / 8 * 8 : 0;      // of eights, so that a chunk keeps its XCD
      return with_act(act, [&](auto aa) {
        constexpr int A = decltype(aa)::value;
        if (small) {
          const Small m = make_small<V>(HW, C / G);
          float2* chan = reinterpret_cast<float2*>(ws);
          const size_t lds = wanted ? (size_t)(m.pl + (m.pl > 1 ? (m.pl + 7) / 8 : 0)) * (C / G) * sizeof(float2) : 0;   // 49 KB at most
          C3D_REQUIRE((int64_t)N * G * m.threads < kMostThreads, "group_norm_bwd: too many samples and groups");
          hipLaunchKernelGGL((gn_small_bwd_kernel<T, V, A>), dim3(N * G), dim3(m.threads), lds, s, dy, di, x, xi, (int)HW, C, G, m.dv, m.pl, mean, rstd,
                             gamma, beta, slope, dx, (int)wanted, chan, dgamma, dbeta);
          C3D_CHECK_LAUNCH();
          if (wanted && N > 1) {
            hipLaunchKernelGGL(gn_channels_kernel, dim3((C + kFoldChannels - 1) / kFoldChannels), dim3(256), 0, s, chan, (int64_t)N, C, dgamma, dbeta);
            C3D_CHECK_LAUNCH();
          }
          return 0;
        }
        return with_depth<V * sizeof(T)>(DeepBackward(), C / V, [&](auto dd) {
          constexpr int DEEP = decltype(dd)::value;
          const Plan p = make_plan(N, HW, C, G, V, DEEP, V * sizeof(T) < 8);
          C3D_REQUIRE(((int64_t)p.tiles * p.nb * N + extra) * p.threads < kMostThreads, "group_norm_bwd: too many samples and channels");
          const int blocks = p.tiles * p.nb * N;
          float2* part = reinterpret_cast<float2*>(ws);
          float2* chan = part + (int64_t)N * G * p.nb * p.split;
          float2* coef = chan + (int64_t)N * p.nb * C;
          const size_t lds = (size_t)(p.pl > 2 ? p.pl : 2) * p.qt * V * sizeof(float2);
          hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, A, DEEP>), dim3(blocks), dim3(p.threads), lds, s, dy, di, x, xi, p, HW, C, G, mean, rstd, gamma, beta,
                             slope, part, wanted ? chan : nullptr);
          C3D_CHECK_LAUNCH();
          const bool fold = p.gpt * p.nb * p.split > kFoldMost;
          if (fold) {
            hipLaunchKernelGGL(gn_bwd_fold_kernel, dim3(N * G), dim3(64), 0, s, part, p, HW, G, coef);
            C3D_CHECK_LAUNCH();
          }
          const size_t lds2 = std::max(p.gpt * sizeof(float2), wanted ? 8 * kFoldChannels * sizeof(double2) : 0);
          const auto apply =
              V * sizeof(T) == 16 && past_caches(N, HW, C, sizeof(T)) ? gn_bwd_apply_kernel<T, V, A, V * sizeof(T) == 16, DEEP> : gn_bwd_apply_kernel<T, V, A, false, DEEP>;
          hipLaunchKernelGGL(apply, dim3(blocks + extra), dim3(p.threads), lds2, s, dy, di, x, xi, p, HW, N, C, G, mean, rstd, gamma,
                             beta, slope, fold ? coef : part, (int)fold, chan, extra, dgamma, dbeta, dx);
          C3D_CHECK_LAUNCH();
          return 0;
        });
      });
    }
    return 2;
  });
}

int check(int N, int64_t HW, int C, int G, int type, int act, float slope) {
  C3D_REQUIRE(N >= 0 && HW >= 0 && C >= 1 && G >= 1, "group_norm: negative size");
  C3D_REQUIRE(C % G == 0, "group_norm: the channels do not divide into the groups");
  C3D_REQUIRE(type >= 0 && type <= 2, "group_norm: type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(act >= ACT_NONE && act <= ACT_SILU, "group_norm: act is 0 (none), 1 (LeakyReLU) or 2 (SiLU)");
  C3D_REQUIRE(act != ACT_LRELU || (slope >= 0.f && slope <= 1.f), "group_norm: slope is in [0, 1]");
  C3D_REQUIRE((int64_t)N * C < (int64_t)1 << 31 && C <= 1 << 20, "group_norm: too many samples or channels");
  return 0;
}

}  // namespace

extern "C" int64_t c3d_group_norm_ws_floats(int N, int64_t HW, int C, int G, int type) {
  if (check(N, HW, C, G, type, 0, 0.f) || N == 0 || HW == 0) return 0;
  if (is_small(HW, C / G)) return N > 1 ? 2 * (int64_t)N * C : 0;
  int64_t most = 0;
  for (int v = 16 / (type == 0 ? 4 : 2); v >= 1; v /= 2) {
    if (C % v) continue;
    const int D = C / G, u = v / gcd(D, v);
    if (!(C / v <= kMostVectors || (int64_t)u * D / v <= kMostVectors || D % v == 0)) continue;
    for (int deep : {DeepForward()(v * (type == 0 ? 4 : 2), C / v), DeepBackward()(v * (type == 0 ? 4 : 2), C / v)}) {
      const Plan p = make_plan(N, HW, C, G, v, deep, v * (type == 0 ? 4 : 2) < 8);
      const int64_t f = 2 * ((int64_t)N * G * p.nb * p.split + (int64_t)N * p.nb * C + (int64_t)N * G);
      most = f > most ? f : most;
    }
  }
  return most;
}

extern "C" int c3d_group_norm(const void* x, int64_t x_ns, int64_t x_ps, int N, int64_t HW, int C, int G, int type, const float* gamma,
                              const float* beta, float eps, int act, float slope, void* y, float* mean, float* rstd, float* ws, c3d_stream stream) {
  if (int rc = check(N, HW, C, G, type, act, slope)) return rc;
  C3D_REQUIRE(eps >= 0.f, "group_norm: eps is negative or not a number");
  if (N == 0 || HW == 0) return 0;
  C3D_REQUIRE(x && y && mean && rstd && (ws || is_small(HW, C / G)), "group_norm: null pointer");
  C3D_REQUIRE(x_ps >= C && (N == 1 || x_ns >= (HW - 1) * x_ps + C), "group_norm: strides overlap");
  const Img xi{x_ns, x_ps};
  hipStream_t s = (hipStream_t)stream;
  if (type == 0) return forward<float>((const float*)x, xi, N, HW, C, G, gamma, beta, eps, act, slope, (float*)y, mean, rstd, ws, s);
  if (type == 1) return forward<__bf16>((const __bf16*)x, xi, N, HW, C, G, gamma, beta, eps, act, slope, (__bf16*)y, mean, rstd, ws, s);
  return forward<_Float16>((const _Float16*)x, xi, N, HW, C, G, gamma, beta, eps, act, slope, (_Float16*)y, mean, rstd, ws, s);
}

extern "C" int c3d_group_norm_bwd(const void* dy, int64_t dy_ns, int64_t dy_ps, const void* x, int64_t x_ns, int64_t x_ps, int N, int64_t HW, int C,
                                  int G, int type, const float* mean, const float* rstd, const float* gamma, const float* beta, int act, float slope,
                                  void* dx, float* dgamma, float* dbeta, float* ws, c3d_stream stream) {
  if (int rc = check(N, HW, C, G, type, act, slope)) return rc;
  if (N == 0 || HW == 0) return 0;
  C3D_REQUIRE(x && dy && dx && mean && rstd && (ws || (N == 1 && is_small(HW, C / G))), "group_norm_bwd: null pointer");
  C3D_REQUIRE(x_ps >= C && (N == 1 || x_ns >= (HW - 1) * x_ps + C), "group_norm_bwd: strides of x overlap");
  C3D_REQUIRE(dy_ps >= C && (N == 1 || dy_ns >= (HW - 1) * dy_ps + C), "group_norm_bwd: strides of dy overlap");
  const Img xi{x_ns, x_ps}, di{dy_ns, dy_ps};
  hipStream_t s = (hipStream_t)stream;
  if (type == 0)
    return backward<float>((const float*)dy, di, (const float*)x, xi, N, HW, C, G, mean, rstd, gamma, beta, act, slope, (float*)dx, dgamma, dbeta, ws, s);
  if (type == 1)
    return backward<__bf16>((const __bf16*)dy, di, (const __bf16*)x, xi, N, HW, C, G, mean, rstd, gamma, beta, act, slope, (__bf16*)dx, dgamma, dbeta,
                            ws, s);
  return backward<_Float16>((const _Float16*)dy, di, (const _Float16*)x, xi, N, HW, C, G, mean, rstd, gamma, beta, act, slope, (_Float16*)dx, dgamma,
                            dbeta, ws, s);
}
