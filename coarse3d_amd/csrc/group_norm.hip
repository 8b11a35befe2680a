// GroupNorm with an activation over channels-last images, forward and backward (gfx950; HBM-bound).
//
// For sample n and group g (D = C / G channels, HW pixels, M = HW * D values):
//     xhat = (x - mean) * rstd,  z = xhat * gamma[c] + beta[c],  y = act(z)
// and, with dz = dy * act'(z), t = dz * gamma:
//     dbeta = sum dz,  dgamma = sum dz * xhat  (over samples and pixels),  dx = rstd * (t - mean(t) - xhat * mean(t * xhat)).
//
// A thread owns V consecutive channels (16 bytes where alignment allows) and walks pixels, so that every load is a whole vector of
// a pixel's row whatever D is; what belongs to a group is only put together when the per-channel partial sums are folded.
#include <initializer_list>
#include <type_traits>
#include "common.h"
#include "../../include/coarse3d_hip.h"

namespace {

constexpr int kThreads = 256;

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
template <class T, int V>
__device__ __forceinline__ void stv(T* p, const float (&r)[V]) {
  Vec<T, V> t;
#pragma unroll
  for (int q = 0; q < V; ++q) t.v[q] = (T)r[q];
  *reinterpret_cast<Vec<T, V>*>(p) = t;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(float z, float slope) {
  if (ACT == ACT_LRELU) return z > 0.f ? z : z * slope;
  if (ACT == ACT_SILU) return z / (1.f + expf(-z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_bwd(float z, float slope) {
  if (ACT == ACT_LRELU) return z > 0.f ? 1.f : slope;
  if (ACT == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

// How an image is cut: `qt` vectors (of Q = C / V) a workgroup, `pl` pixels side by side, `nb` workgroups along a sample's pixels
struct Plan {
  int Q, qt, pl, tiles, nb;
  int64_t ppb;              // pixels a workgroup
};
inline Plan make_plan(int N, int64_t HW, int C, int V) {
  Plan p;
  p.Q = C / V;
  p.qt = p.Q < kThreads ? p.Q : kThreads;
  p.tiles = (p.Q + p.qt - 1) / p.qt;
  p.pl = kThreads / p.qt;
  const int64_t most = (HW + p.pl * 8 - 1) / (p.pl * 8);       // at least eight pixels a thread
  int64_t want = 1024 / ((int64_t)N * p.tiles);
  if (want < 1) want = 1;
  if (want > 512) want = 512;
  p.nb = (int)(most < want ? most : want);
  if (p.nb < 1) p.nb = 1;
  p.ppb = (HW + p.nb - 1) / p.nb;
  return p;
}

struct Img {
  int64_t ns, ps;           // elements from sample to sample and from pixel to pixel
};

// per workgroup and channel: mean and sum of squared deviations of its pixels, [2][N][nb][C].  Values are shifted by the chunk's first
// pixel, so that a mean far from zero costs nothing.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void gn_stats_kernel(const T* __restrict__ x, Img xi, Plan p, int N, int64_t HW, int C,
                                                           float* __restrict__ part) {
  extern __shared__ float red[];
  const int tile = blockIdx.x % p.tiles, b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = tile * p.qt + threadIdx.x % p.qt;
  const bool on = l < p.pl && q < p.Q;
  const int64_t p0 = b * p.ppb, p1 = p0 + p.ppb < HW ? p0 + p.ppb : HW;
  const T* xs = x + n * xi.ns + (int64_t)q * V;
  float shift[V], s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) shift[e] = s1[e] = s2[e] = 0.f;
  if (on && p0 < p1) {
    ldv<T, V>(xs + p0 * xi.ps, shift);
    for (int64_t i = p0 + l; i < p1; i += p.pl) {
      float r[V];
      ldv<T, V>(xs + i * xi.ps, r);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = r[e] - shift[e];
        s1[e] += d;
        s2[e] = fmaf(d, d, s2[e]);
      }
    }
  }
  const int W = p.qt * V;
  if (on) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      red[(l * 2 + 0) * W + (threadIdx.x % p.qt) * V + e] = s1[e];
      red[(l * 2 + 1) * W + (threadIdx.x % p.qt) * V + e] = s2[e];
    }
  }
  __syncthreads();
  if (on && l == 0) {
    const float cnt = (float)(p1 - p0);
    float* o = part + ((int64_t)n * p.nb + b) * C + (int64_t)q * V;
    const int64_t plane = (int64_t)N * p.nb * C;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a1 = 0.f, a2 = 0.f;
      for (int k = 0; k < p.pl; ++k) {
        a1 += red[(k * 2 + 0) * W + threadIdx.x * V + e];
        a2 += red[(k * 2 + 1) * W + threadIdx.x * V + e];
      }
      const bool any = p1 > p0;
      const float mu = any ? a1 / cnt : 0.f;
      o[e] = shift[e] + mu;
      o[plane + e] = any ? a2 - a1 * mu : 0.f;
    }
  }
}

// one workgroup a (sample, group): joins the partial means and squared deviations in 64 bits
__global__ __launch_bounds__(kThreads) void gn_fold_kernel(const float* __restrict__ part, Plan p, int N, int64_t HW, int C, int G, float eps,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ double red[4];
  const int n = blockIdx.x / G, g = blockIdx.x % G, D = C / G;
  const int64_t plane = (int64_t)N * p.nb * C;
  const float* a = part + (int64_t)n * p.nb * C + g * D;
  const double M = (double)HW * D;
  const int total = p.nb * D;
  auto block_sum = [&](double s) {
    s = c3d_wave_sum_d(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  };
  auto count = [&](int b) {
    const int64_t p0 = b * p.ppb, p1 = p0 + p.ppb < HW ? p0 + p.ppb : HW;
    return p1 > p0 ? (double)(p1 - p0) : 0.0;
  };
  double s = 0.0;
  for (int i = threadIdx.x; i < total; i += kThreads) s += count(i / D) * (double)a[(int64_t)(i / D) * C + i % D];
  const double mu = block_sum(s) / M;
  s = 0.0;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int64_t at = (int64_t)(i / D) * C + i % D;
    const double d = (double)a[at] - mu;
    s += (double)a[plane + at] + count(i / D) * d * d;
  }
  const double var = block_sum(s) / M;
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = (float)mu;
    rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)eps));
  }
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(const T* __restrict__ x, Img xi, Plan p, int64_t HW, int C, int G,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta, float slope,
                                                           T* __restrict__ y) {
  const int tile = blockIdx.x % p.tiles, b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = tile * p.qt + threadIdx.x % p.qt;
  if (l >= p.pl || q >= p.Q) return;
  const int64_t p0 = b * p.ppb, p1 = p0 + p.ppb < HW ? p0 + p.ppb : HW;
  const T* xs = x + n * xi.ns + (int64_t)q * V;
  T* ys = y + (int64_t)n * HW * C + (int64_t)q * V;
  float mu[V], sc[V], sh[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = q * V + e, g = n * G + c / (C / G);
    mu[e] = mean[g];
    sc[e] = rstd[g] * (gamma ? gamma[c] : 1.f);
    sh[e] = beta ? beta[c] : 0.f;
  }
  for (int64_t i = p0 + l; i < p1; i += p.pl) {
    float r[V];
    ldv<T, V>(xs + i * xi.ps, r);
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = act_fwd<ACT>(fmaf(r[e] - mu[e], sc[e], sh[e]), slope);
    stv<T, V>(ys + i * C, r);
  }
}

// per workgroup and channel: sum dz and sum dz * xhat, [2][N][nb][C]
template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void gn_bwd_stats_kernel(const T* __restrict__ dy, Img di, const T* __restrict__ x, Img xi, Plan p, int N,
                                                               int64_t HW, int C, int G, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, float slope, float* __restrict__ part) {
  extern __shared__ float red[];
  const int tile = blockIdx.x % p.tiles, b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = tile * p.qt + threadIdx.x % p.qt;
  const bool on = l < p.pl && q < p.Q;
  const int64_t p0 = b * p.ppb, p1 = p0 + p.ppb < HW ? p0 + p.ppb : HW;
  float s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
  if (on) {
    const T* xs = x + n * xi.ns + (int64_t)q * V;
    const T* ds = dy + n * di.ns + (int64_t)q * V;
    float mu[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = q * V + e, g = n * G + c / (C / G);
      mu[e] = mean[g];
      rs[e] = rstd[g];
      ga[e] = gamma ? gamma[c] : 1.f;
      be[e] = beta ? beta[c] : 0.f;
    }
    for (int64_t i = p0 + l; i < p1; i += p.pl) {
      float r[V], d[V];
      ldv<T, V>(xs + i * xi.ps, r);
      ldv<T, V>(ds + i * di.ps, d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (r[e] - mu[e]) * rs[e];
        const float dz = d[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope);
        s1[e] += dz;
        s2[e] = fmaf(dz, xh, s2[e]);
      }
    }
  }
  const int W = p.qt * V;
  if (on) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      red[(l * 2 + 0) * W + (threadIdx.x % p.qt) * V + e] = s1[e];
      red[(l * 2 + 1) * W + (threadIdx.x % p.qt) * V + e] = s2[e];
    }
  }
  __syncthreads();
  if (on && l == 0) {
    float* o = part + ((int64_t)n * p.nb + b) * C + (int64_t)q * V;
    const int64_t plane = (int64_t)N * p.nb * C;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a1 = 0.f, a2 = 0.f;
      for (int k = 0; k < p.pl; ++k) {
        a1 += red[(k * 2 + 0) * W + threadIdx.x * V + e];
        a2 += red[(k * 2 + 1) * W + threadIdx.x * V + e];
      }
      o[e] = a1;
      o[plane + e] = a2;
    }
  }
}

// workgroups [0, N G): mean(t) and mean(t xhat) of a (sample, group) -> coef [2][N][G]; the rest: dgamma, dbeta of one channel each
__global__ __launch_bounds__(kThreads) void gn_bwd_fold_kernel(const float* __restrict__ part, Plan p, int N, int64_t HW, int C, int G,
                                                              const float* __restrict__ gamma, float* __restrict__ coef,
                                                              float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double red[2][4];
  const int D = C / G;
  const int64_t plane = (int64_t)N * p.nb * C;
  double s1 = 0.0, s2 = 0.0;
  const bool group = blockIdx.x < (unsigned)(N * G);
  if (group) {
    const int n = blockIdx.x / G, g = blockIdx.x % G;
    const float* a = part + (int64_t)n * p.nb * C + g * D;
    for (int i = threadIdx.x; i < p.nb * D; i += kThreads) {
      const int64_t at = (int64_t)(i / D) * C + i % D;
      const double ga = gamma ? (double)gamma[g * D + i % D] : 1.0;
      s1 += ga * (double)a[at];
      s2 += ga * (double)a[plane + at];
    }
  } else {
    const int c = blockIdx.x - N * G;
    for (int i = threadIdx.x; i < N * p.nb; i += kThreads) {
      s1 += (double)part[(int64_t)i * C + c];
      s2 += (double)part[plane + (int64_t)i * C + c];
    }
  }
  s1 = c3d_wave_sum_d(s1);
  s2 = c3d_wave_sum_d(s2);
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = s1;
    red[1][threadIdx.x >> 6] = s2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s1 = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    s2 = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (group) {
      const double M = (double)HW * D;
      coef[blockIdx.x] = (float)(s1 / M);
      coef[N * G + blockIdx.x] = (float)(s2 / M);
    } else {
      const int c = blockIdx.x - N * G;
      if (dbeta) dbeta[c] = (float)s1;
      if (dgamma) dgamma[c] = (float)s2;
    }
  }
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void gn_bwd_apply_kernel(const T* __restrict__ dy, Img di, const T* __restrict__ x, Img xi, Plan p, int N,
                                                               int64_t HW, int C, int G, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, float slope, const float* __restrict__ coef,
                                                               T* __restrict__ dx) {
  const int tile = blockIdx.x % p.tiles, b = (blockIdx.x / p.tiles) % p.nb, n = blockIdx.x / (p.tiles * p.nb);
  const int l = threadIdx.x / p.qt, q = tile * p.qt + threadIdx.x % p.qt;
  if (l >= p.pl || q >= p.Q) return;
  const int64_t p0 = b * p.ppb, p1 = p0 + p.ppb < HW ? p0 + p.ppb : HW;
  const T* xs = x + n * xi.ns + (int64_t)q * V;
  const T* ds = dy + n * di.ns + (int64_t)q * V;
  T* os = dx + (int64_t)n * HW * C + (int64_t)q * V;
  float mu[V], rs[V], ga[V], be[V], c1[V], c2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = q * V + e, g = n * G + c / (C / G);
    mu[e] = mean[g];
    rs[e] = rstd[g];
    ga[e] = gamma ? gamma[c] : 1.f;
    be[e] = beta ? beta[c] : 0.f;
    c1[e] = coef[g];
    c2[e] = coef[N * G + g];
  }
  for (int64_t i = p0 + l; i < p1; i += p.pl) {
    float r[V], d[V];
    ldv<T, V>(xs + i * xi.ps, r);
    ldv<T, V>(ds + i * di.ps, d);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float xh = (r[e] - mu[e]) * rs[e];
      const float t = d[e] * act_bwd<ACT>(fmaf(xh, ga[e], be[e]), slope) * ga[e];
      r[e] = rs[e] * (t - c1[e] - xh * c2[e]);
    }
    stv<T, V>(os + i * C, r);
  }
}

// ---------------------------------------------------------------- host side

// widest vector that C, both strides and every pointer allow
inline int vector_width(int esize, int C, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  for (int v = 16 / esize; v > 1; v /= 2) {
    bool ok = C % v == 0;
    for (const void* p : ptrs) ok = ok && (reinterpret_cast<uintptr_t>(p) % (v * esize)) == 0;
    for (int64_t s : strides) ok = ok && s % v == 0;
    if (ok) return v;
  }
  return 1;
}

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
  return with_vector(vector_width(sizeof(T), C, {x, y}, {xi.ns, xi.ps}), [&](auto vv) {
    constexpr int V = decltype(vv)::value;
    if constexpr (V * sizeof(T) <= 16) {
      const Plan p = make_plan(N, HW, C, V);
      const dim3 grid((unsigned)(p.tiles * p.nb * N));
      hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(kThreads), p.pl * 2 * p.qt * V * sizeof(float), s, x, xi, p, N, HW, C, ws);
      C3D_CHECK_LAUNCH();
      hipLaunchKernelGGL(gn_fold_kernel, dim3(N * G), dim3(kThreads), 0, s, ws, p, N, HW, C, G, eps, mean, rstd);
      C3D_CHECK_LAUNCH();
      return with_act(act, [&](auto aa) {
        hipLaunchKernelGGL((gn_apply_kernel<T, V, decltype(aa)::value>), grid, dim3(kThreads), 0, s, x, xi, p, HW, C, G, mean, rstd, gamma, beta, slope, y);
        C3D_CHECK_LAUNCH();
        return 0;
      });
    }
    return 2;
  });
}

template <class T>
int backward(const T* dy, Img di, const T* x, Img xi, int N, int64_t HW, int C, int G, const float* mean, const float* rstd, const float* gamma,
             const float* beta, int act, float slope, T* dx, float* dgamma, float* dbeta, float* ws, hipStream_t s) {
  return with_vector(vector_width(sizeof(T), C, {x, dy, dx}, {xi.ns, xi.ps, di.ns, di.ps}), [&](auto vv) {
    constexpr int V = decltype(vv)::value;
    if constexpr (V * sizeof(T) <= 16) {
      const Plan p = make_plan(N, HW, C, V);
      const dim3 grid((unsigned)(p.tiles * p.nb * N));
      float* coef = ws + 2 * (int64_t)N * p.nb * C;
      return with_act(act, [&](auto aa) {
        constexpr int A = decltype(aa)::value;
        hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, A>), grid, dim3(kThreads), p.pl * 2 * p.qt * V * sizeof(float), s, dy, di, x, xi, p, N, HW, C, G,
                           mean, rstd, gamma, beta, slope, ws);
        C3D_CHECK_LAUNCH();
        hipLaunchKernelGGL(gn_bwd_fold_kernel, dim3(N * G + (dgamma || dbeta ? C : 0)), dim3(kThreads), 0, s, ws, p, N, HW, C, G, gamma, coef, dgamma,
                           dbeta);
        C3D_CHECK_LAUNCH();
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, A>), grid, dim3(kThreads), 0, s, dy, di, x, xi, p, N, HW, C, G, mean, rstd, gamma, beta, slope, coef,
                           dx);
        C3D_CHECK_LAUNCH();
        return 0;
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
  C3D_REQUIRE((int64_t)N * C < (int64_t)1 << 24 && C <= 1 << 20, "group_norm: too many samples or channels");
  return 0;
}

}  // namespace

extern "C" int64_t c3d_group_norm_ws_floats(int N, int64_t HW, int C, int G, int type) {
  if (check(N, HW, C, G, type, 0, 0.f) || N == 0 || HW == 0) return 0;
  int64_t most = 0;
  for (int v = 16 / (type == 0 ? 4 : 2); v >= 1; v /= 2) {
    if (C % v) continue;
    const int64_t f = 2 * (int64_t)N * make_plan(N, HW, C, v).nb * C;
    most = f > most ? f : most;
  }
  return most + 2 * (int64_t)N * G;
}

extern "C" int c3d_group_norm(const void* x, int64_t x_ns, int64_t x_ps, int N, int64_t HW, int C, int G, int type, const float* gamma,
                              const float* beta, float eps, int act, float slope, void* y, float* mean, float* rstd, float* ws, c3d_stream stream) {
  if (int rc = check(N, HW, C, G, type, act, slope)) return rc;
  C3D_REQUIRE(eps >= 0.f, "group_norm: eps is negative or not a number");
  if (N == 0 || HW == 0) return 0;
  C3D_REQUIRE(x && y && mean && rstd && ws, "group_norm: null pointer");
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
  C3D_REQUIRE(x && dy && dx && mean && rstd && ws, "group_norm_bwd: null pointer");
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
