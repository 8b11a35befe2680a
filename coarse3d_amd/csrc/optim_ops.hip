// Operators over the many tensors of an optimiser: the global norm of the gradients, their clipping, and the AdamW step with
// states in 32 bits or in 8 bits.  All of them stream: nothing is read twice, and what bounds them is HBM.
//
// A call takes a host array of tensor records.  Records travel as kernel arguments (at most 4 KB a launch), so that nothing is
// copied to the device ahead of the launch and a captured launch carries its own table; each workgroup finds its record by a
// binary search over the records' first workgroups.
//
// AdamW (decoupled weight decay, step t, beta1 = b1, beta2 = b2):
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// The reference steps torch.optim.AdamW over all parameters (tasks/weak_segmentation/trainer.py:146-151).
#include "common.h"
#include "../../include/coarse3d_hip.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;            // elements a workgroup of the step and of the scaling handles
constexpr int kNormChunk = 16384;       // of the norm: a partial sum (8 bytes) each
constexpr int kBlock = C3D_ADAMW8_BLOCK;
constexpr int64_t kMaxRecord = 1 << 30; // longer tensors are cut into several records: 32-bit indices inside one
constexpr int kMaxBlocks = 1 << 22;     // workgroups a launch: threads stay below 2^32

template <int NP, int MAXT>
struct Table {
  void* ptr[NP][MAXT];
  uint32_t n[MAXT];
  uint32_t first[MAXT];     // first workgroup of the record
  uint32_t unit[MAXT];      // number of 8-bit blocks (norm: of partial sums) ahead of the record in the whole list
  int count;
  uint32_t align;           // NP bits are not kept per record: 1 = every pointer of every record is 16-byte aligned
};

template <class TB>
__device__ __forceinline__ int find_record(const TB& t, uint32_t block) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <class T>
struct alignas(4 * sizeof(T)) Vec4 {
  T v[4];
};

// four consecutive elements from i as floats; past n: 0
template <class T>
__device__ __forceinline__ f32x4 load4(const T* p, uint32_t i, uint32_t n, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec && i + 4 <= n) {
    const Vec4<T> t = *reinterpret_cast<const Vec4<T>*>(p + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = (float)t.v[q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < n) r[q] = (float)p[i + q];
  }
  return r;
}
template <class T>
__device__ __forceinline__ void store4(T* p, uint32_t i, uint32_t n, bool vec, f32x4 x) {
  if (vec && i + 4 <= n) {
    Vec4<T> t;
#pragma unroll
    for (int q = 0; q < 4; ++q) t.v[q] = (T)x[q];
    *reinterpret_cast<Vec4<T>*>(p + i) = t;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < n) p[i + q] = (T)x[q];
  }
}

// ---------------------------------------------------------------- norm and clipping

// squares and sums in 64 bits: no gradient overflows, and the factor that other roundings depend on is the same whatever the
// order of the sum
template <class T, int MAXT>
__global__ __launch_bounds__(kThreads) void grad_sumsq_kernel(Table<1, MAXT> t, double* __restrict__ partial) {
  __shared__ double red[kThreads / 64];
  const int k = find_record(t, blockIdx.x);
  const uint32_t local = blockIdx.x - t.first[k], n = t.n[k];
  const T* g = static_cast<const T*>(t.ptr[0][k]);
  const bool vec = t.align;
  double s = 0.0;
  for (uint32_t i = local * kNormChunk + threadIdx.x * 4; i < n && i < (local + 1) * kNormChunk; i += kThreads * 4) {
    const f32x4 x = load4(g, i, n, vec);
#pragma unroll
    for (int q = 0; q < 4; ++q) s = fma((double)x[q], (double)x[q], s);
  }
  s = c3d_wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[t.unit[k] + local] = (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(1024) void grad_norm_fold_kernel(const double* __restrict__ partial, int64_t n, double max_norm,
                                                             float* __restrict__ norm, float* __restrict__ scale) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = c3d_wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += red[w];
    const double r = sqrt(s);
    *norm = (float)r;
    const double f = max_norm / (r + 1e-6);
    *scale = (float)(f > 1.0 ? 1.0 : f);          // a norm that is not a number stays visible in the factor
  }
}

template <class T, int MAXT>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(Table<1, MAXT> t, const float* __restrict__ scale) {
  const int k = find_record(t, blockIdx.x);
  const uint32_t base = (blockIdx.x - t.first[k]) * kChunk, n = t.n[k];
  T* g = static_cast<T*>(t.ptr[0][k]);
  const bool vec = t.align;
  const float f = *scale;
  for (uint32_t i = base + threadIdx.x * 4; i < n && i < base + kChunk; i += kThreads * 4) {
    f32x4 x = load4(g, i, n, vec);
    x *= f;
    store4(g, i, n, vec, x);
  }
}

// ---------------------------------------------------------------- AdamW

struct Hyper {
  float beta1, omb1, beta2, omb2, eps;
  float decay, step_size, inv_root;       // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  double lr, wd, ln_b1, ln_b2;
  const float* lr_dev;                    // not null: the learning rate / the step count are read on the device
  const float* step_dev;
  const float* grad_scale;
  uint32_t seed, step;
};

// the three numbers that depend on lr and t; in 64 bits where they live on the device (1 - b2^t is a difference of near-equal numbers)
__device__ __forceinline__ void resolve(const Hyper& h, float& decay, float& step_size, float& inv_root, uint32_t& step) {
  decay = h.decay;
  step_size = h.step_size;
  inv_root = h.inv_root;
  step = h.step;
  if (h.step_dev || h.lr_dev) {
    const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
    const double t = h.step_dev ? (double)*h.step_dev : (double)h.step;
    decay = (float)(1.0 - lr * h.wd);
    step_size = (float)(lr / -expm1(t * h.ln_b1));
    inv_root = (float)(1.0 / sqrt(-expm1(t * h.ln_b2)));
    step = (uint32_t)t;
  }
}

template <class P, class G, bool MASTER, int MAXT>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table<MASTER ? 5 : 4, MAXT> t, Hyper h) {
  const int k = find_record(t, blockIdx.x);
  const uint32_t base = (blockIdx.x - t.first[k]) * kChunk, n = t.n[k];
  P* p = static_cast<P*>(t.ptr[0][k]);
  const G* g = static_cast<const G*>(t.ptr[1][k]);
  float* m = static_cast<float*>(t.ptr[2][k]);
  float* v = static_cast<float*>(t.ptr[3][k]);
  float* w = MASTER ? static_cast<float*>(t.ptr[MASTER ? 4 : 0][k]) : nullptr;
  const bool vec = t.align;
  float decay, step_size, inv_root;
  uint32_t step;
  resolve(h, decay, step_size, inv_root, step);
  const float gs = h.grad_scale ? *h.grad_scale : 1.f;
  for (uint32_t i = base + threadIdx.x * 4; i < n && i < base + kChunk; i += kThreads * 4) {
    const f32x4 gi = load4(g, i, n, vec);
    f32x4 mi = load4(m, i, n, vec), vi = load4(v, i, n, vec);
    f32x4 pi = MASTER ? load4(w, i, n, vec) : load4(p, i, n, vec);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = gi[q] * gs;
      mi[q] = mi[q] * h.beta1 + x * h.omb1;
      vi[q] = vi[q] * h.beta2 + (x * x) * h.omb2;
      const float root = sqrtf(vi[q]) * inv_root + h.eps;
      pi[q] = pi[q] * decay - step_size * (mi[q] / root);
    }
    store4(m, i, n, vec, mi);
    store4(v, i, n, vec, vi);
    if (MASTER) store4(w, i, n, vec, pi);
    store4(p, i, n, vec, pi);
  }
}

// ---------------------------------------------------------------- AdamW with states in 8 bits
//
// A block of 256 elements keeps m and r = sqrt(v) as e4m3 numbers times one power of two each, such that the block's largest value
// is in (224, 448].  r and not v: the root halves the exponent's range, so that m and r reach equally far below their block's
// largest value (2^-17.8) and m / r stays bounded; r > 0 is never stored as 0 for the same reason.  A power of two: products with
// it are exact.  Rounding is stochastic (16 bits an element, a hash of seed, step and the element's number): v moves by
// 1 - b2 = 0.1 % a step, which is less than half a code step, and rounding to nearest would freeze it.

__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x9E3779B1u;      // odd multipliers from the golden ratio and the square root of three
  h = (h ^ (h >> 15)) * 0xBB67AE85u;
  return h ^ (h >> 16);
}
__device__ __forceinline__ uint32_t shift_register(uint32_t h) {
  h ^= h << 13;
  h ^= h >> 17;
  return h ^ (h << 5);
}

// exponent k of the block's scale 2^k from the bits of its largest finite magnitude
__device__ __forceinline__ int scale_exponent(uint32_t amax) {
  const int k = (int)(amax >> 23) - 135 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return k < -100 ? -100 : k;
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// |x| * 2^-k -> e4m3 code by stochastic rounding: 16 random bits are added right below the last kept mantissa bit.  Below the
// smallest normal number 2^-6 the value is moved up by 2^-6, which puts the code's last bit at the same place.
__device__ __forceinline__ uint32_t e4m3_code(float ax, float inv, uint32_t rnd16) {
#pragma clang fp contract(off)
  const float a = ax * inv;
  const bool low = a < 0.015625f;
  const float z = low ? a + 0.015625f : a;
  uint32_t c = ((__float_as_uint(z) + (rnd16 << 4)) >> 20) - (low ? 121u * 8u : 120u * 8u);
  return c > 0x7eu ? 0x7eu : c;
}

template <class P, class G, bool MASTER, int MAXT>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(Table<MASTER ? 7 : 6, MAXT> t, Hyper h) {
#pragma clang fp contract(off)
  const int k = find_record(t, blockIdx.x);
  const uint32_t local = blockIdx.x - t.first[k], n = t.n[k];
  P* p = static_cast<P*>(t.ptr[0][k]);
  const G* g = static_cast<const G*>(t.ptr[1][k]);
  uint8_t* m8 = static_cast<uint8_t*>(t.ptr[2][k]);
  uint8_t* r8 = static_cast<uint8_t*>(t.ptr[3][k]);
  float* ms = static_cast<float*>(t.ptr[4][k]);
  float* rs = static_cast<float*>(t.ptr[5][k]);
  float* w = MASTER ? static_cast<float*>(t.ptr[MASTER ? 6 : 0][k]) : nullptr;
  const bool vec = t.align;
  float decay, step_size, inv_root;
  uint32_t step;
  resolve(h, decay, step_size, inv_root, step);
  const float gs = h.grad_scale ? *h.grad_scale : 1.f;
  const uint32_t key = mix32(h.seed + step * 0x9E3779B9u);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j = wave; j < kChunk / kBlock; j += kThreads / 64) {
    const uint32_t b = local * (kChunk / kBlock) + j;       // block of this record
    if (b * (uint32_t)kBlock >= n) break;                   // uniform over the wave
    const uint32_t i = b * kBlock + lane * 4;
    const f32x4 gi = load4(g, i, n, vec);
    f32x4 pi = MASTER ? load4(w, i, n, vec) : load4(p, i, n, vec);
    uint32_t mc = 0, rc = 0;
    if (vec && i + 4 <= n) {
      mc = *reinterpret_cast<const uint32_t*>(m8 + i);
      rc = *reinterpret_cast<const uint32_t*>(r8 + i);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i + q < n) {
          mc |= (uint32_t)m8[i + q] << (8 * q);
          rc |= (uint32_t)r8[i + q] << (8 * q);
        }
    }
    const float msc = ms[b], rsc = rs[b];
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, true);
    const f32x2_t r01 = __builtin_amdgcn_cvt_pk_f32_fp8(rc, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8(rc, true);
    const float mo[4] = {m01[0], m01[1], m23[0], m23[1]}, ro[4] = {r01[0], r01[1], r23[0], r23[1]};
    float mi[4], ri[4];
    uint32_t mmax = 0, rmax = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = gi[q] * gs;
      mi[q] = (mo[q] * msc) * h.beta1 + x * h.omb1;
      const float old = ro[q] * rsc;
      ri[q] = sqrtf((old * old) * h.beta2 + (x * x) * h.omb2);
      const float root = ri[q] * inv_root + h.eps;
      pi[q] = pi[q] * decay - step_size * (mi[q] / root);
      // magnitudes order like their bits; what is not finite does not count
      const uint32_t mb = __float_as_uint(mi[q]) & 0x7fffffffu, rb = __float_as_uint(ri[q]) & 0x7fffffffu;
      if (mb < 0x7f800000u && mb > mmax) mmax = mb;
      if (rb < 0x7f800000u && rb > rmax) rmax = rb;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      mmax = max(mmax, (uint32_t)__shfl_xor((int)mmax, o, 64));
      rmax = max(rmax, (uint32_t)__shfl_xor((int)rmax, o, 64));
    }
    const int mk = scale_exponent(mmax), rk = scale_exponent(rmax);
    const float minv = pow2(-mk), rinv = pow2(-rk);
    uint32_t rnd = mix32(key + (t.unit[k] + b) * (kBlock / 4) + lane);
    uint32_t mo8 = 0, ro8 = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t mb = __float_as_uint(mi[q]), rb = __float_as_uint(ri[q]);
      uint32_t cm = e4m3_code(fabsf(mi[q]), minv, rnd & 0xffffu);
      uint32_t cr = e4m3_code(fabsf(ri[q]), rinv, rnd >> 16);
      if (cr == 0u && ri[q] > 0.f) cr = 1u;
      if ((mb & 0x7fffffffu) >= 0x7f800000u) cm = 0x7fu;
      if ((rb & 0x7fffffffu) >= 0x7f800000u) cr = 0x7fu;
      mo8 |= (cm | ((mb >> 24) & 0x80u)) << (8 * q);
      ro8 |= cr << (8 * q);
      rnd = shift_register(rnd);
    }
    if (vec && i + 4 <= n) {
      *reinterpret_cast<uint32_t*>(m8 + i) = mo8;
      *reinterpret_cast<uint32_t*>(r8 + i) = ro8;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i + q < n) {
          m8[i + q] = (uint8_t)(mo8 >> (8 * q));
          r8[i + q] = (uint8_t)(ro8 >> (8 * q));
        }
    }
    if (lane == 0) {
      ms[b] = pow2(mk);
      rs[b] = pow2(rk);
    }
    if (MASTER) store4(w, i, n, vec, pi);
    store4(p, i, n, vec, pi);
  }
}

// ---------------------------------------------------------------- host side

// Walks the records in tables of at most MAXT and hands each to `launch(table, blocks)`.
// slots: which fields of c3d_opt_tensor the table's pointers are; chunk: elements a workgroup; unit: elements a unit of Table.unit
template <int NP, int MAXT, class F>
int for_each_table(const c3d_opt_tensor* t, int count, const int (&slots)[NP], const int (&bytes)[NP], int chunk, int unit, F launch) {
  Table<NP, MAXT> tab;
  static_assert(sizeof(tab) <= 4096 - sizeof(Hyper), "kernel arguments");
  tab.count = 0;
  tab.align = 1;
  uint32_t blocks = 0, units = 0;
  for (int i = 0; i < count; ++i) {
    for (int64_t at = 0; at < t[i].n; at += kMaxRecord) {
      const uint32_t n = (uint32_t)(t[i].n - at < kMaxRecord ? t[i].n - at : kMaxRecord);
      const uint32_t nb = (n + chunk - 1) / chunk;
      if (tab.count == MAXT || blocks + nb > (uint32_t)kMaxBlocks) {
        if (int rc = launch(tab, blocks)) return rc;
        tab.count = 0;
        tab.align = 1;
        blocks = 0;
      }
      const int c = tab.count++;
      for (int s = 0; s < NP; ++s) {
        char* base = static_cast<char*>(t[i].ptr[slots[s]]);
        // a scale (one for each block) moves with the block, everything else with the element
        tab.ptr[s][c] = base + (bytes[s] < 0 ? at / kBlock * 4 : at * bytes[s]);
        if (bytes[s] >= 0 && (reinterpret_cast<uintptr_t>(tab.ptr[s][c]) & (4 * bytes[s] - 1))) tab.align = 0;
      }
      tab.n[c] = n;
      tab.first[c] = blocks;
      tab.unit[c] = units;
      blocks += nb;
      units += (n + unit - 1) / unit;
    }
  }
  return tab.count ? launch(tab, blocks) : 0;
}

template <class T>
int sumsq(const c3d_opt_tensor* t, int count, double* partial, hipStream_t s) {
  constexpr int M = 192;
  return for_each_table<1, M>(t, count, {1}, {(int)sizeof(T)}, kNormChunk, kNormChunk, [&](const Table<1, M>& tab, uint32_t blocks) {
    hipLaunchKernelGGL((grad_sumsq_kernel<T, M>), dim3(blocks), dim3(kThreads), 0, s, tab, partial);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}
template <class T>
int scale_all(const c3d_opt_tensor* t, int count, const float* scale, hipStream_t s) {
  constexpr int M = 192;
  return for_each_table<1, M>(t, count, {1}, {(int)sizeof(T)}, kChunk, kChunk, [&](const Table<1, M>& tab, uint32_t blocks) {
    hipLaunchKernelGGL((grad_scale_kernel<T, M>), dim3(blocks), dim3(kThreads), 0, s, tab, scale);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}
template <class P, class G, bool MASTER>
int step_all(const c3d_opt_tensor* t, int count, int bits, const Hyper& h, hipStream_t s) {
  constexpr int sp = sizeof(P), sg = sizeof(G);
  if (bits == 32) {
    constexpr int NP = MASTER ? 5 : 4, M = MASTER ? 72 : 88;
    const int slots[5] = {0, 1, 2, 3, 6}, bytes[5] = {sp, sg, 4, 4, 4};
    int sl[NP], by[NP];
    for (int i = 0; i < NP; ++i) sl[i] = slots[i], by[i] = bytes[i];
    return for_each_table<NP, M>(t, count, sl, by, kChunk, kBlock, [&](const Table<NP, M>& tab, uint32_t blocks) {
      hipLaunchKernelGGL((adamw_kernel<P, G, MASTER, M>), dim3(blocks), dim3(kThreads), 0, s, tab, h);
      C3D_CHECK_LAUNCH();
      return 0;
    });
  }
  constexpr int NP = MASTER ? 7 : 6, M = MASTER ? 56 : 64;
  const int slots[7] = {0, 1, 2, 3, 4, 5, 6}, bytes[7] = {sp, sg, 1, 1, -1, -1, 4};
  int sl[NP], by[NP];
  for (int i = 0; i < NP; ++i) sl[i] = slots[i], by[i] = bytes[i];
  return for_each_table<NP, M>(t, count, sl, by, kChunk, kBlock, [&](const Table<NP, M>& tab, uint32_t blocks) {
    hipLaunchKernelGGL((adamw8_kernel<P, G, MASTER, M>), dim3(blocks), dim3(kThreads), 0, s, tab, h);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}

int check_records(const c3d_opt_tensor* t, int count, uint32_t need) {
  C3D_REQUIRE(count >= 0 && (count == 0 || t), "tensor list: null");
  for (int i = 0; i < count; ++i) {
    C3D_REQUIRE(t[i].n >= 0, "tensor list: negative length");
    for (int s = 0; s < 7; ++s) C3D_REQUIRE(t[i].n == 0 || !(need >> s & 1) || t[i].ptr[s], "tensor list: null pointer");
  }
  return 0;
}

}  // namespace

extern "C" int c3d_opt_abi_sizes(int32_t* out2) {
  out2[0] = (int32_t)sizeof(c3d_opt_tensor);
  out2[1] = (int32_t)sizeof(c3d_adamw_desc);
  return 0;
}

extern "C" int64_t c3d_grad_norm_partials(const c3d_opt_tensor* t, int count) {
  int64_t parts = 0;
  for (int i = 0; i < count; ++i)
    for (int64_t at = 0; at < t[i].n; at += kMaxRecord) {
      const int64_t n = t[i].n - at < kMaxRecord ? t[i].n - at : kMaxRecord;
      parts += (n + kNormChunk - 1) / kNormChunk;
    }
  return parts;
}

extern "C" int c3d_grad_norm(const c3d_opt_tensor* t, int count, int type, double max_norm, double* partial, float* norm, float* scale,
                             c3d_stream stream) {
  if (int rc = check_records(t, count, 1u << 1)) return rc;
  C3D_REQUIRE(type >= 0 && type <= 2, "grad_norm: type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(max_norm >= 0.0, "grad_norm: max_norm is negative or not a number");
  C3D_REQUIRE(norm && scale, "grad_norm: null output");
  const int64_t parts = c3d_grad_norm_partials(t, count);
  C3D_REQUIRE(parts == 0 || partial, "grad_norm: null workspace");
  C3D_REQUIRE(parts < (int64_t)1 << 32, "grad_norm: too many elements");
  hipStream_t s = (hipStream_t)stream;
  if (int rc = type == 0 ? sumsq<float>(t, count, partial, s) : type == 1 ? sumsq<__bf16>(t, count, partial, s) : sumsq<_Float16>(t, count, partial, s))
    return rc;
  hipLaunchKernelGGL(grad_norm_fold_kernel, dim3(1), dim3(1024), 0, s, partial, parts, max_norm, norm, scale);
  C3D_CHECK_LAUNCH();
  return 0;
}

extern "C" int c3d_scale_tensors(const c3d_opt_tensor* t, int count, int type, const float* scale, c3d_stream stream) {
  if (int rc = check_records(t, count, 1u << 1)) return rc;
  C3D_REQUIRE(type >= 0 && type <= 2, "scale_tensors: type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(scale, "scale_tensors: null scale");
  hipStream_t s = (hipStream_t)stream;
  return type == 0 ? scale_all<float>(t, count, scale, s) : type == 1 ? scale_all<__bf16>(t, count, scale, s) : scale_all<_Float16>(t, count, scale, s);
}

extern "C" int c3d_adamw_step(const c3d_opt_tensor* t, int count, const c3d_adamw_desc* d, c3d_stream stream) {
  C3D_REQUIRE(d, "adamw: null descriptor");
  C3D_REQUIRE(d->state_bits == 32 || d->state_bits == 8, "adamw: state_bits is 32 or 8");
  C3D_REQUIRE(d->param_type >= 0 && d->param_type <= 2, "adamw: param_type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(d->grad_type == 0 || d->grad_type == d->param_type, "adamw: gradients are fp32 or of the parameters' type");
  C3D_REQUIRE(!(d->has_master && d->param_type == 0), "adamw: fp32 parameters have no master copy");
  C3D_REQUIRE(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0, "adamw: betas are in [0, 1)");
  C3D_REQUIRE(d->eps >= 0.0, "adamw: eps is negative");
  C3D_REQUIRE(d->step_dev || d->step >= 1, "adamw: step counts from 1");
  if (int rc = check_records(t, count, 0xfu | (d->state_bits == 8 ? 0x30u : 0u) | (d->has_master ? 0x40u : 0u))) return rc;
  Hyper h;
  h.beta1 = (float)d->beta1;
  h.omb1 = (float)(1.0 - d->beta1);
  h.beta2 = (float)d->beta2;
  h.omb2 = (float)(1.0 - d->beta2);
  h.eps = (float)d->eps;
  const double tt = (double)d->step;
  h.ln_b1 = log(d->beta1);               // beta 0: -inf, and 1 - 0^t = -expm1(-inf) = 1
  h.ln_b2 = log(d->beta2);
  h.decay = (float)(1.0 - d->lr * d->weight_decay);
  h.step_size = d->step >= 1 ? (float)(d->lr / -expm1(tt * h.ln_b1)) : 0.f;
  h.inv_root = d->step >= 1 ? (float)(1.0 / sqrt(-expm1(tt * h.ln_b2))) : 0.f;
  h.lr = d->lr;
  h.wd = d->weight_decay;
  h.lr_dev = d->lr_dev;
  h.step_dev = d->step_dev;
  h.grad_scale = d->grad_scale;
  h.seed = d->seed;
  h.step = (uint32_t)d->step;
  hipStream_t s = (hipStream_t)stream;
  const int bits = d->state_bits;
  if (d->param_type == 0) return step_all<float, float, false>(t, count, bits, h, s);
  if (d->param_type == 1) {
    if (d->grad_type == 0)
      return d->has_master ? step_all<__bf16, float, true>(t, count, bits, h, s) : step_all<__bf16, float, false>(t, count, bits, h, s);
    return d->has_master ? step_all<__bf16, __bf16, true>(t, count, bits, h, s) : step_all<__bf16, __bf16, false>(t, count, bits, h, s);
  }
  if (d->grad_type == 0)
    return d->has_master ? step_all<_Float16, float, true>(t, count, bits, h, s) : step_all<_Float16, float, false>(t, count, bits, h, s);
  return d->has_master ? step_all<_Float16, _Float16, true>(t, count, bits, h, s) : step_all<_Float16, _Float16, false>(t, count, bits, h, s);
}
