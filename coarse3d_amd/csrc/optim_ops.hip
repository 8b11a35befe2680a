// Operators over the many tensors of an optimiser: the global norm of the gradients, their clipping, and the AdamW step with
// states in 32 bits or in 8 bits.  All of them stream, and what bounds them is HBM.
//
// A call takes a host array of tensor records.  Records travel as kernel arguments (at most 4 KB a launch), so that nothing is
// copied to the device ahead of the launch and a captured launch carries its own table; each wave finds the record of its blocks by
// a vote of its lanes over the records' first blocks.
//
// AdamW (decoupled weight decay, step t, beta1 = b1, beta2 = b2):
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// The reference steps torch.optim.AdamW over all parameters (tasks/weak_segmentation/trainer.py:146-151).
#include <algorithm>
#include <type_traits>
#include "common.h"
#include "../../include/coarse3d_hip.h"

namespace {

constexpr int kThreads = 256, kNormThreads = 512;
constexpr int kBlock = C3D_ADAMW8_BLOCK;   // elements a wave of the step handles at a time (four a lane), and that share a scale
constexpr int64_t kMaxRecord = 1 << 30;    // longer tensors are cut into several records: 32-bit indices inside one
constexpr uint32_t kMaxBlocks = 1u << 25;  // blocks a launch: its threads stay below 2^32
constexpr uint32_t kUnaligned = 1u << 31;
// Blocks a wave has in flight together.  Short waves: there are several generations of them on a CU, so that some load while others
// compute; with twice or four times as many blocks a wave all of them ran in step (9.4 M parameters, 8-bit states: 48 us with 1,
// 51 with 2, 66 with 4; 32-bit ones with the norm: 74, 74, 80).  The norm and the scaling, which compute nothing, want 4 KB a wave
// (38 MB: 30 us with 4 KB, 31 with 2, 33 with 8).
constexpr int kStepBlocks = 2, kStep8Blocks = 1, kNormBlocks = 4, kScaleBlocks = 2, kSmallBlocks = 4;

// The tensors of a launch, as one sequence of blocks: workgroups are dealt blocks and not tensors, so that a hundred biases of 32
// elements cost a hundred waves' loads and not a hundred workgroups.
template <int MAXT>
struct TableHead {
  uint32_t n[MAXT];         // elements; top bit: some pointer is not on the vector grid
  uint32_t first[MAXT];     // first block of the record
  uint32_t count, blocks;   // records; blocks of all of them
  uint32_t before;          // blocks of the launches ahead
};
// pointers as they are: any tensors
template <int NP, int MAXT>
struct Table : TableHead<MAXT> {
  static constexpr int kPointers = NP, kMost = MAXT;
  void* ptr[NP][MAXT];
  __device__ __forceinline__ char* at(int s, int k) const { return static_cast<char*>(ptr[s][k]); }
};
// pointers as 32-bit distances from the lowest of their list, in units of 4 bytes (codes, scales) or 16: nearly twice the tensors in a
// launch (a launch more costs 4 us of a step of 45)
template <int NP, int MAXT>
struct PackedTable : TableHead<MAXT> {
  static constexpr int kPointers = NP, kMost = MAXT;
  char* base[NP];
  uint32_t shift[NP];
  uint32_t off[NP][MAXT];
  __device__ __forceinline__ char* at(int s, int k) const { return base[s] + ((uint64_t)off[s][k] << shift[s]); }
};

using GradTable = Table<1, 240>;

// the record that holds a block (below t.blocks): every lane looks at one record's first block, and the vote counts those at or ahead of
// it -- one load's latency, where a binary search waits for seven loads in turn
template <int MAXT>
__device__ __forceinline__ int find_record(const TableHead<MAXT>& t, uint32_t block) {
  const uint32_t lane = threadIdx.x & 63;
  int k = -1;
#pragma unroll
  for (uint32_t at = 0; at < MAXT; at += 64) {
    const uint32_t i = at + lane;
    k += __popcll(__builtin_amdgcn_ballot_w64(i < t.count && t.first[i < MAXT ? i : MAXT - 1] <= block));
  }
  return k;
}
// number of this wave, in a scalar register: what follows from it (record, pointers) is read through scalar loads
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x / 64) + (threadIdx.x >> 6)); }

template <class T, int V = 4>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};
template <int BYTES>
struct Bits;
template <>
struct Bits<16> {
  typedef uint32_t type __attribute__((ext_vector_type(4)));
};
template <>
struct Bits<8> {
  typedef uint32_t type __attribute__((ext_vector_type(2)));
};
template <>
struct Bits<4> {
  typedef uint32_t type;
};
// V consecutive elements from i: FULL in one access, else one by one and 0 past n.  Left in their own type, so that a load is not
// waited for before its first use.  LAST (the step, loads and stores): nothing reads them again before other gigabytes have passed, so
// they go past the caches (9.4 M parameters, 32-bit states with the norm: 74 -> 67 us; 41 M, 8 bits: 170 -> 162)
template <bool FULL, class T, int V = 4, bool LAST = false>
__device__ __forceinline__ Vec<T, V> loadv(const void* base, uint32_t i, uint32_t n) {
  const T* p = static_cast<const T*>(base);
  if constexpr (FULL && LAST) {
    using B = typename Bits<sizeof(Vec<T, V>)>::type;
    return __builtin_bit_cast(Vec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const B*>(p + i)));
  }
  if constexpr (FULL) return *reinterpret_cast<const Vec<T, V>*>(p + i);
  Vec<T, V> r;
#pragma unroll
  for (int q = 0; q < V; ++q) r.v[q] = i + q < n ? p[i + q] : (T)0;
  return r;
}
template <bool FULL, class T, int V = 4, bool LAST = false>
__device__ __forceinline__ void storev(void* base, uint32_t i, uint32_t n, const float (&x)[V]) {
  T* p = static_cast<T*>(base);
  if constexpr (FULL) {
    Vec<T, V> r;
#pragma unroll
    for (int q = 0; q < V; ++q) r.v[q] = (T)x[q];
    if constexpr (LAST) {
      using B = typename Bits<sizeof(r)>::type;
      __builtin_nontemporal_store(__builtin_bit_cast(B, r), reinterpret_cast<B*>(p + i));
      return;
    }
    *reinterpret_cast<Vec<T, V>*>(p + i) = r;
  } else {
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (i + q < n) p[i + q] = (T)x[q];
  }
}
// The master's value as it is stored: without this the compiler folds the last fp32 operation and the conversion to fp16 into one
// instruction that rounds once, and the parameter is not always its master rounded
__device__ __forceinline__ void as_stored(float (&x)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) asm("" : "+v"(x[q]));
}
// four 8-bit codes, the first in the low byte
template <bool FULL>
__device__ __forceinline__ void store_codes(void* base, uint32_t i, uint32_t n, uint32_t c) {
  uint8_t* p = static_cast<uint8_t*>(base);
  if constexpr (FULL) {
    __builtin_nontemporal_store(c, reinterpret_cast<uint32_t*>(p + i));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < n) p[i + q] = (uint8_t)(c >> (8 * q));
  }
}

// A wave's NB blocks, from number j: where they lie in one record, on the 4-element grid and ahead of its end (all but the last of a
// tensor, as a rule), `full` takes them together, without a branch between their loads; what it leaves (bits of its result), and
// every block elsewhere, `part` takes one by one.
template <int NB, uint32_t BLOCK, class TB, class F, class G>
__device__ __forceinline__ void wave_blocks(const TB& t, uint32_t j, F full, G part) {
  if (j >= t.blocks) return;
  int k = find_record(t, j);
  const uint32_t n = t.n[k], b = j - t.first[k];
  uint32_t left = (1u << NB) - 1;
  if (!(n & kUnaligned) && (uint64_t)(b + NB) * BLOCK <= n) left = full(k, b);
#pragma unroll 1
  for (; left && j < t.blocks; left >>= 1, ++j) {
    while (k + 1 < (int)t.count && t.first[k + 1] <= j) ++k;
    if (left & 1u) part(k, j - t.first[k]);
  }
}

// ---------------------------------------------------------------- norm and clipping

// sum over a workgroup in a fixed order, the same in every thread
template <int THREADS>
__device__ __forceinline__ double group_sum(double s, double* red) {
  s = c3d_wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) s += red[w];
  return s;
}

template <class T>
constexpr int kLane = 16 / sizeof(T);                  // elements a lane of the norm and of the scaling takes: 16 bytes
template <class T>
constexpr int kRun = 64 * kLane<T>;                    // and a wave: their block

// squares and sums in 64 bits (as many a clock as in 32 here): no gradient overflows, and the factor that other roundings depend on
// is the same whatever the order of the sum.  One partial sum a workgroup.  38 MB: 13 us, 4 of them the launch's own.
template <class T, class TB>
__global__ __launch_bounds__(kNormThreads) void grad_sumsq_kernel(TB t, double* __restrict__ partial) {
  constexpr int V = kLane<T>, B = kRun<T>;
  __shared__ double red[kNormThreads / 64];
  const uint32_t lane = threadIdx.x & 63;
  double s = 0.0;
  auto add = [&](const Vec<T, V>& x) {
#pragma unroll
    for (int q = 0; q < V; ++q) s = fma((double)(float)x.v[q], (double)(float)x.v[q], s);
  };
  wave_blocks<kNormBlocks, B>(
      t, wave_id() * kNormBlocks,
      [&](int k, uint32_t b) {
        Vec<T, V> x[kNormBlocks];
#pragma unroll
        for (int u = 0; u < kNormBlocks; ++u) x[u] = loadv<true, T, V>(t.at(0, k), (b + u) * B + lane * V, 0);
#pragma unroll
        for (int u = 0; u < kNormBlocks; ++u) add(x[u]);
        return 0u;
      },
      [&](int k, uint32_t b) { add(loadv<false, T, V>(t.at(0, k), b * B + lane * V, t.n[k] & ~kUnaligned)); });
  s = group_sum<kNormThreads>(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void grad_norm_fold_kernel(const double* __restrict__ partial, int64_t n, double max_norm,
                                                             float* __restrict__ norm, float* __restrict__ scale) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = group_sum<1024>(s, red);
  if (threadIdx.x == 0) {
    const double r = sqrt(s), f = max_norm / (r + 1e-6);
    *norm = (float)r;
    *scale = (float)(f > 1.0 ? 1.0 : f);          // a norm that is not a number stays visible in the factor
  }
}

// Everything in one workgroup and one launch, where all values fit its registers: each wave holds kSmallBlocks blocks of 16 bytes a
// lane.  (Clipping 16 K values: 7 us, 12 in three launches; with four times the blocks a wave it loses, 18 us.)
template <class T, bool CLIP>
__global__ __launch_bounds__(1024) void grad_small_kernel(GradTable t, double max_norm, float* __restrict__ norm, float* __restrict__ scale) {
  constexpr int V = kLane<T>, B = kRun<T>;
  __shared__ double red[16];
  const uint32_t lane = threadIdx.x & 63, wave = wave_id();
  Vec<T, V> x[kSmallBlocks];
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < kSmallBlocks; ++u) {
    const uint32_t j = u * 16 + wave;
#pragma unroll
    for (int q = 0; q < V; ++q) x[u].v[q] = (T)0;
    if (j < t.blocks) {
      const int k = find_record(t, j);
      const uint32_t n = t.n[k] & ~kUnaligned, b = j - t.first[k], i = b * B + lane * V;
      if (!(t.n[k] & kUnaligned) && (b + 1) * B <= n) x[u] = loadv<true, T, V>(t.at(0, k), i, n);
      else x[u] = loadv<false, T, V>(t.at(0, k), i, n);
    }
  }
#pragma unroll
  for (int u = 0; u < kSmallBlocks; ++u)
#pragma unroll
    for (int q = 0; q < V; ++q) s = fma((double)(float)x[u].v[q], (double)(float)x[u].v[q], s);
  s = group_sum<1024>(s, red);
  const double r = sqrt(s), f = max_norm / (r + 1e-6);
  const float factor = (float)(f > 1.0 ? 1.0 : f);
  if (threadIdx.x == 0) {
    *norm = (float)r;
    *scale = factor;
  }
  if constexpr (CLIP) {
#pragma unroll
    for (int u = 0; u < kSmallBlocks; ++u) {
      const uint32_t j = u * 16 + wave;
      if (j < t.blocks) {
        const int k = find_record(t, j);
        const uint32_t n = t.n[k] & ~kUnaligned, b = j - t.first[k], i = b * B + lane * V;
        float o[V];
#pragma unroll
        for (int q = 0; q < V; ++q) o[q] = (float)x[u].v[q] * factor;
        if (!(t.n[k] & kUnaligned) && (b + 1) * B <= n) storev<true, T, V>(t.at(0, k), i, n, o);
        else storev<false, T, V>(t.at(0, k), i, n, o);
      }
    }
  }
}

// (Adding up the partial sums in here instead, in every workgroup, spares a launch and gains nothing: 31 us either way at 38 MB.)
template <class T, class TB>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(TB t, const float* __restrict__ scale) {
  constexpr int V = kLane<T>, B = kRun<T>;
  const uint32_t lane = threadIdx.x & 63;
  const float f = *scale;
  auto scaled = [&](const Vec<T, V>& x, float (&r)[V]) {
#pragma unroll
    for (int q = 0; q < V; ++q) r[q] = (float)x.v[q] * f;
  };
  wave_blocks<kScaleBlocks, B>(
      t, wave_id() * kScaleBlocks,
      [&](int k, uint32_t b) {
        Vec<T, V> x[kScaleBlocks];
#pragma unroll
        for (int u = 0; u < kScaleBlocks; ++u) x[u] = loadv<true, T, V>(t.at(0, k), (b + u) * B + lane * V, 0);
#pragma unroll
        for (int u = 0; u < kScaleBlocks; ++u) {
          float r[V];
          scaled(x[u], r);
          storev<true, T, V>(t.at(0, k), (b + u) * B + lane * V, 0, r);
        }
        return 0u;
      },
      [&](int k, uint32_t b) {
        const uint32_t i = b * B + lane * V, n = t.n[k] & ~kUnaligned;
        float r[V];
        scaled(loadv<false, T, V>(t.at(0, k), i, n), r);
        storev<false, T, V>(t.at(0, k), i, n, r);
      });
}

// ---------------------------------------------------------------- AdamW

struct Hyper {
  float beta1, omb1, beta2, omb2, eps;
  float decay, step_size, inv_root;       // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  double lr, wd, ln_b1, ln_b2;
  double b1, o1, b2, o2;                  // beta, 1 - beta in 64 bits: what decides an 8-bit code
  const float* lr_dev;                    // not null: the learning rate / the step count are read on the device
  const float* step_dev;
  const float* grad_scale;
  uint32_t seed, step;
};

// sqrt to one unit in the last place (the instruction's own accuracy); it does not take numbers below 2^-126, so small ones are moved up
__device__ __forceinline__ float fast_sqrt(float v) {
  const bool low = v < 0x1p-96f;
  const float s = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v);
  return low ? s * 0x1p-32f : s;
}

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

// 28 bytes an fp32 element and some 20 operations: bound by HBM, 9.4 M parameters 52 us = 5.1 TB/s in two launches.
template <class P, class G, bool MASTER, class TB>
__global__ __launch_bounds__(kThreads) void adamw_kernel(TB t, Hyper h) {
  using W = std::conditional_t<MASTER, float, P>;       // what carries the parameter's value
  constexpr int kValue = MASTER ? 4 : 0;
  const uint32_t lane = threadIdx.x & 63;
  struct Regs {
    Vec<W> p;
    Vec<G> g;
    Vec<float> m, v;
  };
  auto load = [&](auto full, int k, uint32_t i, uint32_t n, Regs& r) {
    constexpr bool F = decltype(full)::value;
    r.p = loadv<F, W, 4, true>(t.at(kValue, k), i, n);
    r.g = loadv<F, G, 4, true>(t.at(1, k), i, n);
    r.m = loadv<F, float, 4, true>(t.at(2, k), i, n);
    r.v = loadv<F, float, 4, true>(t.at(3, k), i, n);
  };
  float decay, step_size, inv_root, gs;
  auto step = [&](auto full, int k, uint32_t i, uint32_t n, const Regs& r) {
    constexpr bool F = decltype(full)::value;
    float p[4], m[4], v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = (float)r.g.v[q] * gs;
      m[q] = r.m.v[q] * h.beta1 + x * h.omb1;
      v[q] = r.v.v[q] * h.beta2 + (x * x) * h.omb2;
      p[q] = (float)r.p.v[q] * decay - step_size * (m[q] * __builtin_amdgcn_rcpf(fast_sqrt(v[q]) * inv_root + h.eps));
    }
    storev<F, float, 4, true>(t.at(2, k), i, n, m);
    storev<F, float, 4, true>(t.at(3, k), i, n, v);
    if constexpr (MASTER) {
      as_stored(p);
      storev<F, float, 4, true>(t.at(kValue, k), i, n, p);
    }
    storev<F, P, 4, true>(t.at(0, k), i, n, p);
  };
  auto scalars = [&]() {
    uint32_t count;
    resolve(h, decay, step_size, inv_root, count);
    gs = h.grad_scale ? *h.grad_scale : 1.f;
  };
  wave_blocks<kStepBlocks, kBlock>(
      t, wave_id() * kStepBlocks,
      [&](int k, uint32_t b) {
        Regs r[kStepBlocks];
#pragma unroll
        for (int u = 0; u < kStepBlocks; ++u) load(std::true_type(), k, (b + u) * kBlock + lane * 4, 0, r[u]);
        scalars();
#pragma unroll
        for (int u = 0; u < kStepBlocks; ++u) step(std::true_type(), k, (b + u) * kBlock + lane * 4, 0, r[u]);
        return 0u;
      },
      [&](int k, uint32_t b) {
        const uint32_t i = b * kBlock + lane * 4, n = t.n[k] & ~kUnaligned;
        Regs r;
        load(std::false_type(), k, i, n, r);
        scalars();
        step(std::false_type(), k, i, n, r);
      });
}

// ---------------------------------------------------------------- AdamW with states in 8 bits
//
// A block of 256 elements keeps m and r = sqrt(v) as e4m3 numbers times one power of two each, such that the block's largest value
// is in (224, 448].  r and not v: the root halves the exponent's range, so that m and r reach equally far below their block's
// largest value (2^-17.8) and m / r stays bounded; r > 0 is never stored as 0 for the same reason.  A power of two: products with
// it are exact.  Rounding is stochastic (16 bits an element, a hash of seed, step and the element's number): v moves by
// 1 - b2 = 0.1 % a step, which is less than half a code step, and rounding to nearest would freeze it.
//
// 16 bytes an fp32 element, some 60 instructions: 41 M bf16 parameters with masters 136 us = 4.8 TB/s, 9.4 M fp32 ones 41 us = 3.7 TB/s
// in two launches of about 4 us of their own each.

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

// a = |x| * 2^-k -> e4m3 code by stochastic rounding.  The upper word of a double holds 20 mantissa bits: the code's three and 17
// below them, to whose upper 16 the random bits are added; what lies in the lower word cannot change the carry.  Below the smallest
// normal number 2^-6 the value is moved up by 2^-6, which puts the code's last bit at the same place.
__device__ __forceinline__ uint32_t e4m3_code(double a, uint32_t rnd16) {
  const bool low = (uint32_t)__double2hiint(a) < (uint32_t)(1023 - 6) << 20;
  const uint32_t hi = (uint32_t)__double2hiint(low ? a + 0x1p-6 : a);
  const uint32_t c = ((hi + (rnd16 << 1)) >> 17) - (low ? (1023u - 6u) * 8u : (1023u - 7u) * 8u);
  return c > 0x7eu ? 0x7eu : c;
}

// the same for r = sqrt(vmax) without the root: r = f 2^e, and f > 1.75 where vmax is more than 3.0625 4^e (the rounding of the root to
// fp32 moves nothing across: the square of the middle between 1.75 and its neighbour lies between 3.0625 and its neighbour)
__device__ __forceinline__ int scale_exponent_of_root(uint32_t vmax) {
  const int e2 = (int)(vmax >> 23) - 127, e = e2 >> 1;
  const int k = e - 8 + ((e2 & 1) && (vmax & 0x7fffffu) > 0x440000u ? 1 : 0);
  return k < -100 || vmax == 0 ? -100 : k;
}
// largest of the 64 lanes' numbers, as a scalar: four steps inside rows of sixteen lanes, two across rows, all in the VALU
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define C3D_MAX_STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
  C3D_MAX_STEP(0x111, 0xf);      // row_shr:1, 2, 4, 8: lane 15 of a row has the row's
  C3D_MAX_STEP(0x112, 0xf);
  C3D_MAX_STEP(0x114, 0xf);
  C3D_MAX_STEP(0x118, 0xf);
  C3D_MAX_STEP(0x142, 0xa);      // row_bcast:15 into rows 1 and 3
  C3D_MAX_STEP(0x143, 0xc);      // row_bcast:31 into rows 2 and 3: lane 63 has all
#undef C3D_MAX_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

template <class P, class G, bool MASTER, class TB>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(TB t, Hyper h) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  using W = std::conditional_t<MASTER, float, P>;
  constexpr int kValue = MASTER ? 6 : 0;
  const uint32_t lane = threadIdx.x & 63;
  struct Regs {
    Vec<W> p;
    Vec<G> g;
    uint32_t mc, rc;
    float ms, rs;
  };
  auto load = [&](auto full, int k, uint32_t b, uint32_t n, Regs& r) {
    constexpr bool F = decltype(full)::value;
    const uint32_t i = b * kBlock + lane * 4;
    r.p = loadv<F, W, 4, true>(t.at(kValue, k), i, n);
    r.g = loadv<F, G, 4, true>(t.at(1, k), i, n);
    r.mc = __builtin_bit_cast(uint32_t, loadv<F, uint8_t, 4, true>(t.at(2, k), i, n));
    r.rc = __builtin_bit_cast(uint32_t, loadv<F, uint8_t, 4, true>(t.at(3, k), i, n));
    r.ms = reinterpret_cast<const float*>(t.at(4, k))[b];
    r.rs = reinterpret_cast<const float*>(t.at(5, k))[b];
  };
  float decay, step_size, inv_root, gs;
  uint32_t key;
  auto scalars = [&]() {
    uint32_t count;
    resolve(h, decay, step_size, inv_root, count);
    gs = h.grad_scale ? *h.grad_scale : 1.f;
    key = mix32(h.seed + count * 0x9E3779B9u);
  };
  auto step = [&](int k, uint32_t b, uint32_t n, const Regs& r) {
    const uint32_t i = b * kBlock + lane * 4;
    const f32x2_t m01 = __builtin_amdgcn_cvt_pk_f32_fp8(r.mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(r.mc, true);
    const f32x2_t r01 = __builtin_amdgcn_cvt_pk_f32_fp8(r.rc, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8(r.rc, true);
    const float mo[4] = {m01[0], m01[1], m23[0], m23[1]}, ro[4] = {r01[0], r01[1], r23[0], r23[1]};
    double md[4], rd[4];
    float p[4], m32[4], v32[4];
    uint32_t mmax = 0, vmax = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma clang fp contract(off)
      // in 32 bits, each operation rounded: the parameter's step and the block's scale
      const float x = (float)r.g.v[q] * gs, old_m = mo[q] * r.ms, old_r = ro[q] * r.rs;
      m32[q] = old_m * h.beta1 + x * h.omb1;
      v32[q] = (old_r * old_r) * h.beta2 + (x * x) * h.omb2;
      const float s = fast_sqrt(v32[q]);
      p[q] = fmaf(-step_size, m32[q] * __builtin_amdgcn_rcpf(fmaf(s, inv_root, h.eps)), (float)r.p.v[q] * decay);
      // in 64 bits: what is stored.  Rounding twice would move values that lie next to the border between two codes; the root gets
      // one Newton step, which leaves it 45 bits
      const double xd = x, od = old_r;
      md[q] = fma((double)old_m, h.b1, xd * h.o1);
      const double vd = fma(od * od, h.b2, (xd * xd) * h.o2), sd = s;
      const float e = (float)fma(-sd, sd, vd);
      rd[q] = sd + (double)(s > 0.f ? e * (0.5f * __builtin_amdgcn_rcpf(s)) : 0.f);
      // magnitudes order like their bits; what is not finite does not count
      const uint32_t mb = __float_as_uint(m32[q]) & 0x7fffffffu, vb = __float_as_uint(v32[q]);
      mmax = mb < 0x7f800000u ? max(mmax, mb) : mmax;
      vmax = vb < 0x7f800000u ? max(vmax, vb) : vmax;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      mmax = max(mmax, (uint32_t)__shfl_xor((int)mmax, o, 64));
      vmax = max(vmax, (uint32_t)__shfl_xor((int)vmax, o, 64));
    }
    const int mk = scale_exponent(mmax), rk = scale_exponent(__float_as_uint(sqrtf(__uint_as_float(vmax))));
    const double minv = pow2(-mk), rinv = pow2(-rk);
    uint32_t rnd = mix32(key + (t.before + t.first[k] + b) * (kBlock / 4) + lane);
    uint32_t mc = 0, rc = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t mb = __float_as_uint(m32[q]), vb = __float_as_uint(v32[q]);
      uint32_t cm = e4m3_code(fabs(md[q]) * minv, rnd & 0xffffu);
      uint32_t cr = e4m3_code(rd[q] * rinv, rnd >> 16);
      if (cr == 0u && v32[q] > 0.f) cr = 1u;
      if ((mb & 0x7fffffffu) >= 0x7f800000u) cm = 0x7fu;
      if ((vb & 0x7fffffffu) >= 0x7f800000u) cr = 0x7fu;
      mc |= (cm | ((mb >> 24) & 0x80u)) << (8 * q);
      rc |= cr << (8 * q);
      rnd = shift_register(rnd);
    }
    store_codes<false>(t.at(2, k), i, n, mc);
    store_codes<false>(t.at(3, k), i, n, rc);
    if (lane == 0) {
      reinterpret_cast<float*>(t.at(4, k))[b] = pow2(mk);
      reinterpret_cast<float*>(t.at(5, k))[b] = pow2(rk);
    }
    if constexpr (MASTER) {
      as_stored(p);
      storev<false, float>(t.at(kValue, k), i, n, p);
    }
    storev<false, P>(t.at(0, k), i, n, p);
  };
  // The same result in about half the instructions, for whole blocks without anything special in them; false: nothing was written,
  // take `step`.  Everything is computed in 32 bits and the codes come from the conversion instruction that rounds stochastically (it
  // adds the upper 20 of its random bits below the last kept one); what comes too near the border between two codes for 32 bits to
  // tell (about one block in a hundred) is left to `step`, with what is not finite and roots that are all but zero.
  auto quick = [&](int k, uint32_t b, const Regs& r) -> bool {
#pragma clang fp contract(off)
    const uint32_t i = b * kBlock + lane * 4;
    const f32x2_t m01 = __builtin_amdgcn_cvt_pk_f32_fp8(r.mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(r.mc, true);
    const f32x2_t r01 = __builtin_amdgcn_cvt_pk_f32_fp8(r.rc, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8(r.rc, true);
    const float mo[4] = {m01[0], m01[1], m23[0], m23[1]}, ro[4] = {r01[0], r01[1], r23[0], r23[1]};
    const float c1 = r.ms * h.beta1, c2 = (r.rs * r.rs) * h.beta2;        // powers of two: the products round as they do one by one
    float p[4], m[4], v[4], s[4];
    float mtop = 0.f, vtop = 0.f;
    bool odd = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = (float)r.g.v[q] * gs;
      m[q] = mo[q] * c1 + x * h.omb1;
      v[q] = (ro[q] * ro[q]) * c2 + (x * x) * h.omb2;
      s[q] = __builtin_amdgcn_sqrtf(v[q]);
      p[q] = fmaf(-step_size, m[q] * __builtin_amdgcn_rcpf(fmaf(s[q], inv_root, h.eps)), (float)r.p.v[q] * decay);
      mtop = fmaxf(mtop, fabsf(m[q]));
      vtop = fmaxf(vtop, v[q]);
      odd = odd || __builtin_isunordered(m[q], v[q]);
    }
    const uint32_t mmax = wave_max(__float_as_uint(mtop)), vmax = wave_max(__float_as_uint(vtop));
    const int mk = scale_exponent(mmax), rk = scale_exponent_of_root(vmax);
    const float minv = pow2(-mk), rinv = pow2(-rk);
    uint32_t rnd = mix32(key + (t.before + t.first[k] + b) * (kBlock / 4) + lane);
    uint32_t mc = 0, rc = 0, near_m = ~0u, near_r = ~0u;
#define C3D_CODES(q)                                                                                                        \
  {                                                                                                                        \
    const float a = m[q] * minv, z = __builtin_amdgcn_fmed3f(s[q] * rinv, v[q] > 0.f ? 0x1p-9f : 0.f, 448.f);              \
    const uint32_t um = rnd << 16, ur = rnd & 0xffff0000u;                                                                 \
    mc = __builtin_amdgcn_cvt_sr_fp8_f32(a, um, mc, q);                                                                    \
    rc = __builtin_amdgcn_cvt_sr_fp8_f32(z, ur, rc, q);                                                                    \
    near_m = min(near_m, (__float_as_uint(a) + (um >> 12) + 16u) & 0xfffffu);                                              \
    near_r = min(near_r, (__float_as_uint(z) + (ur >> 12) + 8u) & 0xfffffu);                                               \
    rnd = shift_register(rnd);                                                                                             \
  }
    C3D_CODES(0) C3D_CODES(1) C3D_CODES(2) C3D_CODES(3)
#undef C3D_CODES
    odd = odd || near_m <= 32u || near_r <= 16u;
    if (__builtin_amdgcn_ballot_w64(odd) || mmax >= 0x7f800000u || vmax >= 0x7f800000u || (vmax < 0x12800000u && vmax != 0u) || h.eps == 0.f) return false;
    store_codes<true>(t.at(2, k), i, 0, mc);
    store_codes<true>(t.at(3, k), i, 0, rc);
    if (lane == 0) {
      reinterpret_cast<float*>(t.at(4, k))[b] = pow2(mk);
      reinterpret_cast<float*>(t.at(5, k))[b] = pow2(rk);
    }
    if constexpr (MASTER) {
      as_stored(p);
      storev<true, float, 4, true>(t.at(kValue, k), i, 0, p);
    }
    storev<true, P, 4, true>(t.at(0, k), i, 0, p);
    return true;
  };
  wave_blocks<kStep8Blocks, kBlock>(
      t, wave_id() * kStep8Blocks,
      [&](int k, uint32_t b) {
        Regs r[kStep8Blocks];
#pragma unroll
        for (int u = 0; u < kStep8Blocks; ++u) load(std::true_type(), k, b + u, 0, r[u]);
        scalars();
        uint32_t left = 0;
#pragma unroll
        for (int u = 0; u < kStep8Blocks; ++u) left |= quick(k, b + u, r[u]) ? 0u : 1u << u;
        return left;
      },
      [&](int k, uint32_t b) {
        const uint32_t n = t.n[k] & ~kUnaligned;
        Regs r;
        load(std::false_type(), k, b, n, r);
        scalars();
        step(k, b, n, r);
      });
}

// ---------------------------------------------------------------- host side

// How a list's pointers lie: bytes of an element (negative: a scale, one for each kBlock elements) and the field of c3d_opt_tensor
struct Slot {
  int field, bytes;
  int shift() const { return bytes < 0 || bytes == 1 ? 2 : 4; }
};

// Walks the records in tables of at most TB::kMost and hands each to `launch(table, groups)`.  block: elements; group: blocks a workgroup
template <class TB, class F>
int for_each_table(const c3d_opt_tensor* t, int count, const Slot (&slots)[TB::kPointers], uint32_t block, uint32_t group, F launch) {
  constexpr int NP = TB::kPointers;
  TB tab;
  static_assert(sizeof(tab) <= 4096 - sizeof(Hyper), "kernel arguments");
  tab.count = tab.blocks = tab.before = 0;
  if constexpr (std::is_same_v<TB, PackedTable<NP, TB::kMost>>)
    for (int s = 0; s < NP; ++s) {
      uintptr_t lo = UINTPTR_MAX;
      for (int i = 0; i < count; ++i)
        if (t[i].n) lo = std::min(lo, reinterpret_cast<uintptr_t>(t[i].ptr[slots[s].field]));
      tab.base[s] = reinterpret_cast<char*>(lo);
      tab.shift[s] = slots[s].shift();
    }
  auto flush = [&]() {
    const int rc = tab.count ? launch(tab, (tab.blocks + group - 1) / group) : 0;
    tab.before += tab.blocks;             // modulo 2^32, as the numbers that come of it
    tab.count = tab.blocks = 0;
    return rc;
  };
  for (int i = 0; i < count; ++i) {
    for (int64_t at = 0; at < t[i].n; at += kMaxRecord) {
      const uint32_t n = (uint32_t)(t[i].n - at < kMaxRecord ? t[i].n - at : kMaxRecord);
      const uint32_t nb = (n + block - 1) / block;
      if (tab.count == TB::kMost || tab.blocks + nb > kMaxBlocks)
        if (int rc = flush()) return rc;
      const uint32_t c = tab.count++;
      tab.n[c] = n;
      for (int s = 0; s < NP; ++s) {
        const int bytes = slots[s].bytes;
        // a scale moves with the block, everything else with the element
        char* p = static_cast<char*>(t[i].ptr[slots[s].field]) + (bytes < 0 ? at / kBlock * 4 : at * bytes);
        if (bytes > 0 && (reinterpret_cast<uintptr_t>(p) & (block / 64 * bytes - 1))) tab.n[c] |= kUnaligned;
        if constexpr (std::is_same_v<TB, PackedTable<NP, TB::kMost>>) tab.off[s][c] = (uint32_t)((uint64_t)(p - tab.base[s]) >> tab.shift[s]);
        else tab.ptr[s][c] = p;
      }
      tab.first[c] = tab.blocks;
      tab.blocks += nb;
    }
  }
  return flush();
}

// whether every distance of every list fits PackedTable
template <int NP>
bool packable(const c3d_opt_tensor* t, int count, const Slot (&slots)[NP]) {
  for (int s = 0; s < NP; ++s) {
    uintptr_t lo = UINTPTR_MAX, hi = 0, first = 0;
    uintptr_t off = 0;
    for (int i = 0; i < count; ++i) {
      if (!t[i].n) continue;
      const uintptr_t p = reinterpret_cast<uintptr_t>(t[i].ptr[slots[s].field]);
      if (!hi) first = p;
      off |= p ^ first;
      lo = std::min(lo, p);
      hi = std::max(hi, p + (uintptr_t)(slots[s].bytes < 0 ? t[i].n / kBlock * 4 : t[i].n * slots[s].bytes));
    }
    const int sh = slots[s].shift();
    if ((off & ((1u << sh) - 1)) || (hi > lo && ((hi - lo) >> sh) > UINT32_MAX)) return false;
  }
  return true;
}

template <class T, class F>
int for_each_grad_table(const c3d_opt_tensor* t, int count, int blocks_a_group, F launch) {
  return for_each_table<GradTable>(t, count, {{1, (int)sizeof(T)}}, kRun<T>, blocks_a_group, launch);
}
constexpr int kNormGroup = kNormBlocks * kNormThreads / 64, kScaleGroup = kScaleBlocks * kThreads / 64;
// the whole list in one table and in one workgroup's registers?
template <class T>
bool is_small(const c3d_opt_tensor* t, int count) {
  static_assert(16 * kSmallBlocks <= GradTable::kMost, "a tensor has a block at least");
  int64_t blocks = 0;
  for (int i = 0; i < count && blocks <= 16 * kSmallBlocks; ++i) blocks += (t[i].n + kRun<T> - 1) / kRun<T>;
  return blocks > 0 && blocks <= 16 * kSmallBlocks;
}
template <class T>
int small(const c3d_opt_tensor* t, int count, bool clip, double max_norm, float* norm, float* scale, hipStream_t s) {
  return for_each_grad_table<T>(t, count, 16 * kSmallBlocks, [&](const GradTable& tab, uint32_t) {
    const auto kernel = clip ? grad_small_kernel<T, true> : grad_small_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(1024), 0, s, tab, max_norm, norm, scale);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}
template <class T>
int sumsq(const c3d_opt_tensor* t, int count, double* partial, hipStream_t s) {
  return for_each_grad_table<T>(t, count, kNormGroup, [&](const GradTable& tab, uint32_t groups) {
    hipLaunchKernelGGL((grad_sumsq_kernel<T, GradTable>), dim3(groups), dim3(kNormThreads), 0, s, tab, partial);
    C3D_CHECK_LAUNCH();
    partial += groups;          // one partial sum a workgroup
    return 0;
  });
}
template <class T>
int scale_all(const c3d_opt_tensor* t, int count, const float* scale, hipStream_t s) {
  return for_each_grad_table<T>(t, count, kScaleGroup, [&](const GradTable& tab, uint32_t groups) {
    hipLaunchKernelGGL((grad_scale_kernel<T, GradTable>), dim3(groups), dim3(kThreads), 0, s, tab, scale);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}
template <class P, class G, bool MASTER, bool EIGHT, class TB>
int step_tables(const c3d_opt_tensor* t, int count, const Slot (&slots)[TB::kPointers], const Hyper& h, hipStream_t s) {
  return for_each_table<TB>(t, count, slots, kBlock, (EIGHT ? kStep8Blocks : kStepBlocks) * kThreads / 64, [&](const TB& tab, uint32_t groups) {
    if constexpr (EIGHT) hipLaunchKernelGGL((adamw8_kernel<P, G, MASTER, TB>), dim3(groups), dim3(kThreads), 0, s, tab, h);
    else hipLaunchKernelGGL((adamw_kernel<P, G, MASTER, TB>), dim3(groups), dim3(kThreads), 0, s, tab, h);
    C3D_CHECK_LAUNCH();
    return 0;
  });
}
// The table that takes all tensors in fewer launches, where there is a difference and the addresses allow it
template <class P, class G, bool MASTER, bool EIGHT>
int step_slots(const c3d_opt_tensor* t, int count, const Hyper& h, hipStream_t s) {
  constexpr int sp = sizeof(P), sg = sizeof(G), NP = (EIGHT ? 6 : 4) + MASTER, sm = EIGHT ? 1 : 4;
  constexpr int kArgs = 4096 - sizeof(Hyper) - 16;
  constexpr int kWide = kArgs / (8 * NP + 8), kPacked = (kArgs - 12 * NP - 8) / (4 * NP + 8);
  Slot slots[NP] = {{0, sp}, {1, sg}, {2, sm}, {3, sm}};
  if (EIGHT) slots[4 % NP] = {4, -1}, slots[5 % NP] = {5, -1};
  if (MASTER) slots[NP - 1] = {6, 4};
  if (count > kWide && packable<NP>(t, count, slots)) return step_tables<P, G, MASTER, EIGHT, PackedTable<NP, kPacked>>(t, count, slots, h, s);
  return step_tables<P, G, MASTER, EIGHT, Table<NP, kWide>>(t, count, slots, h, s);
}
template <class P, class G, bool MASTER>
int step_all(const c3d_opt_tensor* t, int count, int bits, const Hyper& h, hipStream_t s) {
  return bits == 8 ? step_slots<P, G, MASTER, true>(t, count, h, s) : step_slots<P, G, MASTER, false>(t, count, h, s);
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

extern "C" int64_t c3d_grad_norm_partials(const c3d_opt_tensor* t, int count, int type) {
  if (type == 0 ? is_small<float>(t, count) : is_small<_Float16>(t, count)) return 0;
  int64_t parts = 0;
  auto add = [&](const GradTable&, uint32_t groups) {
    parts += groups;
    return 0;
  };
  if (type == 0) for_each_grad_table<float>(t, count, kNormGroup, add);
  else for_each_grad_table<_Float16>(t, count, kNormGroup, add);
  return parts;
}

namespace {
int sumsq_any(const c3d_opt_tensor* t, int count, int type, double* partial, hipStream_t s) {
  return type == 0 ? sumsq<float>(t, count, partial, s) : type == 1 ? sumsq<__bf16>(t, count, partial, s) : sumsq<_Float16>(t, count, partial, s);
}
int small_any(const c3d_opt_tensor* t, int count, int type, bool clip, double max_norm, float* norm, float* scale, hipStream_t s) {
  return type == 0   ? small<float>(t, count, clip, max_norm, norm, scale, s)
         : type == 1 ? small<__bf16>(t, count, clip, max_norm, norm, scale, s)
                     : small<_Float16>(t, count, clip, max_norm, norm, scale, s);
}
bool any(const c3d_opt_tensor* t, int count) {
  return std::any_of(t, t + count, [](const c3d_opt_tensor& x) { return x.n > 0; });
}
int fold(const double* partial, int64_t parts, double max_norm, float* norm, float* scale, hipStream_t s) {
  hipLaunchKernelGGL(grad_norm_fold_kernel, dim3(1), dim3(1024), 0, s, partial, parts, max_norm, norm, scale);
  C3D_CHECK_LAUNCH();
  return 0;
}
int check_norm(const c3d_opt_tensor* t, int count, int type, double max_norm, const double* partial, int64_t& parts) {
  if (int rc = check_records(t, count, 1u << 1)) return rc;
  C3D_REQUIRE(type >= 0 && type <= 2, "grad_norm: type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(max_norm >= 0.0, "grad_norm: max_norm is negative or not a number");
  parts = c3d_grad_norm_partials(t, count, type);
  C3D_REQUIRE(parts == 0 || partial, "grad_norm: null workspace");
  return 0;
}
}  // namespace

extern "C" int c3d_grad_norm(const c3d_opt_tensor* t, int count, int type, double max_norm, double* partial, float* norm, float* scale,
                             c3d_stream stream) {
  int64_t parts;
  if (int rc = check_norm(t, count, type, max_norm, partial, parts)) return rc;
  C3D_REQUIRE(norm && scale, "grad_norm: null output");
  hipStream_t s = (hipStream_t)stream;
  if (parts == 0 && any(t, count)) return small_any(t, count, type, false, max_norm, norm, scale, s);
  if (int rc = sumsq_any(t, count, type, partial, s)) return rc;
  return fold(partial, parts, max_norm, norm, scale, s);
}

extern "C" int c3d_clip_grads(const c3d_opt_tensor* t, int count, int type, double max_norm, double* partial, float* norm, float* scale,
                              c3d_stream stream) {
  int64_t parts;
  if (int rc = check_norm(t, count, type, max_norm, partial, parts)) return rc;
  C3D_REQUIRE(norm && scale, "clip_grads: null output");
  hipStream_t s = (hipStream_t)stream;
  if (parts == 0 && any(t, count)) return small_any(t, count, type, true, max_norm, norm, scale, s);
  if (int rc = sumsq_any(t, count, type, partial, s)) return rc;
  if (int rc = fold(partial, parts, max_norm, norm, scale, s)) return rc;
  return type == 0 ? scale_all<float>(t, count, scale, s) : type == 1 ? scale_all<__bf16>(t, count, scale, s) : scale_all<_Float16>(t, count, scale, s);
}

extern "C" int c3d_adamw_step(const c3d_opt_tensor* t, int count, const c3d_adamw_desc* d, c3d_stream stream) {
  C3D_REQUIRE(d, "adamw: null descriptor");
  C3D_REQUIRE(d->state_bits == 32 || d->state_bits == 8, "adamw: state_bits is 32 or 8");
  C3D_REQUIRE(d->param_type >= 0 && d->param_type <= 2, "adamw: param_type is 0 (fp32), 1 (bf16) or 2 (fp16)");
  C3D_REQUIRE(d->grad_type == 0 || d->grad_type == d->param_type, "adamw: gradients are fp32 or of the parameters' type");
  C3D_REQUIRE(!(d->has_master && d->param_type == 0), "adamw: fp32 parameters have no master copy");
  C3D_REQUIRE(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0, "adamw: betas are in [0, 1)");
  // (the reciprocal instruction takes a smaller one for 0, and 0 / eps would not be 0)
  C3D_REQUIRE(d->eps == 0.0 || (float)d->eps >= 0x1p-126f, "adamw: eps is 0 or at least 2^-126");
  C3D_REQUIRE(d->step_dev || d->step >= 1, "adamw: step counts from 1");
  if (int rc = check_records(t, count, 0xfu | (d->state_bits == 8 ? 0x30u : 0u) | (d->has_master ? 0x40u : 0u))) return rc;
  Hyper h;
  h.beta1 = (float)d->beta1;
  h.omb1 = (float)(1.0 - d->beta1);
  h.beta2 = (float)d->beta2;
  h.omb2 = (float)(1.0 - d->beta2);
  h.b1 = d->beta1;
  h.o1 = 1.0 - d->beta1;
  h.b2 = d->beta2;
  h.o2 = 1.0 - d->beta2;
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
