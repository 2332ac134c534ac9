// bound.hip — norms over many tensors, and what is bounded by them, for MI355X (gfx950, CDNA4).
//
//   norm        n = (sum |x|^p)^(1/p) over every element of T tensors, p = 1, 2 or infinity
//   norm scale  y = round(x * min(1, M / (n + eps)))
//   peer norms  n_k = || p_k - c ||_2 over every tensor of peer k, for N peers around one centre
//   bounded     out = round(c + sum_k a_k (p_k - c)),  a_k = w_k * (n_k <= R ? 1 : R / n_k),
//               a_k = 0 (the peer is not read) where n_k is not finite
//
// All four move bytes and compute little: 2 to 6 operations per element read.  The bound is HBM (or, for
// a second pass over fewer than 256 MB, the Infinity Cache), so there are no matrix instructions here.
//
// Norms and products are carried in 64 bits whatever the storage type: a vector FMA in f64 issues at the
// rate of one in f32 on this chip, the kernels wait for memory either way, and the square of any f32 value
// is a normal f64, so no norm of finite 32- or 16-bit values overflows or underflows.  So are averages, but
// for most of the 16-bit types (Average below).  A result is rounded to its storage type once (16-bit types through
// f32: the first rounding moves a result by at most 2^-24 of itself).
//
// Work is cut into units of 1 to 32 KiB of one tensor; a unit never spans tensors.  The norms deal them round
// robin to P workgroups, the kernels that write give each a workgroup of its own in order: either way the chip
// walks every stream as one front (few DRAM rows and pages at a time; ranges instead of round robin cost 9 %
// for 128 peers).  A norm has one partial result per workgroup whatever the size, and they are joined in a fixed
// order, so results do not depend on which workgroup ended first.  Loads need element alignment only (gfx950
// takes 16-byte loads from any address), so tensors that start anywhere take the same path.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>
#include <new>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

#include "dlagg.h"
#include "dlagg_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any element address

template <class T>
__device__ inline const T __attribute__((address_space(1))) * global_ptr(const void* p) {
  return (const T __attribute__((address_space(1)))*)(uintptr_t)p;
}
template <class T>
__device__ inline T __attribute__((address_space(1))) * global_ptr(void* p) {
  return (T __attribute__((address_space(1)))*)(uintptr_t)p;
}
// Tables in device memory are written by an earlier kernel and never by the one that reads them: uniform
// reads through the constant address space become scalar loads.
template <class T>
__device__ inline const T __attribute__((address_space(4))) * const_ptr(const void* p) {
  return (const T __attribute__((address_space(4)))*)(uintptr_t)p;
}

// ---------------------------------------------------------------- elements
template <int DT> struct Elem;
template <> struct Elem<DLA_F32> {
  using bits = uint32_t;
  static constexpr int E = 4;
  static __device__ inline void widen(u32x4 r, double (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = static_cast<double>(__uint_as_float(r[i]));
  }
  static __device__ inline u32x4 narrow(const double (&v)[E]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < E; ++i) r[i] = __float_as_uint(static_cast<float>(v[i]));
    return r;
  }
};
template <> struct Elem<DLA_F64> {
  using bits = uint64_t;
  static constexpr int E = 2;
  static __device__ inline void widen(u32x4 r, double (&v)[E]) { __builtin_memcpy(v, &r, 16); }
  static __device__ inline u32x4 narrow(const double (&v)[E]) {
    u32x4 r;
    __builtin_memcpy(&r, v, 16);
    return r;
  }
};
template <> struct Elem<DLA_BF16> {
  using bits = uint16_t;
  static constexpr int E = 8;
  template <class R>
  static __device__ inline void widen(u32x4 r, R (&v)[E]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = static_cast<R>(__uint_as_float(r[i] << 16));
      v[2 * i + 1] = static_cast<R>(__uint_as_float(r[i] & 0xffff0000u));
    }
  }
  template <class R>
  static __device__ inline u32x4 narrow(const R (&v)[E]) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 f = {static_cast<float>(v[2 * i]), static_cast<float>(v[2 * i + 1])};
      const bf2 b = __builtin_convertvector(f, bf2);  // v_cvt_pk_bf16_f32: nearest even, NaN stays NaN
      uint32_t w;
      __builtin_memcpy(&w, &b, 4);
      r[i] = w;
    }
    return r;
  }
};
template <> struct Elem<DLA_F16> {
  using bits = uint16_t;
  static constexpr int E = 8;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  template <class R>
  static __device__ inline void widen(u32x4 r, R (&v)[E]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h2 h;
      const uint32_t w = r[i];
      __builtin_memcpy(&h, &w, 4);
      v[2 * i] = static_cast<R>(static_cast<float>(h[0]));
      v[2 * i + 1] = static_cast<R>(static_cast<float>(h[1]));
    }
  }
  template <class R>
  static __device__ inline u32x4 narrow(const R (&v)[E]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 h = {static_cast<_Float16>(static_cast<float>(v[2 * i])),
                    static_cast<_Float16>(static_cast<float>(v[2 * i + 1]))};
      uint32_t w;
      __builtin_memcpy(&w, &h, 4);
      r[i] = w;
    }
    return r;
  }
};

// The average's arithmetic: out = c + sum_k a_k (x_k - c), with a_k, the differences and the sum in `real`.  F32 and F64
// take 64 bits.  16-bit types, whose result keeps 8 or 11 bits, take 32 where those hold every term (share32): half the
// registers and no conversions (us, 32 bits / 32 and then 64: 16 x ResNet-34 bf16 130 / 278, 4 x 21.3 M bf16 43 / 66).
struct Average64 {
  using real = double;
  static __device__ inline const double* shares_of(const double* shares, int) { return shares; }
  static __device__ inline double fold(double a, double x, double c, double acc) { return __builtin_fma(a, x - c, acc); }
};
struct Average32 {
  using real = float;
  static __device__ inline const float* shares_of(const double* shares, int n_peers) {  // behind those in 64 bits
    return reinterpret_cast<const float*>(shares + n_peers);
  }
  static __device__ inline float fold(float a, float x, float c, float acc) { return __builtin_fmaf(a, x - c, acc); }
};
template <int DT>
using Average = std::conditional_t<DT == DLA_BF16 || DT == DLA_F16, Average32, Average64>;

// a_k in 32 bits, NaN where 32 bits may not do: a peer's share below their normal range (it would lose bits, or count
// for nothing), or differences, products or sums beyond it.  |x - c| <= n_k, so n_k <= 2^126 keeps differences in range
// and |a_k| n_k <= 2^114 the sums over kMostPeers = 2^11 peers.  A NaN makes every sum of the round NaN, and what is not
// finite is added up again in 64 bits (mean_unit): a round pays for its range only where it needs it.
__device__ inline float share32(double share, double norm) {
  const double a = __builtin_fabs(share);
  const bool fits = a == 0.0 || (a >= 0x1p-126 && a <= 0x1p126 && norm <= 0x1p126 && a * norm <= 0x1p114);
  return fits ? static_cast<float>(share) : __builtin_nanf("");
}

// Elements [j, j + n) of a tensor, n <= E: 16 bytes at once when n == E, else one by one with zeros behind.
template <int DT>
__device__ inline u32x4 load_part(const void* base, int64_t j, int n) {
  using B = typename Elem<DT>::bits;
  constexpr int E = Elem<DT>::E;
  const auto* p = global_ptr<B>(base) + j;
  if (n >= E) return *(const u32x4_any __attribute__((address_space(1)))*)p;
  B v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = i < n ? p[i] : B(0);
  u32x4 r;
  __builtin_memcpy(&r, v, 16);
  return r;
}
// NT: non-temporal, for data that no cache will hold until it is read again.
template <int DT, bool NT = true>
__device__ inline u32x4 load_full(const void* base, int64_t j) {
  using B = typename Elem<DT>::bits;
  const auto* p = (const u32x4_any __attribute__((address_space(1)))*)(global_ptr<B>(base) + j);
  if (NT) return __builtin_nontemporal_load(p);
  return *p;
}
template <int DT>
__device__ inline void store_part(void* base, int64_t j, int n, u32x4 r) {
  using B = typename Elem<DT>::bits;
  constexpr int E = Elem<DT>::E;
  auto* p = global_ptr<B>(base) + j;
  if (n >= E) {
    __builtin_nontemporal_store(r, (u32x4_any __attribute__((address_space(1)))*)p);
    return;
  }
  B v[E];
  __builtin_memcpy(v, &r, 16);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (i < n) p[i] = v[i];
}
__host__ __device__ inline int clamp_part(int64_t left, int most) {
  return left >= most ? most : left > 0 ? static_cast<int>(left) : 0;
}
__host__ __device__ constexpr int elem_bytes(int dt) { return dt == DLA_F64 ? 8 : dt == DLA_F32 ? 4 : 2; }

// ------------------------------------------------------------------- sums
// One term, and two partial results, of a norm.  Infinity norm: the larger, a NaN once seen stays.
template <int NORM>
__device__ inline double norm_term(double acc, double x) {
  if (NORM == DLA_NORM_L2) return __builtin_fma(x, x, acc);
  const double a = __builtin_fabs(x);
  if (NORM == DLA_NORM_L1) return acc + a;
  return a > acc || a != a ? a : acc;
}
template <int NORM>
__device__ inline double norm_join(double a, double b) {
  if (NORM != DLA_NORM_INF) return a + b;
  return b > a || b != b ? b : a;
}
// The workgroup's join of one value per thread, in every thread (a fixed order: lanes by halves, then waves).
template <int NORM>
__device__ inline double block_join(double v, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = norm_join<NORM>(v, __shfl_xor(v, d));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s = norm_join<NORM>(s, lds[w]);
  __syncthreads();
  return s;
}
// Partial results that another workgroup of the same kernel reads go past the L2 of the XCD that wrote them, both
// ways (agent-scope atomics): no workgroup has to write back or invalidate an L2, which a fence of that scope does
// and which cost 40 us over 1 024 workgroups.
__device__ inline void publish(double* p, double v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline double published(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Partials i, i + step, ... of n, in order; 8 loads in flight (each of them is a trip to memory).
template <int NORM>
__device__ inline double join_strided(const double* p, int n, int i, int step) {
  double v = 0;
  for (; i < n; i += 8 * step) {
    double r[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) r[q] = i + q * step < n ? published(p + i + q * step) : 0.0;
#pragma unroll
    for (int q = 0; q < 8; ++q) v = norm_join<NORM>(v, r[q]);
  }
  return v;
}
template <int NORM>
__device__ inline double join_partials(const double* partials, int n, double* lds) {
  const double v = join_strided<NORM>(partials, n, static_cast<int>(threadIdx.x), kThreads);
  const double s = block_join<NORM>(v, lds);
  return NORM == DLA_NORM_L2 ? __builtin_sqrt(s) : s;
}
__device__ inline void put_norm(void* out, int i, int out_dt, double v) {
  if (out_dt == DLA_F64) {
    global_ptr<double>(out)[i] = v;
  } else {
    global_ptr<float>(out)[i] = static_cast<float>(v);
  }
}

// -------------------------------------------------- one list of tensors: norm, and scaling by it
// A launch's tensors travel in the kernel arguments (nothing to copy, nothing a captured graph could find
// changed at replay): as many as fit 4 KB.
constexpr int kNormVec = 8, kScaleVec = 4;          // 16-byte loads in flight per lane: units of 32 and 16 KiB
constexpr int unit_bytes(int vec) { return kThreads * 16 * vec; }
constexpr int kNormTensors = 190, kScaleTensors = 140;
constexpr int kMaxPartials = 1024;                  // workgroups of a list's norm: 4 per CU

template <int M>
struct TensorList {
  const void* p[M];
  uint64_t n_dt[M];   // elements * 4 + dtype
  uint32_t unit0[M];  // first unit
};
template <int M>
struct TensorsInOut {
  TensorList<M> in;
  void* out[M];
};

// The tensor that unit u lies in: how many of the list's first units are <= u, counted by the wave's lanes.
__device__ inline int find_tensor(const uint32_t* unit0, int count, uint32_t u) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int n = 0;
  for (int i0 = 0; i0 < count; i0 += 64) n += __popcll(__ballot(i0 + lane < count && unit0[i0 + lane] <= u));
  return __builtin_amdgcn_readfirstlane(n) - 1;
}

template <int NORM, int DT, bool NT>
__device__ inline void norm_unit(const void* p, int64_t n, int64_t unit, double (&acc)[kNormVec]) {
  constexpr int E = Elem<DT>::E, kVec = kNormVec;
  const int64_t j0 = unit * (kThreads * kVec * E) + static_cast<int>(threadIdx.x) * E;
  u32x4 r[kVec];
  if ((unit + 1) * (kThreads * kVec * E) <= n) {
#pragma unroll
    for (int v = 0; v < kVec; ++v) r[v] = load_full<DT, NT>(p, j0 + v * (kThreads * E));
  } else {
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int64_t j = j0 + v * (kThreads * E);
      r[v] = load_part<DT>(p, j, clamp_part(n - j, E));
    }
  }
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    double x[E];
    Elem<DT>::widen(r[v], x);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[v] = norm_term<NORM>(acc[v], x[i]);
  }
}

// True in every thread of the last of a kernel's workgroups to get here, which then sees what the others' first
// threads published before they did: their stores have completed (vmcnt counts them) when the counter is raised.
// The counters are zero when the kernel starts and zero again when it has ended (they wrap).  Workgroups of one
// row (blockIdx.y) count together: many of them in two steps, 32 counters and then one, because a thousand
// increments of one address take 15 us.
constexpr int kCounterSlots = DLA_COUNTER_BYTES / 128, kSlot = 32;  // one counter per 128-byte line
constexpr uint32_t kFan = 32, kFanFrom = 64;
__device__ inline bool last_to_arrive(uint32_t* counters) {
  __shared__ bool last;
  if (threadIdx.x == 0) {
    const uint32_t n = gridDim.x, b = blockIdx.x;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (n >= kFanFrom && gridDim.y * (kFan + 1) <= kCounterSlots) {
      uint32_t* mine = counters + blockIdx.y * ((kFan + 1) * kSlot);
      const uint32_t fan = b % kFan, of = (n - fan + kFan - 1) / kFan;
      last = atomicInc(mine + (1 + fan) * kSlot, of - 1) == of - 1 && atomicInc(mine, kFan - 1) == kFan - 1;
    } else {
      last = atomicInc(counters + blockIdx.y * kSlot, n - 1) == n - 1;
    }
    asm volatile("" ::: "memory");
  }
  __syncthreads();
  return last;
}

// Workgroup b's part of the norm of a list: partials[b].  With a counter, the last workgroup joins the `joined`
// partials (this launch's and those of the launches before it) into *norm and *out.
template <int NORM, bool NT>
__global__ __launch_bounds__(kThreads) void norm_kernel(const TensorList<kNormTensors> tab, int count, uint32_t units,
                                                        double* to, uint32_t* counter, const double* partials,
                                                        int joined, double* norm, int out_dt, void* out) {
  __shared__ double lds[kWaves];
  const uint32_t b = blockIdx.x, nb = gridDim.x;
  uint32_t first = 0, stop = 0;
  const void* p = nullptr;
  uint64_t nd = 0;
  double acc[kNormVec] = {};
  for (uint64_t at = b; at < units; at += nb) {
    const uint32_t u = static_cast<uint32_t>(at);
    if (u >= stop) {
      const int t = find_tensor(tab.unit0, count, u);
      first = tab.unit0[t];
      stop = t + 1 < count ? tab.unit0[t + 1] : units;
      p = tab.p[t];
      nd = tab.n_dt[t];
    }
    const int64_t n = static_cast<int64_t>(nd >> 2);
    switch (nd & 3) {
      case DLA_F32: norm_unit<NORM, DLA_F32, NT>(p, n, u - first, acc); break;
      case DLA_BF16: norm_unit<NORM, DLA_BF16, NT>(p, n, u - first, acc); break;
      case DLA_F16: norm_unit<NORM, DLA_F16, NT>(p, n, u - first, acc); break;
      default: norm_unit<NORM, DLA_F64, NT>(p, n, u - first, acc); break;
    }
  }
  double v = acc[0];
#pragma unroll
  for (int i = 1; i < kNormVec; ++i) v = norm_join<NORM>(v, acc[i]);
  v = block_join<NORM>(v, lds);
  if (threadIdx.x == 0) publish(to + b, v);
  if (!counter || !last_to_arrive(counter)) return;
  v = join_partials<NORM>(partials, joined, lds);
  if (threadIdx.x == 0) {
    *global_ptr<double>(norm) = v;
    if (out) put_norm(out, 0, out_dt, v);
  }
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_join_kernel(const double* partials, int n, int out_dt, void* out) {
  __shared__ double lds[kWaves];
  const double v = join_partials<NORM>(partials, n, lds);
  if (threadIdx.x == 0) put_norm(out, 0, out_dt, v);
}

template <int DT, bool NT>
__device__ inline void scale_unit(const void* p, void* out, int64_t n, int64_t unit, double ratio) {
  constexpr int E = Elem<DT>::E, kVec = kScaleVec;
  const int64_t j0 = unit * (kThreads * kVec * E) + static_cast<int>(threadIdx.x) * E;
  const bool full = (unit + 1) * (kThreads * kVec * E) <= n;
  u32x4 r[kVec];
  int part[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int64_t j = j0 + v * (kThreads * E);
    part[v] = full ? E : clamp_part(n - j, E);
    r[v] = full ? load_full<DT, NT>(p, j) : load_part<DT>(p, j, part[v]);
  }
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    double x[E];
    Elem<DT>::widen(r[v], x);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] *= ratio;
    store_part<DT>(out, j0 + v * (kThreads * E), part[v], Elem<DT>::narrow(x));
  }
}

// y = round(x * min(1, M / (n + eps))).  One unit per workgroup, dealt from the last to the first: what the norm
// read last is what the caches still hold, and the front stays narrow (0.87 G bf16: 561 us, where 2 048 workgroups
// walking their units took 630).
template <bool NT>
__global__ __launch_bounds__(kThreads) void norm_scale_kernel(const TensorsInOut<kScaleTensors> tab, int count,
                                                              uint32_t units, const double* joined, double max_norm,
                                                              double eps, int in_place, int out_dt, void* norm_out) {
  const double norm = *const_ptr<double>(joined);
  const uint32_t b = blockIdx.x, nb = gridDim.x;
  if (b == 0 && threadIdx.x == 0 && norm_out) put_norm(norm_out, 0, out_dt, norm);
  const double q = max_norm / (norm + eps);
  const double ratio = q > 1.0 ? 1.0 : q;  // NaN stays NaN
  if (in_place && ratio == 1.0) return;    // x * 1 = x: nothing to write
  uint32_t first = 0xffffffffu;
  const void* p = nullptr;
  void* out = nullptr;
  uint64_t nd = 0;
  for (int64_t at = static_cast<int64_t>(units) - 1 - b; at >= 0; at -= nb) {
    const uint32_t u = static_cast<uint32_t>(at);
    if (u < first) {
      const int t = find_tensor(tab.in.unit0, count, u);
      first = tab.in.unit0[t];
      p = tab.in.p[t];
      out = tab.out[t];
      nd = tab.in.n_dt[t];
    }
    const int64_t n = static_cast<int64_t>(nd >> 2);
    switch (nd & 3) {
      case DLA_F32: scale_unit<DLA_F32, NT>(p, out, n, u - first, ratio); break;
      case DLA_BF16: scale_unit<DLA_BF16, NT>(p, out, n, u - first, ratio); break;
      case DLA_F16: scale_unit<DLA_F16, NT>(p, out, n, u - first, ratio); break;
      default: scale_unit<DLA_F64, NT>(p, out, n, u - first, ratio); break;
    }
  }
}

// ------------------------------------------------------------- peers around a centre
// The round's table: a record per tensor, then the peers' pointers (tensor-major), then the weights.  Up to
// kPutWords words travel in the kernels' own arguments (14 tensors of 2 peers take 100, one tensor of 128 peers
// 261); a larger table goes to the workspace first — by a copy kernel that reads the caller's page-locked memory, or
// by value as arguments of put_kernel, as many launches as it takes, which a captured graph keeps.
struct Seg {
  int64_t norm_unit0, mean_unit0;  // first unit of the tensor in each of the two kernels' counts
  uint64_t n_dt;                   // elements * 4 + dtype
  const void* center;
  void* out;
};
struct Layout {      // where element j of a peer (and of the centre) lies, in elements from its pointer:
  int shift;         //   (j >> shift) * stride + (j & (2^shift - 1)) in a tile-interleaved slab
  int64_t stride;
  int64_t center_stride;
};
// 16-byte loads of one peer in a row per lane of the norms: 16 KiB of each stream at a time (8 x 25 M f32 138 us, with
// one load 143); tiles of a slab lie side by side anyway.
constexpr int peer_vec(bool tiled) { return tiled ? 1 : 4; }
constexpr int kMeanThreads = 64;                        // the average: one wave, 1 KiB of each stream
constexpr int kMeanUnit = kMeanThreads * 16;
constexpr int kPutWords = 480;
struct PutWords {
  uint64_t w[kPutWords];
};
__global__ __launch_bounds__(512) void put_kernel(const PutWords words, uint64_t* dst, int n) {
  const int i = static_cast<int>(threadIdx.x);
  if (i < n) global_ptr<uint64_t>(dst)[i] = words.w[i];
}
__global__ __launch_bounds__(kThreads) void fetch_kernel(const uint64_t* src, uint64_t* dst, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n) global_ptr<uint64_t>(dst)[i] = global_ptr<uint64_t>(src)[i];
}

// Where a kernel finds its table: in the workspace, or in its own first argument (the kernel argument segment is
// memory like any other).
struct Table {
  const uint64_t* at;  // null: in the arguments
  int count, n_peers;
};
struct TableParts {
  const Seg* segs;
  const uint64_t* ptrs;
  const double* weights;
};
__device__ inline TableParts parts_of(const Table& tab) {
  const uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  const uint64_t at = tab.at ? reinterpret_cast<uint64_t>(tab.at) : args;
  const uint64_t ptrs = at + static_cast<uint64_t>(tab.count) * sizeof(Seg);
  return {reinterpret_cast<const Seg*>(at), reinterpret_cast<const uint64_t*>(ptrs),
          reinterpret_cast<const double*>(ptrs + static_cast<uint64_t>(tab.count) * tab.n_peers * 8)};
}

template <bool TILED>
__device__ inline int64_t place(const Layout& l, int64_t stride, int64_t j) {
  return TILED ? (j >> l.shift) * stride + (j & ((int64_t{1} << l.shift) - 1)) : j;
}

// The tensor that unit u lies in: a 64-way search by the wave's lanes over the records' first units.
template <int64_t Seg::*UNIT0>
__device__ inline int find_seg(const Seg* segs, int count, int64_t u) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const int below = __popcll(__ballot(i < hi && (global_ptr<Seg>(segs) + (i < hi ? i : lo))->*UNIT0 <= u));
    lo = __builtin_amdgcn_readfirstlane(lo + (below - 1) * step);
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

template <int DT, int G, bool TILED>
__device__ inline void peer_norm_unit(const Layout& l, const void* center, const void* const (&p)[G], int64_t n,
                                      int64_t unit, double (&acc)[G]) {
  constexpr int E = Elem<DT>::E, V = peer_vec(TILED);
  const int64_t j0 = unit * (kThreads * V * E) + static_cast<int>(threadIdx.x) * E;
  u32x4 rc[V], r[G][V];
  if ((unit + 1) * (kThreads * V * E) <= n) {
#pragma unroll
    for (int v = 0; v < V; ++v) rc[v] = load_full<DT>(center, place<TILED>(l, l.center_stride, j0 + v * (kThreads * E)));
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int v = 0; v < V; ++v) r[g][v] = load_full<DT>(p[g], place<TILED>(l, l.stride, j0 + v * (kThreads * E)));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t j = j0 + v * (kThreads * E);
      const int part = clamp_part(n - j, E);
      rc[v] = load_part<DT>(center, place<TILED>(l, l.center_stride, j), part);
#pragma unroll
      for (int g = 0; g < G; ++g) r[g][v] = load_part<DT>(p[g], place<TILED>(l, l.stride, j), part);
    }
  }
  double c[V][E];
#pragma unroll
  for (int v = 0; v < V; ++v) Elem<DT>::widen(rc[v], c[v]);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      double x[E];
      Elem<DT>::widen(r[g][v], x);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const double d = x[i] - c[v][i];
        acc[g] = __builtin_fma(d, d, acc[g]);
      }
    }
}

// Where a peer's joined norm goes; null: not wanted.
struct Joined {
  const double* sq_in;  // given squares, instead of the partials
  double* sq;           // squares
  void* norms;          // roots, of out_dt
  int out_dt;
  double* shares;       // a_k, by max_norm
  float* shares32;      // share32 of them
  double max_norm;
};
// One wave: peer k's squared norm — the sum of its n partials (possibly none), or sq_in[k] — and what follows.
__device__ inline void join_peer(const double* partials, int n, int k, const double* weights, const Joined& to) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  double v = 0;
  if (to.sq_in) {
    v = global_ptr<double>(to.sq_in)[k];
  } else {
    v = join_strided<DLA_NORM_L2>(partials + static_cast<int64_t>(k) * n, n, lane, 64);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  }
  if (lane != 0) return;
  const double norm = __builtin_sqrt(v);
  if (to.sq) global_ptr<double>(to.sq)[k] = v;
  if (to.norms) put_norm(to.norms, k, to.out_dt, norm);
  if (to.shares) {
    const double share = global_ptr<double>(weights)[k] * (norm <= to.max_norm ? 1.0 : to.max_norm / norm);
    const double counted = __builtin_isfinite(norm) ? share : 0.0;
    global_ptr<double>(to.shares)[k] = counted;
    global_ptr<float>(to.shares32)[k] = share32(counted, norm);
  }
}

// partials[k * gridDim.x + b]: workgroup b's part of || p_k - c ||^2 for the peers of group blockIdx.y.  G
// peers are read beside one read of the centre, so the centre costs 1 / G of a peer.  With counters (one per
// group), a group's last workgroup joins its peers.
template <int G, bool TILED>
__global__ __launch_bounds__(kThreads) void peer_norms_kernel(const PutWords words, Table tab, int64_t units, Layout l,
                                                              double* partials, uint32_t* counters, const Joined to) {
  __shared__ double lds[kWaves];
  const TableParts parts = parts_of(tab);
  const Seg* segs = parts.segs;
  const uint64_t* ptrs = parts.ptrs;
  const int count = tab.count, n_peers = tab.n_peers;
  const int64_t b = blockIdx.x, nb = gridDim.x;
  const int k0 = static_cast<int>(blockIdx.y) * G;
  int64_t first = 0, stop = 0, n = 0;
  int dt = 0;
  const void* center = nullptr;
  const void* p[G];
  double acc[G] = {};
  for (int64_t u = b; u < units; u += nb) {
    if (u >= stop) {
      const int t = find_seg<&Seg::norm_unit0>(segs, count, u);
      const auto* s = const_ptr<Seg>(segs) + t;
      first = s->norm_unit0;
      n = static_cast<int64_t>(s->n_dt >> 2);
      dt = static_cast<int>(s->n_dt & 3);
      center = s->center;
      stop = t + 1 < count ? s[1].norm_unit0 : units;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int k = k0 + g < n_peers ? k0 + g : n_peers - 1;  // a spare place reads the last peer again
        p[g] = reinterpret_cast<const void*>(const_ptr<uint64_t>(ptrs)[static_cast<int64_t>(t) * n_peers + k]);
      }
    }
    switch (dt) {
      case DLA_F32: peer_norm_unit<DLA_F32, G, TILED>(l, center, p, n, u - first, acc); break;
      case DLA_BF16: peer_norm_unit<DLA_BF16, G, TILED>(l, center, p, n, u - first, acc); break;
      case DLA_F16: peer_norm_unit<DLA_F16, G, TILED>(l, center, p, n, u - first, acc); break;
      default: peer_norm_unit<DLA_F64, G, TILED>(l, center, p, n, u - first, acc); break;
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const double v = block_join<DLA_NORM_L2>(acc[g], lds);
    if (threadIdx.x == 0 && k0 + g < n_peers) publish(partials + (k0 + g) * nb + b, v);
  }
  if (!counters || !last_to_arrive(counters)) return;
  for (int g = static_cast<int>(threadIdx.x >> 6); g < G && k0 + g < n_peers; g += kWaves)
    join_peer(partials, static_cast<int>(nb), k0 + g, parts.weights, to);
}

// The join as a kernel of its own: one wave per peer.
__global__ __launch_bounds__(64) void peer_join_kernel(const PutWords words, Table tab, const double* partials, int n,
                                                       const Joined to) {
  join_peer(partials, n, static_cast<int>(blockIdx.x), parts_of(tab).weights, to);
}

// G peers' terms, their loads all in flight.
template <class A, int DT, int G, bool TILED>
__device__ inline void fold_peers(const uint64_t* ptrs, const typename A::real* shares, const void* center, int64_t at,
                                  int64_t at_c, bool full, int part, const typename A::real (&c)[Elem<DT>::E],
                                  typename A::real (&acc)[Elem<DT>::E]) {
  using R = typename A::real;
  constexpr int E = Elem<DT>::E;
  u32x4 r[G];
  R a[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    a[g] = const_ptr<R>(shares)[g];
    const void* p = reinterpret_cast<const void*>(const_ptr<uint64_t>(ptrs)[g]);
    const bool counts = a[g] != R(0);  // a peer that does not count is not read: the centre stands in, update 0
    p = counts ? p : center;
    const int64_t from = TILED ? (counts ? at : at_c) : at;
    r[g] = full ? load_full<DT>(p, from) : load_part<DT>(p, from, part);
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    R x[E];
    Elem<DT>::widen(r[g], x);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = A::fold(a[g], x[i], c[i], acc[i]);
  }
}

// Elements [j, j + part) of the average, G peers at a time and then what is left by halves.
template <class A, int DT, int G, bool TILED>
__device__ inline void average(const uint64_t* ptrs, const double* shares_of_all, int n_peers, const void* center, u32x4 rc,
                               int64_t at, int64_t at_c, bool full, int part, typename A::real (&acc)[Elem<DT>::E]) {
  constexpr int E = Elem<DT>::E;
  const typename A::real* shares = A::shares_of(shares_of_all, n_peers);
  typename A::real c[E];
  Elem<DT>::widen(rc, c);
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0;
  int i = 0;
  for (; i + G <= n_peers; i += G) fold_peers<A, DT, G, TILED>(ptrs + i, shares + i, center, at, at_c, full, part, c, acc);
  if (G > 4 && i + 4 <= n_peers) {
    fold_peers<A, DT, 4, TILED>(ptrs + i, shares + i, center, at, at_c, full, part, c, acc);
    i += 4;
  }
  if (G > 2 && i + 2 <= n_peers) {
    fold_peers<A, DT, 2, TILED>(ptrs + i, shares + i, center, at, at_c, full, part, c, acc);
    i += 2;
  }
  if (G > 1 && i < n_peers) fold_peers<A, DT, 1, TILED>(ptrs + i, shares + i, center, at, at_c, full, part, c, acc);
  // where the centre is not finite no peer counts, and the centre stays
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = __builtin_isfinite(c[e]) ? acc[e] + c[e] : c[e];
}

template <int DT, bool TILED>
__device__ inline void mean_unit(const Layout& l, const uint64_t* ptrs, const double* shares, int n_peers,
                                 const void* center, void* out, int64_t n, int64_t unit) {
  using A = Average<DT>;
  constexpr int E = Elem<DT>::E;
  const int64_t j = unit * (kMeanThreads * E) + static_cast<int>(threadIdx.x) * E;
  const int64_t at = place<TILED>(l, l.stride, j), at_c = place<TILED>(l, l.center_stride, j);
  const bool full = (unit + 1) * (kMeanThreads * E) <= n;
  const int part = full ? E : clamp_part(n - j, E);
  const u32x4 rc = full ? load_full<DT>(center, at_c) : load_part<DT>(center, at_c, part);
  typename A::real acc[E];
  average<A, DT, 8, TILED>(ptrs, shares, n_peers, center, rc, at, at_c, full, part, acc);
  u32x4 mean = Elem<DT>::narrow(acc);
  if constexpr (std::is_same_v<A, Average32>) {
    // Not finite: a share that 32 bits do not hold, a sum beyond what given norms promised, or the result's own, which
    // stays so.  Nothing is written yet, so the output may be an input here too; one peer at a time, for the registers.
    bool again = false;
#pragma unroll
    for (int e = 0; e < E; ++e) again |= !__builtin_isfinite(acc[e]);
    if (again) {
      double wide[E];
      average<Average64, DT, 1, TILED>(ptrs, shares, n_peers, center, rc, at, at_c, full, part, wide);
      mean = Elem<DT>::narrow(wide);
    }
  }
  store_part<DT>(out, j, part, mean);
}

// out = round(c + sum_k a_k (p_k - c)).  Units are dealt from the last to the first: what the norms read last is
// what the caches still hold.
template <bool TILED>
__global__ __launch_bounds__(kMeanThreads) void bounded_kernel(const PutWords words, Table tab, int64_t units,
                                                               const double* shares, Layout l) {
  const TableParts parts = parts_of(tab);
  const Seg* segs = parts.segs;
  const uint64_t* ptrs = parts.ptrs;
  const int count = tab.count, n_peers = tab.n_peers;
  for (int64_t u = units - 1 - blockIdx.x; u >= 0; u -= gridDim.x) {
    const int t = find_seg<&Seg::mean_unit0>(segs, count, u);
    const auto* s = const_ptr<Seg>(segs) + t;
    const int64_t first = s->mean_unit0, n = static_cast<int64_t>(s->n_dt >> 2);
    const void* center = s->center;
    void* out = s->out;
    const uint64_t* mine = ptrs + static_cast<int64_t>(t) * n_peers;
    switch (s->n_dt & 3) {
      case DLA_F32: mean_unit<DLA_F32, TILED>(l, mine, shares, n_peers, center, out, n, u - first); break;
      case DLA_BF16: mean_unit<DLA_BF16, TILED>(l, mine, shares, n_peers, center, out, n, u - first); break;
      case DLA_F16: mean_unit<DLA_F16, TILED>(l, mine, shares, n_peers, center, out, n, u - first); break;
      default: mean_unit<DLA_F64, TILED>(l, mine, shares, n_peers, center, out, n, u - first); break;
    }
  }
}

// ------------------------------------------------------------------ host side
int fail(int code, const std::string& msg) { return dla_internal_fail(code, msg.c_str()); }
int hip_fail(const char* what, hipError_t e) {
  return fail(static_cast<int>(e), std::string(what) + ": " + hipGetErrorString(e));
}

bool known_dtype(int dt) { return dt == DLA_F32 || dt == DLA_BF16 || dt == DLA_F16 || dt == DLA_F64; }
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// No element count here exceeds this: 2^56 bytes, far beyond any device, keeps every product below in 64 bits.
constexpr int64_t kMostElems = int64_t{1} << 53;
constexpr double kInfinityCache = 256.0 * (1 << 20);

// The launches a list of tensors takes: tensors [begin, end) of `order` (the non-empty ones), `units` units on
// `blocks` workgroups.
struct ListLaunch {
  int begin, end;
  uint32_t units;
  int blocks;
};

int64_t list_units(int dt, int64_t n, int vec) {
  const int64_t per = unit_bytes(vec) / elem_bytes(dt);
  return (n + per - 1) / per;
}

// `most` workgroups in all, shared by the launches as their units are, or (0) one per unit where a launch takes that many.
bool plan_list(const std::vector<int>& order, const int* dtypes, const int64_t* numels, int vec, int per_launch, int64_t most,
               std::vector<ListLaunch>* out) {
  int64_t total = 0;
  for (int t : order) total += list_units(dtypes[t], numels[t], vec);
  for (size_t i = 0; i < order.size(); i += per_launch) {
    const int end = static_cast<int>(std::min(order.size(), i + per_launch));
    int64_t units = 0;
    for (int q = static_cast<int>(i); q < end; ++q) units += list_units(dtypes[order[q]], numels[order[q]], vec);
    if (units > 0xffffffffll) return false;
    const int64_t share = most ? std::max<int64_t>(1, most * units / total) : dla_internal_grid(units, kThreads);
    out->push_back({static_cast<int>(i), end, static_cast<uint32_t>(units), static_cast<int>(std::min(units, share))});
  }
  return true;
}

template <int M>
void fill_list(TensorList<M>* tab, const ListLaunch& l, const std::vector<int>& order, const int* dtypes,
               const void* const* tensors, const int64_t* numels, int vec) {
  std::memset(tab, 0, sizeof(*tab));
  uint32_t u = 0;
  for (int q = l.begin; q < l.end; ++q) {
    const int t = order[q], i = q - l.begin;
    tab->p[i] = tensors[t];
    tab->n_dt[i] = static_cast<uint64_t>(numels[t]) * 4 + static_cast<uint64_t>(dtypes[t]);
    tab->unit0[i] = u;
    u += static_cast<uint32_t>(list_units(dtypes[t], numels[t], vec));
  }
}

int check_list(const char* what, int n_tensors, const int* dtypes, const void* const* tensors, const int64_t* numels,
               int norm, std::vector<int>* order) {
  if (n_tensors < 0) return fail(DLA_E_INVALID, std::string(what) + ": n_tensors < 0");
  if (n_tensors > 0 && (!dtypes || !tensors || !numels))
    return fail(DLA_E_INVALID, std::string(what) + ": null dtypes / tensors / numels array");
  if (norm != DLA_NORM_L2 && norm != DLA_NORM_L1 && norm != DLA_NORM_INF)
    return fail(DLA_E_INVALID, std::string(what) + ": unknown norm " + std::to_string(norm));
  for (int t = 0; t < n_tensors; ++t) {
    if (!known_dtype(dtypes[t]))
      return fail(DLA_E_INVALID, std::string(what) + ": tensor " + std::to_string(t) + " has unknown dtype " + std::to_string(dtypes[t]));
    if (numels[t] < 0 || numels[t] > kMostElems)
      return fail(DLA_E_INVALID, std::string(what) + ": tensor " + std::to_string(t) + " has a bad element count");
    if (numels[t] == 0) continue;
    if (!tensors[t] || !aligned_to(tensors[t], elem_bytes(dtypes[t])))
      return fail(DLA_E_INVALID, std::string(what) + ": tensor " + std::to_string(t) + " is null or not aligned to its elements");
    order->push_back(t);
  }
  return DLA_OK;
}

struct Span {
  uintptr_t begin, end;
};
Span span_of(const void* p, int64_t n, int bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return {a, a + static_cast<uintptr_t>(n) * bytes};
}
// `outs` sorted by begin and disjoint?
bool disjoint(std::vector<Span>* outs) {
  std::sort(outs->begin(), outs->end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < outs->size(); ++i)
    if ((*outs)[i].begin < (*outs)[i - 1].end) return false;
  return true;
}
// Does `s` meet an output other than by being exactly `own`?
bool meets(const std::vector<Span>& outs, const Span& s, const Span& own) {
  if (s.begin == own.begin) return s.end != own.end;
  if (outs.empty() || s.end <= outs.front().begin || s.begin >= outs.back().end) return false;
  auto it = std::upper_bound(outs.begin(), outs.end(), s.begin, [](uintptr_t v, const Span& o) { return v < o.begin; });
  if (it != outs.end() && it->begin < s.end) return true;
  return it != outs.begin() && std::prev(it)->end > s.begin;
}

// f(norm, nt) with both as constants.
template <class F>
void with_norm(int norm, bool nt, F f) {
  using std::integral_constant;
  const auto by_nt = [&](auto p) {
    if (nt) f(p, std::true_type{});
    else f(p, std::false_type{});
  };
  if (norm == DLA_NORM_L2) by_nt(integral_constant<int, DLA_NORM_L2>{});
  else if (norm == DLA_NORM_L1) by_nt(integral_constant<int, DLA_NORM_L1>{});
  else by_nt(integral_constant<int, DLA_NORM_INF>{});
}

// The workspace of a list's norm: the joined norm, then the partials.
int norm_launches(const char* what, const std::vector<int>& order, const int* dtypes, const void* const* tensors,
                  const int64_t* numels, int norm, bool nt, int out_dtype, void* out, void* counter, double* workspace,
                  int* n_partials, hipStream_t s) {
  std::vector<ListLaunch> launches;
  if (!plan_list(order, dtypes, numels, kNormVec, kNormTensors, kMaxPartials, &launches))
    return fail(DLA_E_INVALID, std::string(what) + ": too many elements");
  double* partials = workspace + 1;
  *n_partials = 0;
  for (const ListLaunch& l : launches) *n_partials += l.blocks;
  double* to = partials;
  for (const ListLaunch& l : launches) {
    TensorList<kNormTensors> tab;
    fill_list(&tab, l, order, dtypes, tensors, numels, kNormVec);
    const dim3 grid(static_cast<unsigned>(l.blocks));
    const int count = l.end - l.begin;
    uint32_t* last = &l == &launches.back() ? static_cast<uint32_t*>(counter) : nullptr;
    with_norm(norm, nt, [&](auto p, auto stream_once) {
      hipLaunchKernelGGL((norm_kernel<p(), stream_once()>), grid, dim3(kThreads), 0, s, tab, count, l.units, to, last,
                         partials, *n_partials, workspace, out_dtype, out);
    });
    to += l.blocks;
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  return DLA_OK;
}

// The joined norm from the partials, where no counter did it (none: the norm of nothing, 0).
int join_launch(const char* what, int norm, const double* workspace, int n_partials, int out_dtype, void* out, hipStream_t s) {
  const double* partials = workspace + 1;
  with_norm(norm, true, [&](auto p, auto) {
    hipLaunchKernelGGL((norm_join_kernel<p()>), dim3(1), dim3(kThreads), 0, s, partials, n_partials, out_dtype, out);
  });
  if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  return DLA_OK;
}

int check_norm_memory(const char* what, int n_tensors, int out_dtype, const void* out, const void* counter,
                      const void* workspace, int64_t workspace_bytes) {
  const std::string w(what);
  if (out && ((out_dtype != DLA_F32 && out_dtype != DLA_F64) || !aligned_to(out, elem_bytes(out_dtype))))
    return fail(DLA_E_INVALID, w + ": the norm goes to an aligned F32 or F64 value");
  if (!aligned_to(counter, 4)) return fail(DLA_E_INVALID, w + ": counter is not aligned");
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < dla_norm_workspace(n_tensors))
    return fail(DLA_E_INVALID, w + ": workspace is null, not aligned or smaller than dla_norm_workspace");
  return DLA_OK;
}

int norm_impl(int n_tensors, const int* dtypes, const void* const* tensors, const int64_t* numels, int norm, int out_dtype,
              void* out, void* counter, void* workspace, int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_list("dla_norm", n_tensors, dtypes, tensors, numels, norm, &order)) return rc;
  if (!out) return fail(DLA_E_INVALID, "dla_norm: null out");
  if (int rc = check_norm_memory("dla_norm", n_tensors, out_dtype, out, counter, workspace, workspace_bytes)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* ws = static_cast<double*>(workspace);
  int n_partials = 0;
  if (int rc = norm_launches("dla_norm", order, dtypes, tensors, numels, norm, true, out_dtype, out, counter, ws, &n_partials, s))
    return rc;
  return counter && n_partials > 0 ? DLA_OK : join_launch("dla_norm", norm, ws, n_partials, out_dtype, out, s);
}

int norm_clip_impl(int n_tensors, const int* dtypes, const void* const* tensors, void* const* outs, const int64_t* numels,
                   int norm, double max_norm, double eps, int out_dtype, void* norm_out, void* counter, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_list("dla_norm_clip", n_tensors, dtypes, tensors, numels, norm, &order)) return rc;
  if (!(max_norm >= 0) || !(eps > 0)) return fail(DLA_E_INVALID, "dla_norm_clip: max_norm must be >= 0 and eps > 0");
  if (int rc = check_norm_memory("dla_norm_clip", n_tensors, out_dtype, norm_out, counter, workspace, workspace_bytes)) return rc;
  if (!order.empty() && !outs) return fail(DLA_E_INVALID, "dla_norm_clip: null outs array");
  std::vector<Span> spans;
  bool in_place = true;
  for (int t : order) {
    if (!outs[t] || !aligned_to(outs[t], elem_bytes(dtypes[t])))
      return fail(DLA_E_INVALID, "dla_norm_clip: out " + std::to_string(t) + " is null or not aligned to its elements");
    spans.push_back(span_of(outs[t], numels[t], elem_bytes(dtypes[t])));
    in_place = in_place && outs[t] == tensors[t];
  }
  const std::vector<Span> own = spans;
  if (!disjoint(&spans)) return fail(DLA_E_ALIAS, "dla_norm_clip: two outputs overlap");
  for (size_t q = 0; q < order.size() && !in_place; ++q)
    if (meets(spans, span_of(tensors[order[q]], numels[order[q]], elem_bytes(dtypes[order[q]])), own[q]))
      return fail(DLA_E_ALIAS, "dla_norm_clip: tensor " + std::to_string(order[q]) + " overlaps an output that is not its own");
  std::vector<ListLaunch> launches;
  int n_partials = 0;
  if (!plan_list(order, dtypes, numels, kScaleVec, kScaleTensors, 0, &launches))
    return fail(DLA_E_INVALID, "dla_norm_clip: too many elements");
  // What the Infinity Cache (256 MB) can hold is kept in the caches for the second read; more streams past them
  // (us, kept / streamed: 21 M bf16 27.4 / 30.8, 40 M f32 79.0 / 82.3; 0.87 G bf16 933 / 889)
  double bytes = 0;
  for (int t : order) bytes += static_cast<double>(numels[t]) * elem_bytes(dtypes[t]);
  const bool nt = bytes > kInfinityCache;
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* ws = static_cast<double*>(workspace);
  if (int rc = norm_launches("dla_norm_clip", order, dtypes, tensors, numels, norm, nt, out_dtype, nullptr, counter, ws, &n_partials, s))
    return rc;
  if (launches.empty()) return norm_out ? join_launch("dla_norm_clip", norm, ws, 0, out_dtype, norm_out, s) : DLA_OK;
  if (!counter)
    if (int rc = join_launch("dla_norm_clip", norm, ws, n_partials, DLA_F64, ws, s)) return rc;
  for (const ListLaunch& l : launches) {
    TensorsInOut<kScaleTensors> tab;
    fill_list(&tab.in, l, order, dtypes, tensors, numels, kScaleVec);
    std::memset(tab.out, 0, sizeof(tab.out));
    for (int q = l.begin; q < l.end; ++q) tab.out[q - l.begin] = outs[order[q]];
    const dim3 grid(static_cast<unsigned>(l.blocks));
    const int count = l.end - l.begin, inp = in_place ? 1 : 0;
    void* no = l.begin == 0 ? norm_out : nullptr;
    if (nt) hipLaunchKernelGGL((norm_scale_kernel<true>), grid, dim3(kThreads), 0, s, tab, count, l.units, ws, max_norm, eps, inp, out_dtype, no);
    else hipLaunchKernelGGL((norm_scale_kernel<false>), grid, dim3(kThreads), 0, s, tab, count, l.units, ws, max_norm, eps, inp, out_dtype, no);
    if (hipError_t e = hipGetLastError()) return hip_fail("dla_norm_clip", e);
  }
  return DLA_OK;
}

// ------------------------------------------------------------------ peers, host side
constexpr int kMostPeers = 2048;

// Peers beside one read of the centre: 8 at most (their loads are all in flight), groups of equal size.  The norms
// take 1 024 workgroups in all, from 8 groups on as many as run at once (2 per CU), which evens out as well there and keeps
// fewer rows open (us, 1 024 / 512: 8 groups, 64 x 12 M bf16 257.6 / 250.1 and 64 x 6 M f32 255.1 / 248.8; 16 groups 492.5 /
// 484.8 and 490.2 / 476.7; but 6 groups 198.5 / 202.9 and 195.2 / 196.7, 5 groups 167.4 / 168.3, 2 groups 71.3 / 73.3, and
// 40 x ResNet-34 bf16 292 / 298).
int peer_groups(int n) { return (n + 7) / 8; }
int64_t peer_blocks(int n) {
  const int groups = peer_groups(n);
  return std::max(1, (groups >= 8 ? 512 : 1024) / groups);
}

int64_t peer_table_words(int64_t n_tensors, int64_t n_peers) {
  return n_tensors * static_cast<int64_t>(sizeof(Seg) / 8) + n_tensors * n_peers + n_peers;
}
int64_t share_words(int64_t n_peers) { return n_peers + (n_peers + 1) / 2; }  // in 64 bits and in 32
int64_t peer_workspace_bytes(int64_t n_tensors, int64_t n_peers) {
  return (peer_table_words(n_tensors, n_peers) + share_words(n_peers) + n_peers * peer_blocks(static_cast<int>(n_peers))) * 8;
}

struct Round {  // a round's arguments, as the entry points give them
  int n_tensors;
  const int* dtypes;
  const void* const* peers;  // [n_tensors * n_peers], tensor-major
  const void* const* centers;
  void* const* outs;  // null: norms only
  const int64_t* numels;
  const double* weights;  // null: norms only
  int n_peers;
  Layout layout;
  bool tiled;
};

int check_round(const char* what, const Round& r, std::vector<int>* order) {
  const std::string w(what);
  if (r.n_peers < 1 || r.n_peers > kMostPeers)
    return fail(DLA_E_INVALID, w + ": n_peers must be 1.." + std::to_string(kMostPeers));
  if (r.n_tensors < 0) return fail(DLA_E_INVALID, w + ": n_tensors < 0");
  if (r.n_tensors > 0 && (!r.dtypes || !r.peers || !r.centers || !r.numels)) return fail(DLA_E_INVALID, w + ": null array");
  for (int t = 0; t < r.n_tensors; ++t) {
    if (!known_dtype(r.dtypes[t]))
      return fail(DLA_E_INVALID, w + ": tensor " + std::to_string(t) + " has unknown dtype " + std::to_string(r.dtypes[t]));
    if (r.numels[t] < 0 || r.numels[t] > kMostElems)
      return fail(DLA_E_INVALID, w + ": tensor " + std::to_string(t) + " has a bad element count");
    if (r.numels[t] == 0) continue;
    const int es = elem_bytes(r.dtypes[t]);
    if (!r.centers[t] || !aligned_to(r.centers[t], es))
      return fail(DLA_E_INVALID, w + ": centre tensor " + std::to_string(t) + " is null or not aligned");
    for (int k = 0; k < r.n_peers; ++k) {
      const void* p = r.peers[static_cast<int64_t>(t) * r.n_peers + k];
      if (!p || !aligned_to(p, es))
        return fail(DLA_E_INVALID, w + ": tensor " + std::to_string(t) + " of peer " + std::to_string(k) + " is null or not aligned");
    }
    order->push_back(t);
  }
  if (!r.outs || r.tiled) return DLA_OK;
  // an output may be the very buffer of its centre or of one of its peers (each element is read before it is
  // written, by the same lane); any other overlap is refused
  std::vector<Span> spans;
  for (int t : *order) {
    const int es = elem_bytes(r.dtypes[t]);
    if (!r.outs[t] || !aligned_to(r.outs[t], es))
      return fail(DLA_E_INVALID, w + ": out " + std::to_string(t) + " is null or not aligned");
    spans.push_back(span_of(r.outs[t], r.numels[t], es));
  }
  const std::vector<Span> own = spans;
  if (!disjoint(&spans)) return fail(DLA_E_ALIAS, w + ": two outputs overlap");
  for (size_t q = 0; q < order->size(); ++q) {
    const int t = (*order)[q], es = elem_bytes(r.dtypes[t]);
    if (meets(spans, span_of(r.centers[t], r.numels[t], es), own[q]))
      return fail(DLA_E_ALIAS, w + ": centre tensor " + std::to_string(t) + " overlaps an output that is not its own");
    for (int k = 0; k < r.n_peers; ++k)
      if (meets(spans, span_of(r.peers[static_cast<int64_t>(t) * r.n_peers + k], r.numels[t], es), own[q]))
        return fail(DLA_E_ALIAS, w + ": tensor " + std::to_string(t) + " of peer " + std::to_string(k) + " overlaps an output that is not its own");
  }
  return DLA_OK;
}

int64_t units_of(int64_t n, int dt, int unit_bytes) {
  const int64_t per = unit_bytes / elem_bytes(dt);
  return (n + per - 1) / per;
}

// Page-locked memory that kernels reach at the same address?
bool mapped_host(const void* p) {
  hipPointerAttribute_t a;
  const bool ok = hipPointerGetAttributes(&a, p) == hipSuccess && a.type == hipMemoryTypeHost && a.devicePointer == p;
  if (!ok) (void)hipGetLastError();
  return ok;
}

// The round's table: in `words` if it fits there, else in the workspace.
int make_table(const char* what, const Round& r, const std::vector<int>& order, int norm_unit, void* table_host,
               int64_t table_host_bytes, uint64_t* workspace, PutWords* words, Table* tab, int64_t* norm_units,
               int64_t* mean_units, hipStream_t s) {
  const int m = static_cast<int>(order.size());
  const int64_t n_words = peer_table_words(m, r.n_peers);
  const bool here = n_words <= kPutWords;
  const bool host = !here && table_host && table_host_bytes >= n_words * 8 && aligned_to(table_host, 8) && mapped_host(table_host);
  std::vector<uint64_t> built(here || host ? 0 : static_cast<size_t>(n_words));
  uint64_t* to = here ? words->w : host ? static_cast<uint64_t*>(table_host) : built.data();
  Seg* segs = reinterpret_cast<Seg*>(to);
  uint64_t* ptrs = to + m * (sizeof(Seg) / 8);
  int64_t un = 0, um = 0;
  for (int q = 0; q < m; ++q) {
    const int t = order[q], dt = r.dtypes[t];
    segs[q] = {un, um, static_cast<uint64_t>(r.numels[t]) * 4 + static_cast<uint64_t>(dt), r.centers[t], r.outs ? r.outs[t] : nullptr};
    for (int k = 0; k < r.n_peers; ++k)
      ptrs[static_cast<int64_t>(q) * r.n_peers + k] = reinterpret_cast<uint64_t>(r.peers[static_cast<int64_t>(t) * r.n_peers + k]);
    un += units_of(r.numels[t], dt, norm_unit);
    um += units_of(r.numels[t], dt, kMeanUnit);
  }
  if (r.weights) std::memcpy(ptrs + static_cast<int64_t>(m) * r.n_peers, r.weights, sizeof(double) * r.n_peers);
  *tab = {here ? nullptr : workspace, m, r.n_peers};
  *norm_units = un;
  *mean_units = um;
  if (host) {
    hipLaunchKernelGGL(fetch_kernel, dim3(static_cast<unsigned>((n_words + kThreads - 1) / kThreads)), dim3(kThreads), 0, s,
                       to, workspace, n_words);
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  for (size_t i = 0; i < built.size(); i += kPutWords) {
    PutWords blob;
    const int n = static_cast<int>(std::min<size_t>(kPutWords, built.size() - i));
    std::memcpy(blob.w, built.data() + i, sizeof(uint64_t) * n);
    hipLaunchKernelGGL(put_kernel, dim3(1), dim3(512), 0, s, blob, workspace + i, n);
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  return DLA_OK;
}

struct NormLaunch {
  const PutWords& words;
  Table tab;
  bool tiled;
  dim3 grid;
  hipStream_t s;
  int64_t units;
  Layout l;
  double* partials;
  uint32_t* counters;
  const Joined& to;
};
template <int G>
void launch_peer_norms(const NormLaunch& a) {
  if (a.tiled)
    hipLaunchKernelGGL((peer_norms_kernel<G, true>), a.grid, dim3(kThreads), 0, a.s, a.words, a.tab, a.units, a.l, a.partials, a.counters, a.to);
  else
    hipLaunchKernelGGL((peer_norms_kernel<G, false>), a.grid, dim3(kThreads), 0, a.s, a.words, a.tab, a.units, a.l, a.partials, a.counters, a.to);
}

// The norms (no sq_in), then the average (outs != null), of one round.
int round_impl(const char* what, const Round& r, double max_norm, const double* sq_in, double* sq_out, int out_dtype,
               void* norms, void* counters, void* table_host, int64_t table_host_bytes, void* workspace,
               int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_round(what, r, &order)) return rc;
  const std::string w(what);
  if (norms && ((out_dtype != DLA_F32 && out_dtype != DLA_F64) || !aligned_to(norms, elem_bytes(out_dtype))))
    return fail(DLA_E_INVALID, w + ": norms must be aligned F32 or F64 values");
  if (!aligned_to(sq_in, 8) || !aligned_to(sq_out, 8)) return fail(DLA_E_INVALID, w + ": squared norms are not aligned");
  if (!aligned_to(counters, 4)) return fail(DLA_E_INVALID, w + ": counters are not aligned");
  if (r.outs && !r.weights) return fail(DLA_E_INVALID, w + ": null weights");
  if (r.outs && !(max_norm >= 0)) return fail(DLA_E_INVALID, w + ": max_norm must be >= 0");
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < peer_workspace_bytes(r.n_tensors, r.n_peers))
    return fail(DLA_E_INVALID, w + ": workspace is null, not aligned or smaller than dla_peer_workspace");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int m = static_cast<int>(order.size()), n = r.n_peers;
  uint64_t* table = static_cast<uint64_t*>(workspace);
  int64_t norm_units = 0, mean_units = 0;
  PutWords words;
  Table tab;
  if (int rc = make_table(what, r, order, unit_bytes(peer_vec(r.tiled)), table_host, table_host_bytes, table, &words,
                          &tab, &norm_units, &mean_units, s))
    return rc;
  double* shares = reinterpret_cast<double*>(table + peer_table_words(r.n_tensors, n));
  double* partials = shares + share_words(n);
  const Joined to = {sq_in, sq_out, norms, out_dtype, r.outs ? shares : nullptr, reinterpret_cast<float*>(shares + n), max_norm};
  int64_t blocks = 0;
  if (!sq_in && m > 0) {
    const int groups = peer_groups(n), g = (n + groups - 1) / groups;
    blocks = std::min(norm_units, peer_blocks(n));
    // large rounds join in a kernel of its own: its launch hides behind the round, the last workgroup's join does
    // not (us, apart / in the last workgroup: 8 x 25 M f32 138.6 / 141.6; but 2 x 85 K f32 with the average 15.5 / 12.7)
    if (blocks * groups > 512) counters = nullptr;
    const NormLaunch a = {words, tab, r.tiled, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>((n + g - 1) / g)), s,
                          norm_units, r.layout, partials, static_cast<uint32_t*>(counters), to};
    switch (g) {
      case 1: launch_peer_norms<1>(a); break;
      case 2: launch_peer_norms<2>(a); break;
      case 3: launch_peer_norms<3>(a); break;
      case 4: launch_peer_norms<4>(a); break;
      case 5: launch_peer_norms<5>(a); break;
      case 6: launch_peer_norms<6>(a); break;
      case 7: launch_peer_norms<7>(a); break;
      default: launch_peer_norms<8>(a); break;
    }
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  if (!counters || blocks == 0) {
    hipLaunchKernelGGL(peer_join_kernel, dim3(static_cast<unsigned>(n)), dim3(64), 0, s, words, tab, partials,
                       static_cast<int>(blocks), to);
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  if (!r.outs || m == 0) return DLA_OK;
  const dim3 grid(static_cast<unsigned>(dla_internal_grid(mean_units, kMeanThreads)));
  // One wave per workgroup and 8 + 1 loads in flight per wave: beyond some 100 KB in flight per CU more waves only
  // keep more DRAM rows open at once.  Rounds of 8 peers and more that read over the Infinity Cache's 256 MB run
  // 14 waves per CU, by reserving LDS that nothing reads (us, 14 / uncapped: 8 x 25 M f32 157 / 165; reading 800 MB in f32,
  // 8 peers 137.7 / 153.5, 16 135.1 / 144.8, 32 137.0 / 142.4, 64 135.8 / 135.1; 320 MB, 8 peers 59.1 / 62.1, 16 58.9 / 59.8;
  // bf16 and f64 alike).  Fewer peers lose by it (4 peers, 800 MB 158.1 / 154.1, 7 peers, 320 MB 63.8 / 59.7), smaller
  // rounds tie (200 MB, 8 peers 39.6 / 39.2, 32 37.4 / 37.3).
  double bytes = 0;
  for (int t : order) bytes += static_cast<double>(r.numels[t]) * elem_bytes(r.dtypes[t]) * (n + 1);
  const int lds = n >= 8 && bytes > kInfinityCache ? 160 * 1024 / 14 : 0;
  if (r.tiled)
    hipLaunchKernelGGL((bounded_kernel<true>), grid, dim3(kMeanThreads), lds, s, words, tab, mean_units, shares, r.layout);
  else hipLaunchKernelGGL((bounded_kernel<false>), grid, dim3(kMeanThreads), lds, s, words, tab, mean_units, shares, r.layout);
  if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  return DLA_OK;
}

// The round of a tile-interleaved slab as a Round of one tensor.
struct SlabRound {
  Round r;
  std::vector<const void*> peers;
  const void* center;
  void* out;
  int dtype;
  int64_t n_elems;
};
int slab_round(const char* what, SlabRound* sr, int dtype, const void* base, int64_t tile_elems, int64_t slab_rows,
               const void* center, int n_peers, int64_t n_elems, void* out, const double* weights) {
  const std::string w(what);
  if (!known_dtype(dtype)) return fail(DLA_E_INVALID, w + ": unknown dtype " + std::to_string(dtype));
  if (n_elems < 0 || n_elems > kMostElems) return fail(DLA_E_INVALID, w + ": bad element count");
  const int es = elem_bytes(dtype);
  if (!base || !aligned_to(base, 16) || tile_elems < 1 || tile_elems > (int64_t{1} << 30) || tile_elems * es < 16 || (tile_elems & (tile_elems - 1)))
    return fail(DLA_E_INVALID, w + ": base must be 16-byte aligned and tile_elems a power of two of >= 16 bytes");
  if (static_cast<double>(n_elems + tile_elems) * es * static_cast<double>(slab_rows) > static_cast<double>(kMostElems))
    return fail(DLA_E_INVALID, w + ": slab_rows x n_elems is beyond any device");
  if (n_peers < 1 || n_peers > kMostPeers || slab_rows < n_peers)
    return fail(DLA_E_INVALID, w + ": need 1 <= n_peers <= slab_rows and n_peers <= " + std::to_string(kMostPeers));
  int shift = 0;
  while ((int64_t{1} << shift) < tile_elems) ++shift;
  sr->dtype = dtype;
  sr->n_elems = n_elems;
  sr->center = center ? center : base;
  sr->out = out;
  for (int k = 0; k < n_peers; ++k) sr->peers.push_back(static_cast<const char*>(base) + k * tile_elems * es);
  const int64_t stride = slab_rows * tile_elems;
  sr->r = {1, &sr->dtype, sr->peers.data(), &sr->center, out ? &sr->out : nullptr, &sr->n_elems, weights, n_peers,
           {shift, stride, center ? tile_elems : stride}, true};
  if (out && n_elems > 0) {
    if (!aligned_to(out, es) || (center && !aligned_to(center, es))) return fail(DLA_E_INVALID, w + ": out / center not aligned");
    const Span o = span_of(out, n_elems, es), b = span_of(base, (n_elems + tile_elems - 1) / tile_elems * stride, es);
    const Span c = span_of(sr->center, n_elems, es);
    if ((o.begin < b.end && b.begin < o.end) || (center && o.begin < c.end && c.begin < o.end && o.begin != c.begin))
      return fail(DLA_E_ALIAS, w + ": out overlaps the slab, or the centre without being it");
  }
  return DLA_OK;
}

// No C++ exception crosses the ABI.
template <class F>
int guarded(const char* what, F f) {
  dla_internal_clear_error();
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return dla_internal_fail(DLA_E_INVALID, "no memory");
  } catch (const std::exception& e) {
    return fail(DLA_E_INVALID, std::string(what) + ": " + e.what());
  } catch (...) {
    return fail(DLA_E_INVALID, std::string(what) + ": unknown error");
  }
}

}  // namespace

extern "C" {

int64_t dla_norm_workspace(int n_tensors) {
  if (n_tensors < 0) return 0;
  return 8 * (static_cast<int64_t>(1) + kMaxPartials + n_tensors / kNormTensors + 1);
}

int dla_norm(int n_tensors, const int* dtypes, const void* const* tensors, const int64_t* numels, int norm, int out_dtype,
             void* out, void* counter, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_norm", [&] {
    return norm_impl(n_tensors, dtypes, tensors, numels, norm, out_dtype, out, counter, workspace, workspace_bytes, stream);
  });
}

int dla_norm_clip(int n_tensors, const int* dtypes, const void* const* tensors, void* const* outs, const int64_t* numels,
                  int norm, double max_norm, double eps, int out_dtype, void* norm_out, void* counter, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  return guarded("dla_norm_clip", [&] {
    return norm_clip_impl(n_tensors, dtypes, tensors, outs, numels, norm, max_norm, eps, out_dtype, norm_out, counter,
                          workspace, workspace_bytes, stream);
  });
}

int64_t dla_peer_workspace(int n_tensors, int n_peers) {
  if (n_tensors < 0 || n_peers < 1 || n_peers > kMostPeers) return 0;
  return peer_workspace_bytes(n_tensors, n_peers);
}

int64_t dla_peer_table(int n_tensors, int n_peers) {
  if (n_tensors < 0 || n_peers < 1 || n_peers > kMostPeers) return 0;
  const int64_t words = peer_table_words(n_tensors, n_peers);
  return words <= kPutWords ? 0 : words * 8;
}

int dla_peer_norms(int n_tensors, const int* dtypes, const void* const* peer_ptrs, const void* const* centers,
                   const int64_t* numels, int n_peers, double* sq_out, int out_dtype, void* norms, void* counters,
                   void* table_host, int64_t table_host_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_peer_norms", [&] {
    const Round r = {n_tensors, dtypes, peer_ptrs, centers, nullptr, numels, nullptr, n_peers, {0, 0, 0}, false};
    return round_impl("dla_peer_norms", r, 0, nullptr, sq_out, out_dtype, norms, counters, table_host,
                      table_host_bytes, workspace, workspace_bytes, stream);
  });
}

int dla_wsum_bounded(int n_tensors, const int* dtypes, const void* const* peer_ptrs, const void* const* centers,
                     void* const* outs, const int64_t* numels, const double* weights, int n_peers, double max_norm,
                     const double* sq, int out_dtype, void* norms, void* counters, void* table_host,
                     int64_t table_host_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_wsum_bounded", [&] {
    if (!outs && n_tensors > 0) return fail(DLA_E_INVALID, "dla_wsum_bounded: null outs array");
    static void* const none[1] = {nullptr};
    const Round r = {n_tensors, dtypes, peer_ptrs, centers, outs ? outs : none, numels, weights, n_peers, {0, 0, 0}, false};
    return round_impl("dla_wsum_bounded", r, max_norm, sq, nullptr, out_dtype, norms, counters, table_host,
                      table_host_bytes, workspace, workspace_bytes, stream);
  });
}

int dla_wsum_bounded_slab_tiled(int dtype, const void* base, int64_t tile_elems, int64_t slab_rows, const void* center,
                                const double* weights, int n_peers, int64_t n_elems, double max_norm, void* out,
                                int out_dtype, void* norms, void* counters, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  return guarded("dla_wsum_bounded_slab_tiled", [&] {
    if (!out && n_elems > 0) return fail(DLA_E_INVALID, "dla_wsum_bounded_slab_tiled: null out");
    SlabRound sr;
    if (int rc = slab_round("dla_wsum_bounded_slab_tiled", &sr, dtype, base, tile_elems, slab_rows, center, n_peers, n_elems, out, weights))
      return rc;
    return round_impl("dla_wsum_bounded_slab_tiled", sr.r, max_norm, nullptr, nullptr, out_dtype, norms, counters,
                      nullptr, 0, workspace, workspace_bytes, stream);
  });
}

}  // extern "C"
