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
// Sums of squares, norms and averages are carried in 64 bits whatever the storage type: a vector FMA in
// f64 issues at the rate of one in f32 on this chip, the kernels wait for memory either way, and the
// square of any f32 value is a normal f64, so no norm of finite 32- or 16-bit values overflows or
// underflows.  A result is rounded to its storage type once (16-bit types through f32: the second
// rounding moves a result by less than 2^-24 of itself before the last one).
//
// Work is cut into units of 4 KiB (16 bytes per lane of a 256-thread workgroup) or 16 KiB of one tensor;
// a unit never spans tensors.  Workgroup b of P takes units [b U / P, (b + 1) U / P): one partial result
// per workgroup whatever the size, added up in a fixed order by the kernel that needs the sum, so the
// results do not depend on which workgroup ended first.  Loads need element alignment only (gfx950
// takes 16-byte loads from any address), so tensors that start anywhere take the same path.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>
#include <string>
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
  static __device__ inline void widen(u32x4 r, double (&v)[E]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = static_cast<double>(__uint_as_float(r[i] << 16));
      v[2 * i + 1] = static_cast<double>(__uint_as_float(r[i] & 0xffff0000u));
    }
  }
  static __device__ inline u32x4 narrow(const double (&v)[E]) {
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
  static __device__ inline void widen(u32x4 r, double (&v)[E]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h2 h;
      const uint32_t w = r[i];
      __builtin_memcpy(&h, &w, 4);
      v[2 * i] = static_cast<double>(static_cast<float>(h[0]));
      v[2 * i + 1] = static_cast<double>(static_cast<float>(h[1]));
    }
  }
  static __device__ inline u32x4 narrow(const double (&v)[E]) {
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
template <int DT>
__device__ inline u32x4 load_full(const void* base, int64_t j) {
  using B = typename Elem<DT>::bits;
  return *(const u32x4_any __attribute__((address_space(1)))*)(global_ptr<B>(base) + j);
}
template <int DT>
__device__ inline void store_part(void* base, int64_t j, int n, u32x4 r) {
  using B = typename Elem<DT>::bits;
  constexpr int E = Elem<DT>::E;
  auto* p = global_ptr<B>(base) + j;
  if (n >= E) {
    *(u32x4_any __attribute__((address_space(1)))*)p = r;
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
template <int NORM>
__device__ inline double join_partials(const double* partials, int n, double* lds) {
  double v = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = norm_join<NORM>(v, global_ptr<double>(partials)[i]);
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
constexpr int kVec = 4;                             // 16-byte loads in flight per lane
constexpr int kUnitBytes = kThreads * 16 * kVec;    // 16 KiB of one tensor
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

template <int NORM, int DT>
__device__ inline void norm_unit(const void* p, int64_t n, int64_t unit, double (&acc)[kVec]) {
  constexpr int E = Elem<DT>::E;
  const int64_t j0 = unit * (kThreads * kVec * E) + static_cast<int>(threadIdx.x) * E;
  u32x4 r[kVec];
  if ((unit + 1) * (kThreads * kVec * E) <= n) {
#pragma unroll
    for (int v = 0; v < kVec; ++v) r[v] = load_full<DT>(p, j0 + v * (kThreads * E));
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

// Workgroup b's part of the norm of a list: partials[b].
template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_kernel(const TensorList<kNormTensors> tab, int count, uint32_t units,
                                                        double* partials) {
  __shared__ double lds[kWaves];
  const uint32_t b = blockIdx.x, nb = gridDim.x;
  uint32_t u = static_cast<uint32_t>(static_cast<uint64_t>(units) * b / nb);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(units) * (b + 1) / nb);
  int t = find_tensor(tab.unit0, count, u);
  double acc[kVec] = {};
  while (u < end) {
    const uint32_t first = tab.unit0[t];
    uint32_t stop = t + 1 < count ? tab.unit0[t + 1] : units;
    if (stop > end) stop = end;
    const void* p = tab.p[t];
    const uint64_t nd = tab.n_dt[t];
    const int64_t n = static_cast<int64_t>(nd >> 2);
    switch (nd & 3) {
      case DLA_F32: for (; u < stop; ++u) norm_unit<NORM, DLA_F32>(p, n, u - first, acc); break;
      case DLA_BF16: for (; u < stop; ++u) norm_unit<NORM, DLA_BF16>(p, n, u - first, acc); break;
      case DLA_F16: for (; u < stop; ++u) norm_unit<NORM, DLA_F16>(p, n, u - first, acc); break;
      default: for (; u < stop; ++u) norm_unit<NORM, DLA_F64>(p, n, u - first, acc); break;
    }
    ++t;
  }
  double v = acc[0];
#pragma unroll
  for (int i = 1; i < kVec; ++i) v = norm_join<NORM>(v, acc[i]);
  v = block_join<NORM>(v, lds);
  if (threadIdx.x == 0) global_ptr<double>(partials)[b] = v;
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_join_kernel(const double* partials, int n, int out_dt, void* out) {
  __shared__ double lds[kWaves];
  const double v = join_partials<NORM>(partials, n, lds);
  if (threadIdx.x == 0) put_norm(out, 0, out_dt, v);
}

template <int DT>
__device__ inline void scale_unit(const void* p, void* out, int64_t n, int64_t unit, double ratio) {
  constexpr int E = Elem<DT>::E;
  const int64_t j0 = unit * (kThreads * kVec * E) + static_cast<int>(threadIdx.x) * E;
  const bool full = (unit + 1) * (kThreads * kVec * E) <= n;
  u32x4 r[kVec];
  int part[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int64_t j = j0 + v * (kThreads * E);
    part[v] = full ? E : clamp_part(n - j, E);
    r[v] = full ? load_full<DT>(p, j) : load_part<DT>(p, j, part[v]);
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

// y = round(x * min(1, M / (n + eps))).  Every workgroup joins the partials itself (8 KB that all of them
// read: less than a launch between the two kernels costs) and then walks its units backwards: what the
// norm read last is what the caches still hold.
template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_scale_kernel(const TensorsInOut<kScaleTensors> tab, int count,
                                                              uint32_t units, const double* partials, int n_partials,
                                                              double max_norm, double eps, int in_place, int out_dt,
                                                              void* norm_out) {
  __shared__ double lds[kWaves];
  const double norm = join_partials<NORM>(partials, n_partials, lds);
  const uint32_t b = blockIdx.x, nb = gridDim.x;
  if (b == 0 && threadIdx.x == 0 && norm_out) put_norm(norm_out, 0, out_dt, norm);
  const double q = max_norm / (norm + eps);
  const double ratio = q > 1.0 ? 1.0 : q;  // NaN stays NaN
  if (in_place && ratio == 1.0) return;    // x * 1 = x: nothing to write
  const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(units) * b / nb);
  uint32_t u = static_cast<uint32_t>(static_cast<uint64_t>(units) * (b + 1) / nb);
  if (u == begin) return;
  int t = find_tensor(tab.in.unit0, count, u - 1);
  while (u > begin) {
    const uint32_t first = tab.in.unit0[t];
    const uint32_t stop = first > begin ? first : begin;
    const void* p = tab.in.p[t];
    void* out = tab.out[t];
    const uint64_t nd = tab.in.n_dt[t];
    const int64_t n = static_cast<int64_t>(nd >> 2);
    switch (nd & 3) {
      case DLA_F32: for (; u > stop; --u) scale_unit<DLA_F32>(p, out, n, u - 1 - first, ratio); break;
      case DLA_BF16: for (; u > stop; --u) scale_unit<DLA_BF16>(p, out, n, u - 1 - first, ratio); break;
      case DLA_F16: for (; u > stop; --u) scale_unit<DLA_F16>(p, out, n, u - 1 - first, ratio); break;
      default: for (; u > stop; --u) scale_unit<DLA_F64>(p, out, n, u - 1 - first, ratio); break;
    }
    --t;
  }
}

// ------------------------------------------------------------- peers around a centre
// The round's table in device memory: a record per tensor, then the peers' pointers (tensor-major), then the
// weights.  It goes there by value, as arguments of put_kernel, so a captured graph holds its own copy.
struct Seg {
  int64_t unit0;  // first unit (4 KiB of one tensor of one peer)
  int64_t n;
  const void* center;
  void* out;
  int64_t dt;
};
struct Layout {      // where element j of a peer (and of the centre) lies, in elements from its pointer:
  int shift;         //   (j >> shift) * stride + (j & (2^shift - 1)) in a tile-interleaved slab
  int64_t stride;
  int64_t center_stride;
};
constexpr int kPeerUnit = kThreads * 16;
constexpr int kPutWords = 480;
struct PutWords {
  uint64_t w[kPutWords];
};
__global__ __launch_bounds__(512) void put_kernel(const PutWords words, uint64_t* dst, int n) {
  const int i = static_cast<int>(threadIdx.x);
  if (i < n) global_ptr<uint64_t>(dst)[i] = words.w[i];
}

template <bool TILED>
__device__ inline int64_t place(const Layout& l, int64_t stride, int64_t j) {
  return TILED ? (j >> l.shift) * stride + (j & ((int64_t{1} << l.shift) - 1)) : j;
}

// The tensor that unit u lies in: a 64-way search by the wave's lanes over the records' first units.
__device__ inline int find_seg(const Seg* segs, int count, int64_t u) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const int below = __popcll(__ballot(i < hi && global_ptr<Seg>(segs)[i < hi ? i : lo].unit0 <= u));
    lo = __builtin_amdgcn_readfirstlane(lo + (below - 1) * step);
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

template <int DT, int G, bool TILED>
__device__ inline void peer_norm_unit(const Layout& l, const void* center, const void* const (&p)[G], int64_t n,
                                      int64_t unit, double (&acc)[G]) {
  constexpr int E = Elem<DT>::E;
  const int64_t j = unit * (kThreads * E) + static_cast<int>(threadIdx.x) * E;
  const int64_t at = place<TILED>(l, l.stride, j), at_c = place<TILED>(l, l.center_stride, j);
  u32x4 rc, r[G];
  if ((unit + 1) * (kThreads * E) <= n) {
    rc = load_full<DT>(center, at_c);
#pragma unroll
    for (int g = 0; g < G; ++g) r[g] = load_full<DT>(p[g], at);
  } else {
    const int part = clamp_part(n - j, E);
    rc = load_part<DT>(center, at_c, part);
#pragma unroll
    for (int g = 0; g < G; ++g) r[g] = load_part<DT>(p[g], at, part);
  }
  double c[E];
  Elem<DT>::widen(rc, c);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    double x[E];
    Elem<DT>::widen(r[g], x);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const double d = x[i] - c[i];
      acc[g] = __builtin_fma(d, d, acc[g]);
    }
  }
}

// partials[k * gridDim.x + b]: workgroup b's part of || p_k - c ||^2 for the peers of group blockIdx.y.  G
// peers are read beside one read of the centre, so the centre costs 1 / G of a peer.
template <int G, bool TILED>
__global__ __launch_bounds__(kThreads) void peer_norms_kernel(const Seg* segs, int count, int64_t units,
                                                              const uint64_t* ptrs, int n_peers, Layout l,
                                                              double* partials) {
  __shared__ double lds[kWaves];
  const int64_t b = blockIdx.x, nb = gridDim.x;
  const int k0 = static_cast<int>(blockIdx.y) * G;
  int64_t u = units * b / nb;
  const int64_t end = units * (b + 1) / nb;
  int t = find_seg(segs, count, u);
  double acc[G] = {};
  while (u < end) {
    const auto* s = const_ptr<Seg>(segs) + t;
    const int64_t first = s->unit0, n = s->n;
    int64_t stop = t + 1 < count ? s[1].unit0 : units;
    if (stop > end) stop = end;
    const void* center = s->center;
    const void* p[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int k = k0 + g < n_peers ? k0 + g : n_peers - 1;  // a spare place reads the last peer again
      p[g] = reinterpret_cast<const void*>(const_ptr<uint64_t>(ptrs)[static_cast<int64_t>(t) * n_peers + k]);
    }
    switch (s->dt) {
      case DLA_F32: for (; u < stop; ++u) peer_norm_unit<DLA_F32, G, TILED>(l, center, p, n, u - first, acc); break;
      case DLA_BF16: for (; u < stop; ++u) peer_norm_unit<DLA_BF16, G, TILED>(l, center, p, n, u - first, acc); break;
      case DLA_F16: for (; u < stop; ++u) peer_norm_unit<DLA_F16, G, TILED>(l, center, p, n, u - first, acc); break;
      default: for (; u < stop; ++u) peer_norm_unit<DLA_F64, G, TILED>(l, center, p, n, u - first, acc); break;
    }
    ++t;
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const double v = block_join<DLA_NORM_L2>(acc[g], lds);
    if (threadIdx.x == 0 && k0 + g < n_peers) global_ptr<double>(partials)[(k0 + g) * nb + b] = v;
  }
}

// sq[k] = the sum of peer k's partials (n of them, possibly none); norms[k] = its root.
__global__ __launch_bounds__(kThreads) void peer_join_kernel(const double* partials, int n, double* sq, int out_dt,
                                                             void* norms) {
  __shared__ double lds[kWaves];
  const int k = static_cast<int>(blockIdx.x);
  double v = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) v += global_ptr<double>(partials)[static_cast<int64_t>(k) * n + i];
  v = block_join<DLA_NORM_L2>(v, lds);
  if (threadIdx.x == 0) {
    global_ptr<double>(sq)[k] = v;
    if (norms) put_norm(norms, k, out_dt, __builtin_sqrt(v));
  }
}

// The peers that count, in list order, in LDS: their share a_k and their pointer for the tensor at hand.
struct Live {
  double* share;
  uint64_t* ptr;
  int* k;
};

template <int DT, int G, bool TILED>
__device__ inline void fold_peers(const Live& live, int i0, int64_t at, int part, bool full,
                                  const double (&c)[Elem<DT>::E], double (&acc)[Elem<DT>::E]) {
  constexpr int E = Elem<DT>::E;
  u32x4 r[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const void* p = reinterpret_cast<const void*>(live.ptr[i0 + g]);
    r[g] = full ? load_full<DT>(p, at) : load_part<DT>(p, at, part);
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const double a = live.share[i0 + g];
    double x[E];
    Elem<DT>::widen(r[g], x);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = __builtin_fma(a, x[i] - c[i], acc[i]);
  }
}

template <int DT, bool TILED>
__device__ inline void bounded_unit(const Layout& l, const Live& live, int m, const void* center, void* out, int64_t n,
                                    int64_t unit) {
  constexpr int E = Elem<DT>::E;
  const int64_t j = unit * (kThreads * E) + static_cast<int>(threadIdx.x) * E;
  const int64_t at = place<TILED>(l, l.stride, j), at_c = place<TILED>(l, l.center_stride, j);
  const bool full = (unit + 1) * (kThreads * E) <= n;
  const int part = full ? E : clamp_part(n - j, E);
  double c[E], acc[E] = {};
  Elem<DT>::widen(full ? load_full<DT>(center, at_c) : load_part<DT>(center, at_c, part), c);
  int i = 0;
  for (; i + 8 <= m; i += 8) fold_peers<DT, 8, TILED>(live, i, at, part, full, c, acc);
  if (i + 4 <= m) {
    fold_peers<DT, 4, TILED>(live, i, at, part, full, c, acc);
    i += 4;
  }
  if (i + 2 <= m) {
    fold_peers<DT, 2, TILED>(live, i, at, part, full, c, acc);
    i += 2;
  }
  if (i < m) fold_peers<DT, 1, TILED>(live, i, at, part, full, c, acc);
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] += c[e];
  store_part<DT>(out, j, part, Elem<DT>::narrow(acc));
}

// out = round(c + sum_k a_k (p_k - c)).  Units are walked from the last to the first: what the norms read
// last is what the caches still hold.
template <bool TILED>
__global__ __launch_bounds__(kThreads) void bounded_kernel(const Seg* segs, int count, int64_t units,
                                                           const uint64_t* ptrs, const double* weights, int n_peers,
                                                           Layout l, double max_norm, const double* sq, int out_dt,
                                                           void* norms) {
  extern __shared__ double lds[];
  __shared__ int n_live;
  Live live;
  live.share = lds;
  live.ptr = reinterpret_cast<uint64_t*>(lds + n_peers);
  live.k = reinterpret_cast<int*>(lds + 2 * n_peers);
  if (threadIdx.x < 64) {
    int m = 0;
    for (int k0 = 0; k0 < n_peers; k0 += 64) {
      const int k = k0 + static_cast<int>(threadIdx.x);
      double norm = 0, share = 0;
      if (k < n_peers) {
        norm = __builtin_sqrt(global_ptr<double>(sq)[k]);
        share = global_ptr<double>(weights)[k] * (norm <= max_norm ? 1.0 : max_norm / norm);
        if (blockIdx.x == 0 && norms) put_norm(norms, k, out_dt, norm);
      }
      const bool counts = k < n_peers && __builtin_isfinite(norm) && share != 0.0;
      const uint64_t mask = __ballot(counts);
      if (counts) {
        const int at = m + __popcll(mask & ((uint64_t{1} << threadIdx.x) - 1));
        live.share[at] = share;
        live.k[at] = k;
      }
      m += __popcll(mask);
    }
    if (threadIdx.x == 0) n_live = m;
  }
  __syncthreads();
  const int m = __builtin_amdgcn_readfirstlane(n_live);
  const int64_t b = blockIdx.x, nb = gridDim.x;
  const int64_t begin = units * b / nb;
  int64_t u = units * (b + 1) / nb;
  if (u == begin) return;
  int t = find_seg(segs, count, u - 1);
  while (u > begin) {
    const auto* s = const_ptr<Seg>(segs) + t;
    const int64_t first = s->unit0, n = s->n;
    const int64_t stop = first > begin ? first : begin;
    const void* center = s->center;
    void* out = s->out;
    for (int i = threadIdx.x; i < m; i += kThreads)
      live.ptr[i] = global_ptr<uint64_t>(ptrs)[static_cast<int64_t>(t) * n_peers + live.k[i]];
    __syncthreads();
    switch (s->dt) {
      case DLA_F32: for (; u > stop; --u) bounded_unit<DLA_F32, TILED>(l, live, m, center, out, n, u - 1 - first); break;
      case DLA_BF16: for (; u > stop; --u) bounded_unit<DLA_BF16, TILED>(l, live, m, center, out, n, u - 1 - first); break;
      case DLA_F16: for (; u > stop; --u) bounded_unit<DLA_F16, TILED>(l, live, m, center, out, n, u - 1 - first); break;
      default: for (; u > stop; --u) bounded_unit<DLA_F64, TILED>(l, live, m, center, out, n, u - 1 - first); break;
    }
    __syncthreads();  // live.ptr is filled again for the next tensor
    --t;
  }
}

// ------------------------------------------------------------------ host side
int fail(int code, const std::string& msg) { return dla_internal_fail(code, msg.c_str()); }
int hip_fail(const char* what, hipError_t e) { return fail(static_cast<int>(e), std::string(what) + ": " + hipGetErrorString(e)); }

bool known_dtype(int dt) { return dt == DLA_F32 || dt == DLA_BF16 || dt == DLA_F16 || dt == DLA_F64; }
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// No element count here exceeds this: 2^56 bytes, far beyond any device, keeps every product below in 64 bits.
constexpr int64_t kMostElems = int64_t{1} << 53;

// The launches a list of tensors takes: tensors [begin, end) of `order` (the non-empty ones), `units` units
// on `blocks` workgroups whose partials start at `partial0`.
struct ListLaunch {
  int begin, end;
  uint32_t units;
  int blocks, partial0;
};

int64_t list_units(int dt, int64_t n) {
  const int64_t per = kUnitBytes / elem_bytes(dt);
  return (n + per - 1) / per;
}

bool plan_list(const std::vector<int>& order, const int* dtypes, const int64_t* numels, int per_launch, int most_blocks,
               std::vector<ListLaunch>* out, int* partials) {
  int64_t total = 0;
  for (int t : order) total += list_units(dtypes[t], numels[t]);
  int p0 = 0;
  for (size_t i = 0; i < order.size(); i += per_launch) {
    const int end = static_cast<int>(std::min(order.size(), i + per_launch));
    int64_t units = 0;
    for (int q = static_cast<int>(i); q < end; ++q) units += list_units(dtypes[order[q]], numels[order[q]]);
    if (units > 0xffffffffll) return false;
    int64_t blocks = std::min<int64_t>(units, most_blocks);
    if (total > units) blocks = std::max<int64_t>(1, std::min<int64_t>(blocks, most_blocks * units / total));
    out->push_back({static_cast<int>(i), end, static_cast<uint32_t>(units), static_cast<int>(blocks), p0});
    p0 += static_cast<int>(blocks);
  }
  *partials = p0;
  return true;
}

template <int M>
void fill_list(TensorList<M>* tab, const ListLaunch& l, const std::vector<int>& order, const int* dtypes,
               const void* const* tensors, const int64_t* numels) {
  std::memset(tab, 0, sizeof(*tab));
  uint32_t u = 0;
  for (int q = l.begin; q < l.end; ++q) {
    const int t = order[q], i = q - l.begin;
    tab->p[i] = tensors[t];
    tab->n_dt[i] = static_cast<uint64_t>(numels[t]) * 4 + static_cast<uint64_t>(dtypes[t]);
    tab->unit0[i] = u;
    u += static_cast<uint32_t>(list_units(dtypes[t], numels[t]));
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
    if (!known_dtype(dtypes[t])) return fail(DLA_E_INVALID, std::string(what) + ": tensor " + std::to_string(t) + " has unknown dtype " + std::to_string(dtypes[t]));
    if (numels[t] < 0 || numels[t] > kMostElems) return fail(DLA_E_INVALID, std::string(what) + ": tensor " + std::to_string(t) + " has a bad element count");
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

int norm_impl(int n_tensors, const int* dtypes, const void* const* tensors, const int64_t* numels, int norm, int out_dtype,
              void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_list("dla_norm", n_tensors, dtypes, tensors, numels, norm, &order)) return rc;
  if (out && ((out_dtype != DLA_F32 && out_dtype != DLA_F64) || !aligned_to(out, elem_bytes(out_dtype))))
    return fail(DLA_E_INVALID, "dla_norm: out must be an aligned F32 or F64 value");
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < dla_norm_workspace(n_tensors))
    return fail(DLA_E_INVALID, "dla_norm: workspace is null, not aligned or smaller than dla_norm_workspace");
  std::vector<ListLaunch> launches;
  int n_partials = 0;
  if (!plan_list(order, dtypes, numels, kNormTensors, kMaxPartials, &launches, &n_partials))
    return fail(DLA_E_INVALID, "dla_norm: too many elements");
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* partials = static_cast<double*>(workspace);
  for (const ListLaunch& l : launches) {
    TensorList<kNormTensors> tab;
    fill_list(&tab, l, order, dtypes, tensors, numels);
    const dim3 grid(static_cast<unsigned>(l.blocks));
    const int count = l.end - l.begin;
    double* to = partials + l.partial0;
    if (norm == DLA_NORM_L2) hipLaunchKernelGGL((norm_kernel<DLA_NORM_L2>), grid, dim3(kThreads), 0, s, tab, count, l.units, to);
    else if (norm == DLA_NORM_L1) hipLaunchKernelGGL((norm_kernel<DLA_NORM_L1>), grid, dim3(kThreads), 0, s, tab, count, l.units, to);
    else hipLaunchKernelGGL((norm_kernel<DLA_NORM_INF>), grid, dim3(kThreads), 0, s, tab, count, l.units, to);
    if (hipError_t e = hipGetLastError()) return hip_fail("dla_norm", e);
  }
  if (out) {
    if (norm == DLA_NORM_L2) hipLaunchKernelGGL((norm_join_kernel<DLA_NORM_L2>), dim3(1), dim3(kThreads), 0, s, partials, n_partials, out_dtype, out);
    else if (norm == DLA_NORM_L1) hipLaunchKernelGGL((norm_join_kernel<DLA_NORM_L1>), dim3(1), dim3(kThreads), 0, s, partials, n_partials, out_dtype, out);
    else hipLaunchKernelGGL((norm_join_kernel<DLA_NORM_INF>), dim3(1), dim3(kThreads), 0, s, partials, n_partials, out_dtype, out);
    if (hipError_t e = hipGetLastError()) return hip_fail("dla_norm", e);
  }
  return DLA_OK;
}

int norm_scale_impl(int n_tensors, const int* dtypes, const void* const* tensors, void* const* outs, const int64_t* numels,
                    int norm, double max_norm, double eps, int out_dtype, void* norm_out, const void* workspace,
                    int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_list("dla_norm_scale", n_tensors, dtypes, tensors, numels, norm, &order)) return rc;
  if (!(max_norm >= 0) || !(eps >= 0)) return fail(DLA_E_INVALID, "dla_norm_scale: max_norm and eps must be >= 0");
  if (norm_out && ((out_dtype != DLA_F32 && out_dtype != DLA_F64) || !aligned_to(norm_out, elem_bytes(out_dtype))))
    return fail(DLA_E_INVALID, "dla_norm_scale: norm_out must be an aligned F32 or F64 value");
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < dla_norm_workspace(n_tensors))
    return fail(DLA_E_INVALID, "dla_norm_scale: workspace is null, not aligned or smaller than dla_norm_workspace");
  if (!order.empty() && !outs) return fail(DLA_E_INVALID, "dla_norm_scale: null outs array");
  std::vector<Span> spans;
  bool in_place = true;
  for (int t : order) {
    if (!outs[t] || !aligned_to(outs[t], elem_bytes(dtypes[t])))
      return fail(DLA_E_INVALID, "dla_norm_scale: out " + std::to_string(t) + " is null or not aligned to its elements");
    spans.push_back(span_of(outs[t], numels[t], elem_bytes(dtypes[t])));
    in_place = in_place && outs[t] == tensors[t];
  }
  const std::vector<Span> own = spans;
  if (!disjoint(&spans)) return fail(DLA_E_ALIAS, "dla_norm_scale: two outputs overlap");
  for (size_t q = 0; q < order.size() && !in_place; ++q)
    if (meets(spans, span_of(tensors[order[q]], numels[order[q]], elem_bytes(dtypes[order[q]])), own[q]))
      return fail(DLA_E_ALIAS, "dla_norm_scale: tensor " + std::to_string(order[q]) + " overlaps an output that is not its own");
  std::vector<ListLaunch> parts, launches;
  int n_partials = 0, unused = 0;
  if (!plan_list(order, dtypes, numels, kNormTensors, kMaxPartials, &parts, &n_partials) ||
      !plan_list(order, dtypes, numels, kScaleTensors, 2 * kMaxPartials, &launches, &unused))
    return fail(DLA_E_INVALID, "dla_norm_scale: too many elements");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const double* partials = static_cast<const double*>(workspace);
  for (const ListLaunch& l : launches) {
    TensorsInOut<kScaleTensors> tab;
    fill_list(&tab.in, l, order, dtypes, tensors, numels);
    std::memset(tab.out, 0, sizeof(tab.out));
    for (int q = l.begin; q < l.end; ++q) tab.out[q - l.begin] = outs[order[q]];
    const dim3 grid(static_cast<unsigned>(l.blocks));
    const int count = l.end - l.begin, inp = in_place ? 1 : 0;
    void* no = l.begin == 0 ? norm_out : nullptr;
    if (norm == DLA_NORM_L2) hipLaunchKernelGGL((norm_scale_kernel<DLA_NORM_L2>), grid, dim3(kThreads), 0, s, tab, count, l.units, partials, n_partials, max_norm, eps, inp, out_dtype, no);
    else if (norm == DLA_NORM_L1) hipLaunchKernelGGL((norm_scale_kernel<DLA_NORM_L1>), grid, dim3(kThreads), 0, s, tab, count, l.units, partials, n_partials, max_norm, eps, inp, out_dtype, no);
    else hipLaunchKernelGGL((norm_scale_kernel<DLA_NORM_INF>), grid, dim3(kThreads), 0, s, tab, count, l.units, partials, n_partials, max_norm, eps, inp, out_dtype, no);
    if (hipError_t e = hipGetLastError()) return hip_fail("dla_norm_scale", e);
  }
  if (launches.empty() && norm_out) {  // nothing to scale: the norm of nothing is 0
    hipLaunchKernelGGL((norm_join_kernel<DLA_NORM_L1>), dim3(1), dim3(kThreads), 0, s, partials, 0, out_dtype, norm_out);
    if (hipError_t e = hipGetLastError()) return hip_fail("dla_norm_scale", e);
  }
  return DLA_OK;
}

// ------------------------------------------------------------------ peers, host side
constexpr int kPeerBlocks = 1024;  // workgroups of the norms: 4 per CU
constexpr int kMostPeers = 2048;   // their shares and pointers in LDS: 20 bytes each

int64_t peer_table_words(int64_t n_tensors, int64_t n_peers) {
  return n_tensors * static_cast<int64_t>(sizeof(Seg) / 8) + n_tensors * n_peers + n_peers;
}
int64_t peer_workspace_bytes(int64_t n_tensors, int64_t n_peers) {
  return (peer_table_words(n_tensors, n_peers) + n_peers /* sq */ + n_peers * kPeerBlocks) * 8;
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
  if (r.n_peers < 1 || r.n_peers > kMostPeers) return fail(DLA_E_INVALID, w + ": n_peers must be 1.." + std::to_string(kMostPeers));
  if (r.n_tensors < 0) return fail(DLA_E_INVALID, w + ": n_tensors < 0");
  if (r.n_tensors > 0 && (!r.dtypes || !r.peers || !r.centers || !r.numels)) return fail(DLA_E_INVALID, w + ": null array");
  for (int t = 0; t < r.n_tensors; ++t) {
    if (!known_dtype(r.dtypes[t])) return fail(DLA_E_INVALID, w + ": tensor " + std::to_string(t) + " has unknown dtype " + std::to_string(r.dtypes[t]));
    if (r.numels[t] < 0 || r.numels[t] > kMostElems) return fail(DLA_E_INVALID, w + ": tensor " + std::to_string(t) + " has a bad element count");
    if (r.numels[t] == 0) continue;
    const int es = elem_bytes(r.dtypes[t]);
    if (!r.centers[t] || !aligned_to(r.centers[t], es)) return fail(DLA_E_INVALID, w + ": centre tensor " + std::to_string(t) + " is null or not aligned");
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
    if (!r.outs[t] || !aligned_to(r.outs[t], es)) return fail(DLA_E_INVALID, w + ": out " + std::to_string(t) + " is null or not aligned");
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

// Writes the round's table into `dst` (device); *units: the units of all tensors.
int put_table(const char* what, const Round& r, const std::vector<int>& order, uint64_t* dst, int64_t* units, hipStream_t s) {
  const int m = static_cast<int>(order.size());
  std::vector<uint64_t> words(static_cast<size_t>(peer_table_words(m, r.n_peers)));
  Seg* segs = reinterpret_cast<Seg*>(words.data());
  uint64_t* ptrs = words.data() + m * (sizeof(Seg) / 8);
  int64_t u = 0;
  for (int q = 0; q < m; ++q) {
    const int t = order[q];
    segs[q] = {u, r.numels[t], r.centers[t], r.outs ? r.outs[t] : nullptr, r.dtypes[t]};
    for (int k = 0; k < r.n_peers; ++k)
      ptrs[static_cast<int64_t>(q) * r.n_peers + k] = reinterpret_cast<uint64_t>(r.peers[static_cast<int64_t>(t) * r.n_peers + k]);
    const int64_t per = kPeerUnit / elem_bytes(r.dtypes[t]);
    u += (r.numels[t] + per - 1) / per;
  }
  if (r.weights) std::memcpy(ptrs + static_cast<int64_t>(m) * r.n_peers, r.weights, sizeof(double) * r.n_peers);
  for (size_t i = 0; i < words.size(); i += kPutWords) {
    PutWords blob;
    const int n = static_cast<int>(std::min<size_t>(kPutWords, words.size() - i));
    std::memcpy(blob.w, words.data() + i, sizeof(uint64_t) * n);
    hipLaunchKernelGGL(put_kernel, dim3(1), dim3(512), 0, s, blob, dst + i, n);
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  *units = u;
  return DLA_OK;
}

template <int G>
void launch_peer_norms(bool tiled, dim3 grid, hipStream_t s, const Seg* segs, int m, int64_t units, const uint64_t* ptrs,
                       int n, const Layout& l, double* partials) {
  if (tiled) hipLaunchKernelGGL((peer_norms_kernel<G, true>), grid, dim3(kThreads), 0, s, segs, m, units, ptrs, n, l, partials);
  else hipLaunchKernelGGL((peer_norms_kernel<G, false>), grid, dim3(kThreads), 0, s, segs, m, units, ptrs, n, l, partials);
}

// The norms (sq != null, or outs == null), then the average (outs != null), of one round.
int round_impl(const char* what, const Round& r, double max_norm, const double* sq_in, double* sq_out, int out_dtype,
               void* norms, void* workspace, int64_t workspace_bytes, void* stream) {
  std::vector<int> order;
  if (int rc = check_round(what, r, &order)) return rc;
  const std::string w(what);
  if (norms && ((out_dtype != DLA_F32 && out_dtype != DLA_F64) || !aligned_to(norms, elem_bytes(out_dtype))))
    return fail(DLA_E_INVALID, w + ": norms must be aligned F32 or F64 values");
  if (r.outs && !r.weights) return fail(DLA_E_INVALID, w + ": null weights");
  if (r.outs && !(max_norm >= 0)) return fail(DLA_E_INVALID, w + ": max_norm must be >= 0");
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < peer_workspace_bytes(r.n_tensors, r.n_peers))
    return fail(DLA_E_INVALID, w + ": workspace is null, not aligned or smaller than dla_peer_workspace");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int m = static_cast<int>(order.size()), n = r.n_peers;
  uint64_t* table = static_cast<uint64_t*>(workspace);
  int64_t units = 0;
  if (m > 0)
    if (int rc = put_table(what, r, order, table, &units, s)) return rc;
  const Seg* segs = reinterpret_cast<const Seg*>(table);
  const uint64_t* ptrs = table + m * (sizeof(Seg) / 8);
  const double* weights = reinterpret_cast<const double*>(ptrs + static_cast<int64_t>(m) * n);
  double* sq = sq_out ? sq_out : reinterpret_cast<double*>(table + peer_table_words(r.n_tensors, n));
  double* partials = reinterpret_cast<double*>(table + peer_table_words(r.n_tensors, n) + n);
  if (!sq_in) {
    int64_t blocks = 0;
    if (m > 0) {
      // peers beside one read of the centre: 8 at most (their loads are all in flight), groups of equal size
      const int groups = (n + 7) / 8, g = (n + groups - 1) / groups;
      blocks = std::min<int64_t>(units, std::max<int64_t>(1, kPeerBlocks / groups));
      const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((n + g - 1) / g));
      switch (g) {
        case 1: launch_peer_norms<1>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 2: launch_peer_norms<2>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 3: launch_peer_norms<3>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 4: launch_peer_norms<4>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 5: launch_peer_norms<5>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 6: launch_peer_norms<6>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        case 7: launch_peer_norms<7>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
        default: launch_peer_norms<8>(r.tiled, grid, s, segs, m, units, ptrs, n, r.layout, partials); break;
      }
      if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
    }
    hipLaunchKernelGGL(peer_join_kernel, dim3(static_cast<unsigned>(n)), dim3(kThreads), 0, s, partials,
                       static_cast<int>(blocks), sq, out_dtype, norms);
    if (hipError_t e = hipGetLastError()) return hip_fail(what, e);
  }
  if (!r.outs) return DLA_OK;
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(units, 2 * kPeerBlocks));
  const size_t lds = static_cast<size_t>(n) * 20;
  const double* from = sq_in ? sq_in : sq;
  void* put = sq_in ? norms : nullptr;
  if (r.tiled) hipLaunchKernelGGL((bounded_kernel<true>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), lds, s, segs, m, units, ptrs, weights, n, r.layout, max_norm, from, out_dtype, put);
  else hipLaunchKernelGGL((bounded_kernel<false>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), lds, s, segs, m, units, ptrs, weights, n, r.layout, max_norm, from, out_dtype, put);
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
  if (!base || !aligned_to(base, 16) || tile_elems * es < 16 || tile_elems > (int64_t{1} << 40) || (tile_elems & (tile_elems - 1)))
    return fail(DLA_E_INVALID, w + ": base must be 16-byte aligned and tile_elems a power of two of >= 16 bytes");
  if (n_peers < 1 || n_peers > kMostPeers || slab_rows < n_peers) return fail(DLA_E_INVALID, w + ": need 1 <= n_peers <= slab_rows and n_peers <= " + std::to_string(kMostPeers));
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
  return 8 * (static_cast<int64_t>(kMaxPartials) + n_tensors / kNormTensors + 1);
}

int dla_norm(int n_tensors, const int* dtypes, const void* const* tensors, const int64_t* numels, int norm, int out_dtype,
             void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_norm", [&] {
    return norm_impl(n_tensors, dtypes, tensors, numels, norm, out_dtype, out, workspace, workspace_bytes, stream);
  });
}

int dla_norm_scale(int n_tensors, const int* dtypes, const void* const* tensors, void* const* outs, const int64_t* numels,
                   int norm, double max_norm, double eps, int out_dtype, void* norm_out, const void* workspace,
                   int64_t workspace_bytes, void* stream) {
  return guarded("dla_norm_scale", [&] {
    return norm_scale_impl(n_tensors, dtypes, tensors, outs, numels, norm, max_norm, eps, out_dtype, norm_out, workspace,
                           workspace_bytes, stream);
  });
}

int64_t dla_peer_workspace(int n_tensors, int n_peers) {
  if (n_tensors < 0 || n_peers < 1 || n_peers > kMostPeers) return 0;
  return peer_workspace_bytes(n_tensors, n_peers);
}

int dla_peer_norms(int n_tensors, const int* dtypes, const void* const* peer_ptrs, const void* const* centers,
                   const int64_t* numels, int n_peers, double* sq_out, int out_dtype, void* norms, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  return guarded("dla_peer_norms", [&] {
    const Round r = {n_tensors, dtypes, peer_ptrs, centers, nullptr, numels, nullptr, n_peers, {0, 0, 0}, false};
    return round_impl("dla_peer_norms", r, 0, nullptr, sq_out, out_dtype, norms, workspace, workspace_bytes, stream);
  });
}

int dla_wsum_bounded(int n_tensors, const int* dtypes, const void* const* peer_ptrs, const void* const* centers,
                     void* const* outs, const int64_t* numels, const double* weights, int n_peers, double max_norm,
                     const double* sq, int out_dtype, void* norms, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_wsum_bounded", [&] {
    if (!outs && n_tensors > 0) return fail(DLA_E_INVALID, "dla_wsum_bounded: null outs array");
    static void* const none[1] = {nullptr};
    const Round r = {n_tensors, dtypes, peer_ptrs, centers, outs ? outs : none, numels, weights, n_peers, {0, 0, 0}, false};
    return round_impl("dla_wsum_bounded", r, max_norm, sq, nullptr, out_dtype, norms, workspace, workspace_bytes, stream);
  });
}

int dla_wsum_bounded_slab_tiled(int dtype, const void* base, int64_t tile_elems, int64_t slab_rows, const void* center,
                                const double* weights, int n_peers, int64_t n_elems, double max_norm, void* out,
                                int out_dtype, void* norms, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded("dla_wsum_bounded_slab_tiled", [&] {
    if (!out && n_elems > 0) return fail(DLA_E_INVALID, "dla_wsum_bounded_slab_tiled: null out");
    SlabRound sr;
    if (int rc = slab_round("dla_wsum_bounded_slab_tiled", &sr, dtype, base, tile_elems, slab_rows, center, n_peers, n_elems, out, weights)) return rc;
    return round_impl("dla_wsum_bounded_slab_tiled", sr.r, max_norm, nullptr, nullptr, out_dtype, norms, workspace, workspace_bytes, stream);
  });
}

}  // extern "C"
