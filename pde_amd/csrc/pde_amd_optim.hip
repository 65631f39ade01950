// C ABI (include/pde_amd.h) of the weight update that follows a loss's backward pass: the norm of the gradients of many
// tensors, their scaling by it, and the AdamW step that applies the scaling while it reads the gradients.
//
// Every kernel walks a LIST of tensors.  A tensor is cut into units, the units of all tensors of a launch are numbered
// through, and workgroups take units by number, so the work of a workgroup does not depend on how the elements are
// spread over tensors.  The list travels in the kernel's arguments (at most 4 KiB): nothing is copied to the device
// first, and a captured graph holds its own list.  All of it is bound by memory, or by launches where it is small.
#include "../../include/pde_amd.h"
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace pde_amd {
namespace {

constexpr int NT = 256;                  // threads of every workgroup
constexpr int UNIT_BYTES = 16384;        // bytes of a unit of the norm and scaling kernels: 4 16-byte loads per thread
constexpr int NORM_BLOCKS = 1024;        // workgroups of a launch: 4 per CU on 256 CUs
constexpr int SCALE_BLOCKS = 1024;
constexpr int SCALE_RUN = 32;            // neighbouring units that go to workgroups of one XCD
constexpr int LIST = 255;                // tensors of a launch
constexpr int STEP_UNIT = NT * 4;        // the update kernel: elements of a unit, a workgroup for each
constexpr int STEP_RUN = 64;             // the same for the update
constexpr int STEP_LIST = 319;
constexpr int PREP_LIST = 255;           // tensors of a launch of the norm kernel ahead of it

// Reads with the nontemporal hint leave the 256 MB memory-side cache alone and are faster where the data is not in it, as
// after a forward and backward pass; without the hint a second reader finds it there.  In us with / without the hint, data
// out of the cache ahead of each call:
//   norm    16 MB 8.0 / 8.4   64 MB 14.8 / 16.4   256 MB 44.4 / 48.6   1 GB 158 / 179
//   clip    16 MB 14.0 / 14.8   32 MB 25.5 / 24.4   64 MB 41.3 / 43.3   256 MB 139 / 154   1 GB 548 / 636
//   update  16 MB 10.3 / 13.1   64 MB 25.1 / 29.4   256 MB 81.6 / 92.7   1 GB 313 / 347   (bytes of all its tensors)
// (data in the cache: norm 64 MB 12.5 / 14.1, 192 MB 32.1 / 31.9; update 64 MB 22.4 / 22.4, 192 MB 61.6 / 56.1).
// So the update always has it, norm and scaling from STREAM_BYTES on, and the norm ahead of an update leaves the last
// KEEP_BYTES of the gradients in the cache (151 M bf16: 715 us for the step, 747 with none left).
constexpr int64_t STREAM_BYTES = 64ll << 20;
constexpr int64_t KEEP_BYTES = 224ll << 20;

// 16 bytes (and 8) of elements at any element-aligned address: gfx950 loads and stores them in one instruction
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h8 __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned short h4 __attribute__((ext_vector_type(4), aligned(2)));

// addresses come as numbers out of a list: said to be global memory, they are read with global rather than flat loads
template <class T> using gptr = __attribute__((address_space(1))) T*;

// conversions of the hardware: to nearest, ties to even; NaN stays NaN
__device__ __forceinline__ float bf16_to_float(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ float f16_to_float(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ unsigned short float_to_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ __forceinline__ unsigned short float_to_f16(float x) {
  // A multiplication ahead of this and the conversion would become one v_fma_mixlo_f16, which rounds the exact product: not
  // the fp32 product's rounding where that lies on the middle of two fp16 values and the exact one beside it.
  asm("" : "+v"(x));
  return __builtin_bit_cast(unsigned short, (_Float16)x);
}

template <int DT> struct Elem;
template <> struct Elem<PDE_AMD_F32> {
  typedef float T;
  typedef f4 V;
  static constexpr int W = 4;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
};
template <> struct Elem<PDE_AMD_BF16> {
  typedef unsigned short T;
  typedef h8 V;
  static constexpr int W = 8;
  static __device__ __forceinline__ float get(T x) { return bf16_to_float(x); }
  static __device__ __forceinline__ T put(float x) { return float_to_bf16(x); }
};
template <> struct Elem<PDE_AMD_F16> {
  typedef unsigned short T;
  typedef h8 V;
  static constexpr int W = 8;
  static __device__ __forceinline__ float get(T x) { return f16_to_float(x); }
  static __device__ __forceinline__ T put(float x) { return float_to_f16(x); }
};


// A tensor in a list: its address with the dtype in the top byte, the number of its first unit, and the elements of its
// last one; all its other units are whole.
constexpr uint32_t NONE = 0xffffffffu;

template <int CAPACITY> struct Tensors {
  uint64_t ptr[CAPACITY];
  uint32_t first[CAPACITY + 1];          // first[n] = units of the launch; NONE behind
  uint16_t last[CAPACITY];
  int32_t n;
  uint32_t units;
  uint32_t per_block;                    // units of a workgroup, where it takes neighbouring ones
  uint32_t stream_until;                 // units below are read with the nontemporal hint
};
constexpr uint64_t ADDRESS_MASK = 0xffffffffffffffull;      // device addresses have 48 bits
typedef Tensors<LIST> TensorList;
static_assert(sizeof(TensorList) <= 4000, "the list has to fit the kernel's arguments");
static_assert(UNIT_BYTES / 2 <= 65535, "");

__host__ __device__ constexpr int unit_shift(int dtype) { return dtype == PDE_AMD_F32 ? 12 : 13; }      // log2 of a unit's elements
__host__ __device__ constexpr int64_t unit_elements(int dtype) { return 1ll << unit_shift(dtype); }
static_assert(unit_elements(PDE_AMD_F32) * 4 == UNIT_BYTES && unit_elements(PDE_AMD_BF16) * 2 == UNIT_BYTES, "");

// Which tensor holds a unit: the last one whose first unit is not beyond it (tensors without elements share a first unit
// with their successor and are never the last such one).  Each wave holds the first units across its lanes and counts:
// one round trip to the kernel's arguments, where a search of them takes one for every halving.  Units below the launch's
// number only: first[n] and what lies behind it are never counted.
template <int CAPACITY> struct Finder {
  static_assert((CAPACITY + 1) % 64 == 0, "the lanes read whole rows");
  static constexpr int WORDS = (CAPACITY + 1) / 64;
  uint32_t first[WORDS];

  __device__ __forceinline__ explicit Finder(const uint32_t* units) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) first[w] = units[w * 64 + (int)(threadIdx.x & 63)];
  }
  __device__ __forceinline__ int operator()(uint32_t u) const {
    int count = 0;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) count += __popcll(__ballot(first[w] <= u));
    return count - 1;
  }
};

template <bool STREAM, class V, class T> __device__ __forceinline__ V load(gptr<T> p) {
  return STREAM ? __builtin_nontemporal_load((gptr<const V>)p) : *(gptr<const V>)p;
}
template <class V, class T> __device__ __forceinline__ void stream_out(gptr<T> p, V v) { __builtin_nontemporal_store(v, (gptr<V>)p); }

// ------------------------------------------------------------------------------------------------
// norms: (sum |x|^p)^(1/p) over all elements of the list, in two launches: partial values by workgroups, and their sum.
// Sums run in fp64: the square of any fp32 value is exact there and neither overflows nor vanishes, and the result does not
// depend on how the units are dealt out beyond the last bits of a double (conversion and fp64 fma together take less than
// half of the vector units' time at the memory's rate).
// Bound by HBM: 680 M fp32 (2.72 GB) in 397 us = 6.85 TB/s (a 2 GiB copy runs at 4.9 TB/s); 151 M bf16 with the norms of
// 192 tensors in 46.8 + 4.6 us.  What it takes: runs of neighbouring units per workgroup with the next unit's loads under
// way during the sums (461 us without), 1024 workgroups of 256 (512, 1024, 2048, 4096: 479, 397, 416, 418 us, the bf16 case
// 77, 55, 54, 62), nontemporal loads.  Small lists are two launches and their latency: 147 k values in 48 tensors
// 4.0 + 1.8 us.
// ------------------------------------------------------------------------------------------------
enum { NORM_INF = 0, NORM_ONE = 1, NORM_TWO = 2 };

// the larger of two magnitudes, NaN if either is
__device__ __forceinline__ double join_max(double a, double b) { return (a > b || a != a) ? a : b; }

template <int P> __device__ __forceinline__ double join(double a, double b) { return P == NORM_INF ? join_max(a, b) : a + b; }

template <int P> struct Acc {
  double s0 = 0.0, s1 = 0.0;
  unsigned m = 0;                        // P = inf: bits of the largest magnitude; a NaN's bits are larger than infinity's
  __device__ __forceinline__ void add(float x, int k) {
    if (P == NORM_INF) {
      const unsigned b = __float_as_uint(x) & 0x7fffffffu;
      m = b > m ? b : m;
    } else {
      const double d = (double)x;
      double& s = k & 1 ? s1 : s0;
      s = P == NORM_TWO ? fma(d, d, s) : s + fabs(d);
    }
  }
  __device__ __forceinline__ double value() const { return P == NORM_INF ? (double)__uint_as_float(m) : s0 + s1; }
};

// value of all threads of the workgroup, in thread 0
template <int P> __device__ __forceinline__ double block_join(double v, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_down(v, o, 64));
  __syncthreads();                       // the previous use of lds
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = join<P>(v, lds[w]);
  return v;
}

template <int P> __device__ __forceinline__ float norm_of(double s) { return (float)(P == NORM_TWO ? sqrt(s) : s); }

// The norm made of `count` partial values, in every thread of the workgroup; every kernel adds them up in this order, so
// that all find the same bits.  In two halves, so that other loads can be issued between: loads return in order, and
// those of the partial values are the ones waited for first.
template <int P> struct PartialValues {
  double mine[4];
  const double* partial;
  int count;
  __device__ __forceinline__ PartialValues(const double* __restrict__ p, int n) : partial(p), count(n) {
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[k] = k * NT + (int)threadIdx.x < n ? p[k * NT + (int)threadIdx.x] : 0.0;
  }
  __device__ __forceinline__ float norm(double* lds) const {
    double v = join<P>(join<P>(mine[0], mine[1]), join<P>(mine[2], mine[3]));
    for (int i = 4 * NT + (int)threadIdx.x; i < count; i += NT) v = join<P>(v, partial[i]);
    v = block_join<P>(v, lds);
    __syncthreads();
    if (threadIdx.x == 0) lds[0] = v;
    __syncthreads();
    return norm_of<P>(lds[0]);
  }
};

// One unit of a tensor of a list: address, first element, number of elements
struct Unit {
  uint64_t ptr;
  int64_t at;
  int count, dtype;
  bool stream;
  template <class L> __device__ __forceinline__ Unit(const L& list, int t, uint32_t u) {
    const uint64_t p = list.ptr[t];
    ptr = p & ADDRESS_MASK;
    dtype = (int)(p >> 56);
    at = (int64_t)(u - list.first[t]) * unit_elements(dtype);
    count = u + 1 == list.first[t + 1] ? (int)list.last[t] : (int)unit_elements(dtype);
    stream = u < list.stream_until;
  }
};

// A thread's share of a unit: STEPS loads of 16 bytes.  In the last unit of a tensor the loads that would pass its end
// are left out (zeros), and its last elements, fewer than a load holds, are taken one by one.
template <int DT> struct Share {
  typedef Elem<DT> E;
  typedef typename E::V V;
  typedef typename E::T T;
  static constexpr int STEPS = UNIT_BYTES / (NT * 16);
  V v[STEPS];
  gptr<T> x;
  int count;

  __device__ __forceinline__ explicit Share(const Unit& unit) : x((gptr<T>)unit.ptr + unit.at), count(unit.count) {
    if (whole() && unit.stream) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) v[s] = __builtin_nontemporal_load((gptr<const V>)(x + place(s)));
    } else if (whole()) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) v[s] = *(gptr<const V>)(x + place(s));
    } else {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        v[s] = V(0);
        if (place(s) + E::W <= count) v[s] = *(gptr<const V>)(x + place(s));
      }
    }
  }
  __device__ __forceinline__ static int place(int s) { return (s * NT + (int)threadIdx.x) * E::W; }
  __device__ __forceinline__ bool whole() const { return count == (int)unit_elements(DT); }
  __device__ __forceinline__ int single() const { return (count & ~(E::W - 1)) + (int)threadIdx.x; }      // < count: this thread has one

  template <int P> __device__ __forceinline__ void add(Acc<P>& acc) const {
    if (single() < count) acc.add(E::get(x[single()]), 0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int k = 0; k < E::W; ++k) acc.add(E::get(v[s][k]), k);
  }
  __device__ __forceinline__ void scale(float c) {
    if (single() < count) x[single()] = E::put(E::get(x[single()]) * c);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int k = 0; k < E::W; ++k) v[s][k] = E::put(E::get(v[s][k]) * c);
      if (place(s) + E::W <= count) *(gptr<V>)(x + place(s)) = v[s];
    }
  }
};

template <int P> __device__ __forceinline__ void add_unit(const Unit& x, Acc<P>& acc) {
  switch (x.dtype) {
    case PDE_AMD_F32: Share<PDE_AMD_F32>(x).add(acc); break;
    case PDE_AMD_BF16: Share<PDE_AMD_BF16>(x).add(acc); break;
    default: Share<PDE_AMD_F16>(x).add(acc); break;
  }
}

// `units` whole units in a row, each one's loads under way while the one before is added up
template <int DT, int P, bool STREAM> __device__ __forceinline__ void add_run(const Unit& from, uint32_t units, Acc<P>& acc) {
  typedef Elem<DT> E;
  typedef typename E::V V;
  constexpr int STEPS = Share<DT>::STEPS;
  gptr<const typename E::T> x = (gptr<const typename E::T>)from.ptr + from.at + (int)threadIdx.x * E::W;
  V v[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) v[s] = load<STREAM, V>(x + s * NT * E::W);
  for (uint32_t i = 1; i < units; ++i) {
    x += unit_elements(DT);
    V next[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) next[s] = load<STREAM, V>(x + s * NT * E::W);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int k = 0; k < E::W; ++k) acc.add(E::get(v[s][k]), k);
      v[s] = next[s];
    }
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int k = 0; k < E::W; ++k) acc.add(E::get(v[s][k]), k);
}

template <int P, bool STREAM> __device__ __forceinline__ void add_run_of(const Unit& from, uint32_t units, Acc<P>& acc) {
  switch (from.dtype) {
    case PDE_AMD_F32: add_run<PDE_AMD_F32, P, STREAM>(from, units, acc); break;
    case PDE_AMD_BF16: add_run<PDE_AMD_BF16, P, STREAM>(from, units, acc); break;
    default: add_run<PDE_AMD_F16, P, STREAM>(from, units, acc); break;
  }
}

// EACH = false: one partial value per workgroup, partial[block].
// EACH = true: one per workgroup and tensor it touches, partial[block + tensor]: from one value to the next a workgroup
// moves to a later tensor or the launch to the next workgroup, so no two share a place.  A place that is passed over
// (tensors without elements; a tensor that ends with a workgroup's run) is set to 0 by the one before it, so that all of
// them together, blocks + n - 1, add up to the total.
template <int P, bool EACH, int CAPACITY, class L>
__device__ __forceinline__ void norm_partial(const L& list, double* __restrict__ partial) {
  __shared__ double lds[NT / 64];
  const uint32_t units = list.units;
  const uint32_t u0 = blockIdx.x * list.per_block, u1 = min(u0 + list.per_block, units);
  const Finder<CAPACITY> find(list.first);
  Acc<P> acc;
  int t = 0;
  for (uint32_t u = u0; u < u1;) {
    const int next = find(u);
    if (EACH && u > u0) {
      const double v = block_join<P>(acc.value(), lds);
      if (threadIdx.x == 0)
        for (int i = t; i < next; ++i) partial[blockIdx.x + i] = i == t ? v : 0.0;
      acc = Acc<P>();
    } else if (EACH && u == 0 && threadIdx.x == 0) {
      for (int i = 0; i < next; ++i) partial[i] = 0.0;
    }
    t = next;
    const Unit x(list, t, u);
    uint32_t end = list.first[t + 1];
    const bool ragged = end <= u1 && (int)list.last[t] != (int)unit_elements(x.dtype);      // the tensor's last unit is here, and is not whole
    end = min(end, u1);
    const uint32_t run = end - u - (ragged ? 1 : 0);
    if (run == 0) {
      add_unit(x, acc);
    } else {
      if (x.stream) add_run_of<P, true>(x, run, acc);
      else add_run_of<P, false>(x, run, acc);
      if (ragged) add_unit(Unit(list, t, end - 1), acc);
    }
    u = end;
  }
  const double v = block_join<P>(acc.value(), lds);
  const int last = !EACH ? 0 : u1 < units ? find(u1) : list.n - 1;
  if (threadIdx.x == 0) {
    partial[blockIdx.x + (EACH ? t : 0)] = v;
    if (EACH)
      for (int i = t + 1; i <= last; ++i) partial[blockIdx.x + i] = 0.0;
  }
}

template <int P, bool EACH>
__global__ __launch_bounds__(NT) void norm_partial_kernel(const TensorList list, double* __restrict__ partial) {
  norm_partial<P, EACH, LIST>(list, partial);
}

// one workgroup: the norm
template <int P>
__global__ __launch_bounds__(NT) void norm_total_kernel(const double* __restrict__ partial, int count, float* __restrict__ total) {
  __shared__ double lds[NT / 64];
  const float norm = PartialValues<P>(partial, count).norm(lds);
  if (threadIdx.x == 0) *total = norm;
}

struct FirstUnits {
  uint32_t first[LIST + 1];
  int32_t n;
  uint32_t per_block;
};

// a wave per tensor: its partial values and its norm; the last workgroup: the norm of everything, from the partial values
// of this launch and those that lie ahead of them (`all` in number)
template <int P>
__global__ __launch_bounds__(NT) void norm_each_kernel(const FirstUnits list, const double* __restrict__ partial, float* __restrict__ each,
                                                          const double* __restrict__ start, int all, float* __restrict__ total) {
  __shared__ double lds[NT / 64];
  if (blockIdx.x == gridDim.x - 1) {
    if (!total) return;
    const float norm = PartialValues<P>(start, all).norm(lds);
    if (threadIdx.x == 0) *total = norm;
    return;
  }
  const int t = blockIdx.x * (NT / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= list.n) return;
  double v = 0.0;
  if (list.first[t] < list.first[t + 1]) {
    const int b0 = (int)(list.first[t] / list.per_block), b1 = (int)((list.first[t + 1] - 1) / list.per_block);
    for (int b = b0 + lane; b <= b1; b += 64) v = join<P>(v, partial[b + t]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_down(v, o, 64));
  if (lane == 0) each[t] = norm_of<P>(v);
}

// ------------------------------------------------------------------------------------------------
// scaling by min(1, max_norm / (norm + 1e-6)), in 32 bits with one rounding to the tensor's type.  The +1e-6 (a norm of
// zero) is torch.nn.utils.clip_grad_norm_'s.  A factor of exactly one leaves every value as it is, so nothing is read or
// written then; a NaN norm makes the factor NaN.
// Bound by HBM: 151 M fp32, norm and scaling together 314 us = 5.8 TB/s of what they move (read twice, written once;
// 318 us without neighbouring units on one XCD).  The norm cannot be had without reading everything before anything is written, so a list beyond the caches is
// read twice; a form that kept it in registers and LDS would need all workgroups resident at once and waiting for each
// other, which two calls on two streams could not promise.
// Up to SCALE_BLOCKS units a workgroup takes one and reads it while the norm is added up (6.5 M bf16 7.6 us; 13.4
// with the read behind the norm and the rounding in software); beyond, SCALE_BLOCKS workgroups go through the units, so that a step that needs no clipping
// ends after the norm (a workgroup per unit scales 151 M fp32 in the same time, within 1 %, and starts 37 k workgroups for
// nothing otherwise; 256, 512, 2048 workgroups: 408, 320, 325 us where 1024 take 311).
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float clip_factor(float max_norm, float total) {
  const float c = max_norm / (total + 1e-6f);
  return c > 1.0f ? 1.0f : c;
}

// The norm comes as partial values, which every workgroup adds up for itself (a launch less), or, count < 0, as *given.
template <int P> struct Factor {
  const PartialValues<P> values;
  const float* given;
  float* total;
  float max_norm;
  __device__ __forceinline__ Factor(const double* partial, int count, const float* given_, float max_norm_, float* total_)
      : values(partial, count), given(given_), total(total_), max_norm(max_norm_) {}
  __device__ __forceinline__ float get(double* lds) const {
    const float norm = values.count < 0 ? *given : values.norm(lds);
    if (total && blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
    return clip_factor(max_norm, norm);
  }
};

template <int DT, int P> __device__ __forceinline__ void scale_only_unit(const Unit& x, const Factor<P>& factor, double* lds) {
  Share<DT> share(x);                    // under way while the norm is added up
  const float c = factor.get(lds);
  if (c != 1.0f) share.scale(c);
}

// Workgroups go to the 8 XCDs in turn: of 8 * RUN units each XCD takes RUN neighbours.  What is left over at the end of the
// grid is taken in order.
template <int RUN> __device__ __forceinline__ uint32_t unit_of_block() {
  constexpr uint32_t GROUP = 8 * RUN;
  const uint32_t from = blockIdx.x / GROUP * GROUP, in = blockIdx.x % GROUP;
  return from + GROUP <= gridDim.x ? from + in % 8 * RUN + in / 8 : blockIdx.x;
}

template <int P>
__global__ __launch_bounds__(NT) void scale_kernel(const TensorList list, const double* __restrict__ partial, int count,
                                                   const float* __restrict__ given, float max_norm, float* __restrict__ total) {
  __shared__ double lds[NT / 64];
  const Factor<P> factor(partial, count, given, max_norm, total);
  const Finder<LIST> find(list.first);
  const uint32_t units = list.units;
  if (units <= gridDim.x) {
    // a workgroup per unit: reading it at once costs nothing beside the wait for the norm, even where the factor is 1
    const Unit x(list, find(blockIdx.x), blockIdx.x);
    switch (x.dtype) {
      case PDE_AMD_F32: scale_only_unit<PDE_AMD_F32>(x, factor, lds); break;
      case PDE_AMD_BF16: scale_only_unit<PDE_AMD_BF16>(x, factor, lds); break;
      default: scale_only_unit<PDE_AMD_F16>(x, factor, lds); break;
    }
    return;
  }
  const float c = factor.get(lds);
  if (c == 1.0f) return;
  for (uint32_t u = unit_of_block<SCALE_RUN>(); u < units; u += gridDim.x) {
    const Unit x(list, find(u), u);
    switch (x.dtype) {
      case PDE_AMD_F32: Share<PDE_AMD_F32>(x).scale(c); break;
      case PDE_AMD_BF16: Share<PDE_AMD_BF16>(x).scale(c); break;
      default: Share<PDE_AMD_F16>(x).scale(c); break;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// AdamW.  With c the clipping factor, per element
//   g' = c g;  m <- b1 m + (1 - b1) g';  v <- b2 v + (1 - b2) g'^2
//   w <- (1 - lr wd) w - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in 32 bits; a 16-bit parameter is w rounded once, with w itself kept.  The step count t of every tensor lives on the
// device, so a captured step counts on, and a step that is skipped for a norm that is not finite does not.
//
// Two launches: the first makes the partial values of the norm and, in a workgroup of its own, what depends on t (the
// powers in fp64, one thread per tensor); the second updates, and writes the counts that the first only read.
// Bound by HBM: 453 M fp32 (28 bytes an element, 12.7 GB) with the norm's own read of 1.8 GB 2301 us = 6.3 TB/s; 151 M bf16
// (28 bytes: gradient 2, master and moments 12 + 12, parameter 2) with the norm 705 us = 6.4 TB/s; counters show the bytes of
// the formula and no others.  A workgroup reads its 1024 elements of all tensors, and only then writes.  On the former
// case: 2800 us with 2048 workgroups that go through the units, 2480 / 2410 / 2365 us with 4096 / 2048 / 1024 elements per
// workgroup and 16 neighbouring units on one XCD, 2330 / 2301 / 2400 us with 32 / 64 / 128.  The sum over the 1024 partial
// values in every workgroup costs nothing beside that (a kernel between instead: 2405 us at 32).  Each further launch of the
// norm, one for 255 tensors, brings up to 1024 values more, and these cost: 151 M fp32 in 192 / 300 / 600 / 1200 tensors 774 /
// 857 / 997 / 1156 us, 450 M 2423 / 2447 / 2767 / 3154.
// ------------------------------------------------------------------------------------------------
struct Prep {                            // what the update needs of a tensor's step
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, step_size, inv_sqrt_bias2;
  float step, pad[3];
};

// Both lists of a step hold neighbours of the caller's table, base + k in place k; a tensor without a gradient has no units.
struct PrepList : Tensors<PREP_LIST> {
  int32_t base;
  float lr[PDE_AMD_ADAMW_MAX_GROUPS];
};
static_assert(sizeof(PrepList) <= 4000, "");

__device__ __forceinline__ void prepare_steps(const PrepList& list, const pde_amd_adamw_tensor* __restrict__ table,
                                              const pde_amd_adamw_group* __restrict__ groups, Prep* __restrict__ prep) {
  for (int i = threadIdx.x; i < list.n; i += NT) {
    if (list.first[i] == list.first[i + 1]) continue;
    const pde_amd_adamw_tensor& t = table[list.base + i];
    const pde_amd_adamw_group& g = groups[t.group];
    const double lr = (double)(g.lr_device ? *g.lr_device : list.lr[t.group]);
    Prep p;
    p.step = *t.step + 1.0f;
    const double bias1 = 1.0 - pow(g.beta1, (double)p.step), bias2 = 1.0 - pow(g.beta2, (double)p.step);
    p.beta1 = (float)g.beta1;
    p.one_minus_beta1 = (float)(1.0 - g.beta1);
    p.beta2 = (float)g.beta2;
    p.one_minus_beta2 = (float)(1.0 - g.beta2);
    p.eps = (float)g.eps;
    p.decay = (float)(1.0 - lr * g.weight_decay);
    p.step_size = (float)(lr / bias1);
    p.inv_sqrt_bias2 = (float)(1.0 / sqrt(bias2));
    prep[list.base + i] = p;
  }
}

__global__ __launch_bounds__(NT) void adamw_norm_kernel(const PrepList list, const pde_amd_adamw_tensor* __restrict__ table,
                                                        const pde_amd_adamw_group* __restrict__ groups, Prep* __restrict__ prep,
                                                        double* __restrict__ partial, const float* __restrict__ given,
                                                        float* __restrict__ given_copy) {
  // the last workgroup prepares; without a norm it is the only one.  A given norm is copied: the caller's may lie in memory
  // that the update writes.
  if (blockIdx.x == gridDim.x - 1) {
    if (given && threadIdx.x == 0) *given_copy = *given;
    prepare_steps(list, table, groups, prep);
  } else {
    norm_partial<NORM_TWO, false, PREP_LIST>(list, partial);
  }
}

// The groups' settings into device memory, out of the kernel's arguments: where a schedule moves them at every step, none
// waits for a copy.  Bound by the launch, 1.7 us on the GPU: such a step over 48 tensors of 3000 takes 17.0 us, 12.3 with
// settings that stay (33.6 with a copy of the settings from the host).
struct GroupList {
  pde_amd_adamw_group group[PDE_AMD_ADAMW_MAX_GROUPS];
};
static_assert(sizeof(GroupList) <= 4000, "");

__global__ __launch_bounds__(64) void adamw_groups_kernel(const GroupList list, int32_t n, pde_amd_adamw_group* __restrict__ out) {
  if ((int)threadIdx.x < n) out[threadIdx.x] = list.group[threadIdx.x];
}
static_assert(PDE_AMD_ADAMW_MAX_GROUPS <= 64, "a thread for each");

struct StepList {
  uint64_t grad[STEP_LIST];
  uint32_t first[STEP_LIST + 1];
  int32_t base;
};
static_assert(sizeof(StepList) <= 3900, "");

struct ClipArgs {                        // where the update finds its clipping factor
  const double* partial;
  const float* given;                    // the norm, when it is not made of partial values
  float* total;                          // where the norm is written, or NULL
  int32_t count;
  int32_t skip_nonfinite;
  float max_norm;                        // < 0: no clipping
};

__device__ __forceinline__ void adamw_one(float g, float& w, float& m, float& v, float c, const Prep& p) {
  g *= c;
  m = p.beta1 * m + p.one_minus_beta1 * g;
  v = p.beta2 * v + p.one_minus_beta2 * (g * g);
  w = p.decay * w - p.step_size * (m / (sqrtf(v) * p.inv_sqrt_bias2 + p.eps));
}

// A thread's 4 neighbouring elements: read, updated, written
template <bool BF16, bool WHOLE> struct Quad {
  f4 g, w, m, v;
  h4 h;
  gptr<float> pw, pm, pv;
  gptr<const float> g32;
  gptr<const unsigned short> g16;
  gptr<unsigned short> out;
  int count, i;

  __device__ __forceinline__ Quad(const pde_amd_adamw_tensor& t, uint64_t grad, int64_t at, int count_) : count(count_), i((int)threadIdx.x * 4) {
    pw = (gptr<float>)(uint64_t)(BF16 ? (void*)t.master : t.param) + at;
    pm = (gptr<float>)(uint64_t)t.exp_avg + at;
    pv = (gptr<float>)(uint64_t)t.exp_avg_sq + at;
    g32 = (gptr<const float>)grad + at;                       // the gradient, one of these
    g16 = (gptr<const unsigned short>)grad + at;
    out = (gptr<unsigned short>)(uint64_t)t.param + at;       // BF16: the rounded weight
  }
  __device__ __forceinline__ bool mine() const { return WHOLE || i + 4 <= count; }

  __device__ __forceinline__ void read() {
    if (!mine()) return;
    if (BF16) h = load<true, h4>(g16 + i);
    else g = load<true, f4>(g32 + i);
    w = load<true, f4>(pw + i);
    m = load<true, f4>(pm + i);
    v = load<true, f4>(pv + i);
  }

  __device__ __forceinline__ void update(float c, const Prep& p) {
    if (!mine()) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float wk = w[k], mk = m[k], vk = v[k];
      adamw_one(BF16 ? bf16_to_float(h[k]) : g[k], wk, mk, vk, c, p);
      w[k] = wk; m[k] = mk; v[k] = vk;
      if (BF16) h[k] = float_to_bf16(wk);
    }
    stream_out(pw + i, w);
    stream_out(pm + i, m);
    stream_out(pv + i, v);
    if (BF16) stream_out(out + i, h);
  }

  // the last elements of a tensor whose size is no multiple of 4
  __device__ __forceinline__ void update_tail(float c, const Prep& p) {
    const int j = (count & ~3) + (int)threadIdx.x;
    if (j >= count) return;
    float wk = pw[j], mk = pm[j], vk = pv[j];
    adamw_one(BF16 ? bf16_to_float(g16[j]) : g32[j], wk, mk, vk, c, p);
    pw[j] = wk; pm[j] = mk; pv[j] = vk;
    if (BF16) out[j] = float_to_bf16(wk);
  }
};

template <bool BF16, bool WHOLE>
__device__ __forceinline__ void adamw_unit(const pde_amd_adamw_tensor& t, uint64_t grad, int64_t at, int count, bool owner, const Prep& p,
                                           const ClipArgs& a, double* lds) {
  const bool need = a.max_norm >= 0.0f || a.skip_nonfinite;
  const PartialValues<NORM_TWO> values(a.partial, a.count);
  Quad<BF16, WHOLE> x(t, grad, at, count);
  x.read();                              // under way while the norm is added up
  float c = 1.0f;
  if (need) {
    const float norm = a.given ? *a.given : values.norm(lds);
    if (a.total && blockIdx.x == 0 && threadIdx.x == 0) *a.total = norm;
    if (a.max_norm >= 0.0f) c = clip_factor(a.max_norm, norm);
    if (a.skip_nonfinite && !(fabsf(norm) < INFINITY)) return;
  }
  if (owner && threadIdx.x == 0) *t.step = p.step;
  x.update(c, p);
  if (!WHOLE) x.update_tail(c, p);
}

__global__ __launch_bounds__(NT) void adamw_update_kernel(const StepList list, const ClipArgs clip, const pde_amd_adamw_tensor* __restrict__ table,
                                                               const Prep* __restrict__ prep) {
  __shared__ double lds[NT / 64];
  const uint32_t u = unit_of_block<STEP_RUN>();
  const int k = Finder<STEP_LIST>(list.first)(u);
  const pde_amd_adamw_tensor& t = table[list.base + k];
  const uint32_t unit = u - list.first[k];
  const int64_t at = (int64_t)unit * STEP_UNIT, left = t.numel - at;
  const int count = (int)(left < STEP_UNIT ? left : STEP_UNIT);
  const uint64_t grad = list.grad[k];
  const Prep p = prep[list.base + k];
  if (t.dtype == PDE_AMD_BF16) {
    if (count == STEP_UNIT) adamw_unit<true, true>(t, grad, at, count, unit == 0, p, clip, lds);
    else adamw_unit<true, false>(t, grad, at, count, unit == 0, p, clip, lds);
  } else {
    if (count == STEP_UNIT) adamw_unit<false, true>(t, grad, at, count, unit == 0, p, clip, lds);
    else adamw_unit<false, false>(t, grad, at, count, unit == 0, p, clip, lds);
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
int launch_status() { return hipGetLastError() == hipSuccess ? PDE_AMD_OK : PDE_AMD_EHIP; }

int64_t pieces(int64_t n, int64_t of) { return n / of + (n % of != 0); }
int64_t units_of(int64_t n, int32_t dtype) { return (n >> unit_shift(dtype)) + ((n & (unit_elements(dtype) - 1)) != 0); }
int64_t bytes_of(int64_t n, int32_t dtype) { return n * (dtype == PDE_AMD_F32 ? 4 : 2); }

constexpr int64_t MAX_UNITS = (1ll << 31) - 1;                // of a call: unit numbers stay in 32 bits,
constexpr int64_t MAX_STEP_UNITS = (1ll << 32) / NT - 1;      // and of an update's launch: the threads of its grid too

int check_tensors(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int64_t& bytes) {
  if (n < 0 || (n > 0 && (!tensors || !numel || !dtypes))) return PDE_AMD_EINVAL;
  int64_t units = 0;
  bytes = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || (numel[i] > 0 && !tensors[i]) || dtypes[i] < PDE_AMD_F32 || dtypes[i] > PDE_AMD_F16) return PDE_AMD_EINVAL;
    const int64_t u = units_of(numel[i], dtypes[i]);
    if (u > MAX_UNITS - units) return PDE_AMD_ESHAPE;
    units += u;
    bytes += bytes_of(numel[i], dtypes[i]);
  }
  return PDE_AMD_OK;
}

// Appends a tensor to a list under construction; `streamed` counts down the bytes that are read past the cache.
template <class L> void append(L& list, int32_t& k, uint32_t& units, const void* ptr, int64_t numel, int32_t dtype, int64_t& streamed) {
  const int64_t whole = unit_elements(dtype), over = numel & (whole - 1);
  list.ptr[k] = ((uint64_t)(uintptr_t)ptr & ADDRESS_MASK) | ((uint64_t)dtype << 56);
  list.last[k] = (uint16_t)(over ? over : whole);
  list.first[k++] = units;
  const uint32_t u = (uint32_t)units_of(numel, dtype);
  if (streamed > 0) {
    const int64_t s = pieces(streamed, UNIT_BYTES);
    list.stream_until = units + (uint32_t)(s < u ? s : u);
  }
  streamed -= (int64_t)u * UNIT_BYTES;
  units += u;
}

template <size_t N> void end_of(uint32_t (&first)[N], int32_t from) {
  for (size_t i = (size_t)from; i < N; ++i) first[i] = NONE;
}

// closes the list; returns the workgroups of the norm's launch over it, each with per_block neighbouring units
template <class L> uint32_t close(L& list, int32_t k, uint32_t units) {
  list.first[k] = list.units = units;
  list.n = k;
  end_of(list.first, k + 1);
  list.per_block = (uint32_t)pieces(units, NORM_BLOCKS);
  if (!units) list.per_block = 1;
  return (uint32_t)pieces(units, list.per_block);
}

int32_t fill(TensorList& list, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t at, int32_t n, int64_t& streamed,
             uint32_t& blocks) {
  uint32_t units = 0;
  int32_t k = 0;
  list.stream_until = 0;
  while (k < LIST && at + k < n) {
    const int32_t i = at + k;
    append(list, k, units, tensors[i], numel[i], dtypes[i], streamed);
  }
  blocks = close(list, k, units);
  return k;
}

int64_t streamed_of(int64_t bytes) { return bytes >= STREAM_BYTES ? bytes : 0; }      // bytes read with the nontemporal hint, from the first on

// the partial values of all launches, one behind the other; returns their number.  `list` is left as the last launch had it
template <int P>
int norm_partials(TensorList& list, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int64_t bytes,
                  double* partial, hipStream_t st) {
  int64_t streamed = streamed_of(bytes);
  int count = 0;
  for (int32_t at = 0; at < n;) {
    uint32_t blocks;
    at += fill(list, tensors, numel, dtypes, at, n, streamed, blocks);
    if (blocks) norm_partial_kernel<P, false><<<blocks, NT, 0, st>>>(list, partial + count);
    count += (int)blocks;
  }
  return count;
}

template <int P>
int run_norm(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int64_t bytes, float* total, float* each, double* ws,
             hipStream_t st) {
  if (!each) {
    TensorList list;
    const int count = norm_partials<P>(list, tensors, numel, dtypes, n, bytes, ws, st);
    norm_total_kernel<P><<<1, NT, 0, st>>>(ws, count, total);
    return launch_status();
  }
  int64_t streamed = streamed_of(bytes);
  int count = 0;
  for (int32_t at = 0; at < n;) {
    TensorList list;
    uint32_t blocks;
    const int32_t took = fill(list, tensors, numel, dtypes, at, n, streamed, blocks);
    if (blocks) norm_partial_kernel<P, true><<<blocks, NT, 0, st>>>(list, ws + count);
    FirstUnits fu;
    for (int32_t i = 0; i <= took; ++i) fu.first[i] = list.first[i];
    fu.n = took;
    fu.per_block = list.per_block;
    const int here = blocks ? (int)blocks + took - 1 : 0;
    norm_each_kernel<P><<<(unsigned)pieces(took, NT / 64) + 1, NT, 0, st>>>(fu, ws + count, each + at, ws, count + here,
                                                                               at + took == n ? total : nullptr);
    count += here;
    at += took;
  }
  if (!n) norm_total_kernel<P><<<1, NT, 0, st>>>(ws, 0, total);
  return launch_status();
}

// scaling by the norm of the partial values, or, count < 0, by *given.  `filled`: the list of all tensors, where one holds
// them and it is there already
template <int P>
int run_scale(const TensorList* filled, void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int64_t bytes,
              const double* partial, int count, const float* given, float max_norm, float* total, hipStream_t st) {
  int64_t streamed = streamed_of(bytes);
  bool wrote = total == nullptr;
  TensorList own;
  for (int32_t at = 0; at < n;) {
    uint32_t blocks;
    at += filled ? n : fill(own, (const void* const*)tensors, numel, dtypes, at, n, streamed, blocks);
    const TensorList& list = filled ? *filled : own;
    const uint32_t units = list.units;
    if (!units) continue;
    scale_kernel<P><<<units < SCALE_BLOCKS ? units : SCALE_BLOCKS, NT, 0, st>>>(list, partial, count, given, max_norm, wrote ? nullptr : total);
    wrote = true;
  }
  if (!wrote) norm_total_kernel<P><<<1, NT, 0, st>>>(partial, count, total);      // no elements at all
  return launch_status();
}

template <int P>
int run_norm_clip(void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int64_t bytes, float max_norm, float* total,
                  double* ws, hipStream_t st) {
  TensorList list;
  const int count = norm_partials<P>(list, (const void* const*)tensors, numel, dtypes, n, bytes, ws, st);
  return run_scale<P>(n <= LIST ? &list : nullptr, tensors, numel, dtypes, n, bytes, ws, count, nullptr, max_norm, total, st);
}

size_t norm_workspace(int32_t n) {
  return ((size_t)pieces(n < 1 ? 1 : n, PREP_LIST < LIST ? PREP_LIST : LIST) * NORM_BLOCKS + (size_t)n + LIST) * sizeof(double);
}

size_t align64(size_t b) { return (b + 63) & ~(size_t)63; }

}  // namespace
}  // namespace pde_amd

using namespace pde_amd;

extern "C" {

size_t pde_amd_multi_workspace_bytes(int32_t n_tensors) {
  if (n_tensors < 0) return 0;
  return align64(norm_workspace(n_tensors)) + 64 + (size_t)n_tensors * sizeof(Prep);
}

int pde_amd_multi_norm(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, int32_t norm_type,
                       float* total, float* each, void* workspace, size_t workspace_bytes, void* stream) {
  int64_t bytes;
  const int status = check_tensors(tensors, numel, dtypes, n_tensors, bytes);
  if (status != PDE_AMD_OK) return status;
  if (!total || !workspace) return PDE_AMD_EINVAL;
  if (workspace_bytes < pde_amd_multi_workspace_bytes(n_tensors)) return PDE_AMD_EWORKSPACE;
  double* ws = (double*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (norm_type) {
    case NORM_INF: return run_norm<NORM_INF>(tensors, numel, dtypes, n_tensors, bytes, total, each, ws, st);
    case NORM_ONE: return run_norm<NORM_ONE>(tensors, numel, dtypes, n_tensors, bytes, total, each, ws, st);
    case NORM_TWO: return run_norm<NORM_TWO>(tensors, numel, dtypes, n_tensors, bytes, total, each, ws, st);
    default: return PDE_AMD_EINVAL;
  }
}

int pde_amd_multi_clip(void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, float max_norm,
                       const float* total, void* stream) {
  int64_t bytes;
  const int status = check_tensors((const void* const*)tensors, numel, dtypes, n_tensors, bytes);
  if (status != PDE_AMD_OK) return status;
  if (!total || !(max_norm >= 0.0f)) return PDE_AMD_EINVAL;
  return run_scale<NORM_TWO>(nullptr, tensors, numel, dtypes, n_tensors, bytes, nullptr, -1, total, max_norm, nullptr, (hipStream_t)stream);
}

int pde_amd_multi_norm_clip(void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, int32_t norm_type,
                            float max_norm, float* total, void* workspace, size_t workspace_bytes, void* stream) {
  int64_t bytes;
  const int status = check_tensors((const void* const*)tensors, numel, dtypes, n_tensors, bytes);
  if (status != PDE_AMD_OK) return status;
  if (!total || !workspace || !(max_norm >= 0.0f)) return PDE_AMD_EINVAL;
  if (workspace_bytes < pde_amd_multi_workspace_bytes(n_tensors)) return PDE_AMD_EWORKSPACE;
  double* ws = (double*)workspace;
  hipStream_t st = (hipStream_t)stream;
  switch (norm_type) {
    case NORM_INF: return run_norm_clip<NORM_INF>(tensors, numel, dtypes, n_tensors, bytes, max_norm, total, ws, st);
    case NORM_ONE: return run_norm_clip<NORM_ONE>(tensors, numel, dtypes, n_tensors, bytes, max_norm, total, ws, st);
    case NORM_TWO: return run_norm_clip<NORM_TWO>(tensors, numel, dtypes, n_tensors, bytes, max_norm, total, ws, st);
    default: return PDE_AMD_EINVAL;
  }
}

int pde_amd_multi_adamw_groups(const pde_amd_adamw_group* groups, int32_t n_groups, pde_amd_adamw_group* groups_device, void* stream) {
  if (n_groups < 1 || n_groups > PDE_AMD_ADAMW_MAX_GROUPS || !groups || !groups_device) return PDE_AMD_EINVAL;
  GroupList list = {};
  for (int32_t g = 0; g < n_groups; ++g) list.group[g] = groups[g];
  adamw_groups_kernel<<<1, 64, 0, (hipStream_t)stream>>>(list, n_groups, groups_device);
  return launch_status();
}

int pde_amd_multi_adamw(const pde_amd_adamw_tensor* table, const pde_amd_adamw_tensor* table_device, const void* const* grads, int32_t n_tensors,
                        const pde_amd_adamw_group* groups_device, int32_t n_groups, const float* lr, float max_norm, int32_t skip_nonfinite,
                        const float* total_in, float* total, void* workspace, size_t workspace_bytes, void* stream) {
  if (n_tensors < 0 || n_groups < 1 || n_groups > PDE_AMD_ADAMW_MAX_GROUPS || !groups_device || !lr || !workspace || max_norm != max_norm)
    return PDE_AMD_EINVAL;
  if (n_tensors > 0 && (!table || !table_device || !grads)) return PDE_AMD_EINVAL;
  const bool need_norm = max_norm >= 0.0f || skip_nonfinite, make_norm = need_norm && !total_in;
  if (make_norm && !total) return PDE_AMD_EINVAL;
  if (workspace_bytes < pde_amd_multi_workspace_bytes(n_tensors)) return PDE_AMD_EWORKSPACE;
  int64_t units = 0, bytes = 0;
  for (int32_t i = 0; i < n_tensors; ++i) {
    const pde_amd_adamw_tensor& t = table[i];
    if (t.numel < 0 || t.group < 0 || t.group >= n_groups || (t.dtype != PDE_AMD_F32 && t.dtype != PDE_AMD_BF16)) return PDE_AMD_EINVAL;
    if (t.numel > 0 && grads[i] && (!t.param || !t.exp_avg || !t.exp_avg_sq || !t.step || (t.dtype == PDE_AMD_BF16 && !t.master))) return PDE_AMD_EINVAL;
    const int64_t u = units_of(t.numel, t.dtype);
    if (u > MAX_UNITS - units || pieces(t.numel, STEP_UNIT) > MAX_STEP_UNITS) return PDE_AMD_ESHAPE;
    units += u;
    if (grads[i]) bytes += bytes_of(t.numel, t.dtype);
  }
  hipStream_t st = (hipStream_t)stream;
  double* partial = (double*)workspace;
  float* given_copy = (float*)((char*)workspace + align64(norm_workspace(n_tensors)));
  Prep* prep = (Prep*)((char*)given_copy + 64);
  const float* given = need_norm ? total_in : nullptr;
  int64_t streamed = bytes > KEEP_BYTES ? bytes - KEEP_BYTES : 0;
  int count = 0;
  bool any = false;
  for (int32_t at = 0; at < n_tensors;) {
    PrepList list;
    uint32_t u = 0;
    int32_t k = 0;
    list.stream_until = 0;
    list.base = at;
    while (k < PREP_LIST && at < n_tensors) {
      append(list, k, u, grads[at], grads[at] ? table[at].numel : 0, table[at].dtype, streamed);
      ++at;
    }
    const uint32_t blocks = close(list, k, u);
    if (!blocks) continue;
    for (int32_t g = 0; g < n_groups; ++g) list.lr[g] = lr[g];
    adamw_norm_kernel<<<(make_norm ? blocks : 0) + 1, NT, 0, st>>>(list, table_device, groups_device, prep, partial + count, given, given_copy);
    if (make_norm) count += (int)blocks;
    any = true;
  }
  if (!any && make_norm) norm_total_kernel<NORM_TWO><<<1, NT, 0, st>>>(partial, 0, total);
  ClipArgs clip;
  clip.partial = partial;
  clip.given = given ? given_copy : nullptr;
  clip.total = make_norm ? total : nullptr;
  clip.count = count;
  clip.skip_nonfinite = skip_nonfinite ? 1 : 0;
  clip.max_norm = max_norm;
  for (int32_t at = 0; at < n_tensors;) {
    StepList list;
    uint32_t u = 0;
    int32_t k = 0;
    list.base = at;
    for (; k < STEP_LIST && at < n_tensors; ++k, ++at) {
      const uint32_t more = grads[at] ? (uint32_t)pieces(table[at].numel, STEP_UNIT) : 0;
      if (more > (uint32_t)MAX_STEP_UNITS - u) break;
      list.grad[k] = (uint64_t)(uintptr_t)grads[at];
      list.first[k] = u;
      u += more;
    }
    list.first[k] = u;
    end_of(list.first, k + 1);
    if (!u) continue;
    adamw_update_kernel<<<u, NT, 0, st>>>(list, clip, table_device, prep);
    clip.total = nullptr;
  }
  return launch_status();
}

}  // extern "C"
