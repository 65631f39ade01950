// C ABI (include/pde_amd.h) of the weight update that follows a loss's backward pass: the norm of the gradients of many
// tensors, their scaling by it, and the AdamW step that applies the scaling while it reads the gradients.
//
// Every kernel walks a LIST of tensors.  A tensor is cut into units of UNIT elements, the units of all tensors are
// numbered through, and a workgroup takes a contiguous run of them, so the work per workgroup does not depend on how
// the elements are spread over tensors.  The list travels in the kernel's arguments (at most 4 KiB): nothing is copied
// to the device first, and a captured graph holds its own list.
#include "../../include/pde_amd.h"
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace pde_amd {
namespace {

constexpr int NT = 256;                  // threads of a workgroup
constexpr int UNIT = 4096;               // elements of a unit: 4 16-byte loads of fp32 per thread, 2 of a 16-bit type
constexpr int MAX_BLOCKS = 2048;         // workgroups of a launch: 8 per CU on 256 CUs
constexpr int LIST = 192;                // tensors of one launch of the norm and scaling kernels
constexpr int STEP_LIST = 224;           // tensors of one launch of the update kernel

// 16 bytes (and 8) of elements at any element-aligned address: gfx950 loads and stores them in one instruction
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h8 __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned short h4 __attribute__((ext_vector_type(4), aligned(2)));

// addresses come as numbers out of a list: said to be global memory, they are read with global rather than flat loads
template <class T> using gptr = __attribute__((address_space(1))) T*;

struct TensorList {
  uint64_t ptr[LIST];
  uint64_t size[LIST];                   // elements, dtype in the top 8 bits
  uint32_t first[LIST + 1];              // number of the tensor's first unit; first[n] = units of the launch
  int32_t n;
  uint32_t per_block;                    // units of a workgroup
};
static_assert(sizeof(TensorList) <= 4000, "the list has to fit the kernel's arguments");

__device__ __forceinline__ float bf16_to_float(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ float f16_to_float(unsigned short h) {
  _Float16 f;
  __builtin_memcpy(&f, &h, 2);
  return (float)f;
}
// round to nearest, ties to even (one rounding of a value held in 32 bits); NaN stays NaN
__device__ __forceinline__ unsigned short float_to_bf16(float x) {
  const unsigned u = __float_as_uint(x);
  if (x != x) return (unsigned short)((u >> 16) | 0x40u);
  return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ unsigned short float_to_f16(float x) {
  const _Float16 f = (_Float16)x;
  unsigned short h;
  __builtin_memcpy(&h, &f, 2);
  return h;
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

// the tensor that holds unit u: the last one whose first unit is <= u (tensors without elements share a first unit with
// their successor and are never the last such one)
__device__ __forceinline__ int find_tensor(const uint32_t* first, int n, uint32_t u) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= u) lo = mid; else hi = mid;
  }
  return lo;
}

// ------------------------------------------------------------------------------------------------
// norms.  Sums run in fp64: the square of any fp32 value is exact there and neither overflows nor vanishes, and the
// result does not depend on how the units are dealt out beyond the last bits of a double.
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

template <int DT, int P> __device__ __forceinline__ void add_unit(uint64_t ptr, long at, int count, Acc<P>& acc) {
  typedef Elem<DT> E;
  typedef typename E::V V;
  const gptr<const typename E::T> x = (gptr<const typename E::T>)ptr + at;
  constexpr int STEPS = UNIT / (NT * E::W);
  if (count == UNIT) {
    V v[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) v[s] = *(gptr<const V>)(x + (s * NT + (int)threadIdx.x) * E::W);
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int k = 0; k < E::W; ++k) acc.add(E::get(v[s][k]), k);
    return;
  }
  for (int i = threadIdx.x; i < count; i += NT) acc.add(E::get(x[i]), 0);
}

template <int P> __device__ __forceinline__ void add_unit_of(uint64_t ptr, uint64_t size, uint32_t unit, Acc<P>& acc) {
  const long n = (long)(size & 0xffffffffffffffull), at = (long)unit * UNIT;
  const int count = (int)(n - at < UNIT ? n - at : UNIT);
  switch ((int)(size >> 56)) {
    case PDE_AMD_F32: add_unit<PDE_AMD_F32, P>(ptr, at, count, acc); break;
    case PDE_AMD_BF16: add_unit<PDE_AMD_BF16, P>(ptr, at, count, acc); break;
    default: add_unit<PDE_AMD_F16, P>(ptr, at, count, acc); break;
  }
}

// EACH = false: one partial value per workgroup, partial[block].
// EACH = true: one per workgroup and tensor it touches, partial[block + tensor]: from one value to the next a workgroup
// moves to the next tensor or the launch to the next workgroup, so no two share a place.
template <int P, bool EACH>
__global__ __launch_bounds__(NT) void norm_partial_kernel(const TensorList list, double* __restrict__ partial) {
  __shared__ double lds[NT / 64];
  const uint32_t u0 = blockIdx.x * list.per_block;
  const uint32_t u1 = min(u0 + list.per_block, list.first[list.n]);
  int t = find_tensor(list.first, list.n, u0);
  Acc<P> acc;
  for (uint32_t u = u0; u < u1; ++u) {
    while (u >= list.first[t + 1]) {
      if (EACH && u > u0 && u == list.first[t + 1] && list.first[t] < list.first[t + 1]) {
        const double v = block_join<P>(acc.value(), lds);
        if (threadIdx.x == 0) partial[blockIdx.x + t] = v;
        acc = Acc<P>();
      }
      ++t;
    }
    add_unit_of<P>(list.ptr[t], list.size[t], u - list.first[t], acc);
  }
  const double v = block_join<P>(acc.value(), lds);
  if (threadIdx.x == 0) partial[blockIdx.x + (EACH ? t : 0)] = v;
}

template <int P> __device__ __forceinline__ float norm_of(double s) { return (float)(P == NORM_TWO ? sqrt(s) : s); }

// one workgroup: the value of all partial values, and the norm
template <int P>
__global__ __launch_bounds__(NT) void norm_total_kernel(const double* __restrict__ partial, int count, float* __restrict__ total) {
  __shared__ double lds[NT / 64];
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += NT) v = join<P>(v, partial[i]);
  v = block_join<P>(v, lds);
  if (threadIdx.x == 0) *total = norm_of<P>(v);
}

struct FirstUnits {
  uint32_t first[LIST + 1];
  int32_t n;
  uint32_t per_block;
};

// a wave per tensor: the value of its partial values, its norm, and the value for the total
template <int P>
__global__ __launch_bounds__(NT) void norm_each_kernel(const FirstUnits list, const double* __restrict__ partial, float* __restrict__ each,
                                                       double* __restrict__ sums) {
  const int t = blockIdx.x * (NT / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= list.n) return;
  double v = 0.0;
  if (list.first[t] < list.first[t + 1]) {
    const int b0 = (int)(list.first[t] / list.per_block), b1 = (int)((list.first[t + 1] - 1) / list.per_block);
    for (int b = b0 + lane; b <= b1; b += 64) v = join<P>(v, partial[b + t]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_down(v, o, 64));
  if (lane == 0) {
    each[t] = norm_of<P>(v);
    sums[t] = v;
  }
}

// ------------------------------------------------------------------------------------------------
// scaling by min(1, max_norm / (norm + 1e-6)), in 32 bits with one rounding to the tensor's type.  The +1e-6 (a norm of
// zero) and the order of operations are torch.nn.utils.clip_grad_norm_'s.  A factor of exactly one leaves every value as
// it is, so nothing is read or written then; a NaN norm makes the factor NaN.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float clip_factor(float max_norm, float total) {
  const float c = max_norm / (total + 1e-6f);
  return c > 1.0f ? 1.0f : c;
}

template <int DT> __device__ __forceinline__ void scale_unit(uint64_t ptr, long at, int count, float c) {
  typedef Elem<DT> E;
  typedef typename E::V V;
  const gptr<typename E::T> x = (gptr<typename E::T>)ptr + at;
  constexpr int STEPS = UNIT / (NT * E::W);
  if (count == UNIT) {
    V v[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) v[s] = *(gptr<const V>)(x + (s * NT + (int)threadIdx.x) * E::W);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int k = 0; k < E::W; ++k) v[s][k] = E::put(E::get(v[s][k]) * c);
      *(gptr<V>)(x + (s * NT + (int)threadIdx.x) * E::W) = v[s];
    }
    return;
  }
  for (int i = threadIdx.x; i < count; i += NT) x[i] = E::put(E::get(x[i]) * c);
}

__global__ __launch_bounds__(NT) void scale_kernel(const TensorList list, const float* __restrict__ total, float max_norm) {
  const float c = clip_factor(max_norm, *total);
  if (c == 1.0f) return;
  const uint32_t u0 = blockIdx.x * list.per_block;
  const uint32_t u1 = min(u0 + list.per_block, list.first[list.n]);
  int t = find_tensor(list.first, list.n, u0);
  for (uint32_t u = u0; u < u1; ++u) {
    while (u >= list.first[t + 1]) ++t;
    const uint64_t size = list.size[t];
    const long n = (long)(size & 0xffffffffffffffull), at = (long)(u - list.first[t]) * UNIT;
    const int count = (int)(n - at < UNIT ? n - at : UNIT);
    switch ((int)(size >> 56)) {
      case PDE_AMD_F32: scale_unit<PDE_AMD_F32>(list.ptr[t], at, count, c); break;
      case PDE_AMD_BF16: scale_unit<PDE_AMD_BF16>(list.ptr[t], at, count, c); break;
      default: scale_unit<PDE_AMD_F16>(list.ptr[t], at, count, c); break;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// AdamW.  With c the clipping factor, per element
//   g' = c g;  m <- b1 m + (1 - b1) g';  v <- b2 v + (1 - b2) g'^2
//   w <- (1 - lr wd) w - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in 32 bits; a 16-bit parameter is w rounded once, with w itself kept.  The step count t of every tensor lives on the
// device, so a captured step counts on, and a step that is skipped for a norm that is not finite does not.
// ------------------------------------------------------------------------------------------------
struct Prep {                            // what the update needs of a tensor's step, made by one thread
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, step_size, inv_sqrt_bias2;
};

struct StepHead {                        // ahead of the Preps in the workspace
  float factor;                          // clipping factor
  int32_t skip;                          // 1: the norm is not finite and the caller wants such steps skipped
  int32_t pad[6];
};

struct PrepArgs {
  uint32_t index[STEP_LIST];             // the tensor's place in the caller's table
  int32_t n;
  int32_t skip_nonfinite;
  float max_norm;                        // < 0: no clipping
  pde_amd_adamw_group group[PDE_AMD_ADAMW_MAX_GROUPS];
};
static_assert(sizeof(PrepArgs) <= 4000, "");

__global__ __launch_bounds__(NT) void adamw_prep_kernel(const PrepArgs a, const pde_amd_adamw_tensor* __restrict__ table,
                                                        const float* __restrict__ total, StepHead* __restrict__ head,
                                                        Prep* __restrict__ prep) {
  const bool clip = a.max_norm >= 0.0f;
  const float norm = total ? *total : 0.0f;
  const bool skip = a.skip_nonfinite && !(fabsf(norm) < INFINITY);
  if (threadIdx.x == 0) {
    head->factor = clip ? clip_factor(a.max_norm, norm) : 1.0f;
    head->skip = skip ? 1 : 0;
  }
  if (skip) return;
  for (int i = threadIdx.x; i < a.n; i += NT) {
    const pde_amd_adamw_tensor& t = table[a.index[i]];
    const pde_amd_adamw_group& g = a.group[t.group];
    const double lr = g.lr_device ? (double)*g.lr_device : g.lr;
    const float step = *t.step + 1.0f;
    *t.step = step;
    const double bias1 = 1.0 - pow(g.beta1, (double)step), bias2 = 1.0 - pow(g.beta2, (double)step);
    Prep p;
    p.beta1 = (float)g.beta1;
    p.one_minus_beta1 = (float)(1.0 - g.beta1);
    p.beta2 = (float)g.beta2;
    p.one_minus_beta2 = (float)(1.0 - g.beta2);
    p.eps = (float)g.eps;
    p.decay = (float)(1.0 - lr * g.weight_decay);
    p.step_size = (float)(lr / bias1);
    p.inv_sqrt_bias2 = (float)(1.0 / sqrt(bias2));
    prep[i] = p;
  }
}

struct StepList {
  uint64_t grad[STEP_LIST];
  uint32_t first[STEP_LIST + 1];
  uint32_t index[STEP_LIST];
  int32_t n;
  uint32_t per_block;
};
static_assert(sizeof(StepList) <= 4000, "");

__device__ __forceinline__ void adamw_one(float g, float& w, float& m, float& v, float c, const Prep& p) {
  g *= c;
  m = p.beta1 * m + p.one_minus_beta1 * g;
  v = p.beta2 * v + p.one_minus_beta2 * (g * g);
  w = p.decay * w - p.step_size * (m / (sqrtf(v) * p.inv_sqrt_bias2 + p.eps));
}

template <bool BF16>
__device__ __forceinline__ void adamw_unit(const pde_amd_adamw_tensor& t, uint64_t grad, long at, int count, float c, const Prep& p) {
  const gptr<float> w = (gptr<float>)(uint64_t)(BF16 ? (void*)t.master : t.param) + at;
  const gptr<float> m = (gptr<float>)(uint64_t)t.exp_avg + at, v = (gptr<float>)(uint64_t)t.exp_avg_sq + at;
  const gptr<const float> g32 = (gptr<const float>)grad + at;                        // the gradient, one of these
  const gptr<const unsigned short> g16 = (gptr<const unsigned short>)grad + at;
  const gptr<unsigned short> out = (gptr<unsigned short>)(uint64_t)t.param + at;      // BF16: the rounded weight
  if (count == UNIT) {
#pragma unroll
    for (int s = 0; s < UNIT / (NT * 4); ++s) {
      const int i = (s * NT + (int)threadIdx.x) * 4;
      f4 g4, w4 = *(gptr<const f4>)(w + i), m4 = *(gptr<const f4>)(m + i), v4 = *(gptr<const f4>)(v + i);
      if (BF16) {
        const h4 h = *(gptr<const h4>)(g16 + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) g4[k] = bf16_to_float(h[k]);
      } else {
        g4 = *(gptr<const f4>)(g32 + i);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float wk = w4[k], mk = m4[k], vk = v4[k];
        adamw_one(g4[k], wk, mk, vk, c, p);
        w4[k] = wk; m4[k] = mk; v4[k] = vk;
      }
      *(gptr<f4>)(w + i) = w4;
      *(gptr<f4>)(m + i) = m4;
      *(gptr<f4>)(v + i) = v4;
      if (BF16) {
        h4 h;
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = float_to_bf16(w4[k]);
        *(gptr<h4>)(out + i) = h;
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < count; i += NT) {
    float wk = w[i], mk = m[i], vk = v[i];
    adamw_one(BF16 ? bf16_to_float(g16[i]) : g32[i], wk, mk, vk, c, p);
    w[i] = wk; m[i] = mk; v[i] = vk;
    if (BF16) out[i] = float_to_bf16(wk);
  }
}

__global__ __launch_bounds__(NT) void adamw_update_kernel(const StepList list, const pde_amd_adamw_tensor* __restrict__ table,
                                                          const StepHead* __restrict__ head, const Prep* __restrict__ prep) {
  if (head->skip) return;
  const float c = head->factor;
  const uint32_t u0 = blockIdx.x * list.per_block;
  const uint32_t u1 = min(u0 + list.per_block, list.first[list.n]);
  int k = find_tensor(list.first, list.n, u0);
  for (uint32_t u = u0; u < u1; ++u) {
    while (u >= list.first[k + 1]) ++k;
    const pde_amd_adamw_tensor& t = table[list.index[k]];
    const long at = (long)(u - list.first[k]) * UNIT;
    const int count = (int)(t.numel - at < UNIT ? t.numel - at : UNIT);
    if (t.dtype == PDE_AMD_BF16) adamw_unit<true>(t, list.grad[k], at, count, c, prep[k]);
    else adamw_unit<false>(t, list.grad[k], at, count, c, prep[k]);
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
int launch_status() { return hipGetLastError() == hipSuccess ? PDE_AMD_OK : PDE_AMD_EHIP; }

int64_t units_of(int64_t n) { return n / UNIT + (n % UNIT != 0); }

// workgroups and units per workgroup of a launch over `units` units
void deal(int64_t units, uint32_t& per_block, uint32_t& blocks) {
  const int64_t per = (units + MAX_BLOCKS - 1) / MAX_BLOCKS;
  per_block = (uint32_t)(per < 1 ? 1 : per);
  blocks = (uint32_t)((units + per_block - 1) / per_block);
}

constexpr int64_t MAX_UNITS = 1ll << 31;      // of a launch: unit numbers stay in 32 bits

int check_tensors(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n) {
  if (n < 0 || (n > 0 && (!tensors || !numel || !dtypes))) return PDE_AMD_EINVAL;
  int64_t units = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || (numel[i] > 0 && !tensors[i]) || dtypes[i] < PDE_AMD_F32 || dtypes[i] > PDE_AMD_F16) return PDE_AMD_EINVAL;
    if (numel[i] > (MAX_UNITS - units) * UNIT) return PDE_AMD_ESHAPE;
    units += units_of(numel[i]);
  }
  return PDE_AMD_OK;
}

// fills `list` with tensors [at, ...) and returns how many it took
int32_t fill(TensorList& list, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t at, int32_t n, uint32_t& blocks) {
  int64_t units = 0;
  int32_t k = 0;
  for (; k < LIST && at + k < n; ++k) {
    list.ptr[k] = (uint64_t)(uintptr_t)tensors[at + k];
    list.size[k] = (uint64_t)numel[at + k] | ((uint64_t)dtypes[at + k] << 56);
    list.first[k] = (uint32_t)units;
    units += units_of(numel[at + k]);
  }
  list.first[k] = (uint32_t)units;
  list.n = k;
  deal(units, list.per_block, blocks);
  return k;
}

int32_t launches_of(int32_t n) { return (n + LIST - 1) / LIST; }

template <int P>
int run_norm(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, float* total, float* each, double* ws,
             hipStream_t st) {
  double* sums = ws;                     // EACH: [n] values of the tensors, then the partial values of a launch
  double* partial = each ? ws + n : ws;  // otherwise: the partial values of all launches, one behind the other
  int count = 0;
  for (int32_t at = 0; at < n;) {
    TensorList list;
    uint32_t blocks;
    const int32_t took = fill(list, tensors, numel, dtypes, at, n, blocks);
    if (each) {
      if (blocks) norm_partial_kernel<P, true><<<blocks, NT, 0, st>>>(list, partial);
      FirstUnits fu;
      for (int32_t i = 0; i <= took; ++i) fu.first[i] = list.first[i];
      fu.n = took;
      fu.per_block = list.per_block;
      norm_each_kernel<P><<<(took + 3) / 4, NT, 0, st>>>(fu, partial, each + at, sums + at);
    } else if (blocks) {
      norm_partial_kernel<P, false><<<blocks, NT, 0, st>>>(list, partial + count);
      count += (int)blocks;
    }
    at += took;
  }
  norm_total_kernel<P><<<1, NT, 0, st>>>(each ? sums : partial, each ? n : count, total);
  return launch_status();
}

int norm_any(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n, int32_t norm_type, float* total, float* each,
             double* ws, hipStream_t st) {
  switch (norm_type) {
    case NORM_INF: return run_norm<NORM_INF>(tensors, numel, dtypes, n, total, each, ws, st);
    case NORM_ONE: return run_norm<NORM_ONE>(tensors, numel, dtypes, n, total, each, ws, st);
    case NORM_TWO: return run_norm<NORM_TWO>(tensors, numel, dtypes, n, total, each, ws, st);
    default: return PDE_AMD_EINVAL;
  }
}

size_t norm_workspace(int32_t n) {
  return ((size_t)launches_of(n < 1 ? 1 : n) * MAX_BLOCKS + (size_t)(n < 0 ? 0 : n) + LIST) * sizeof(double);
}

size_t align64(size_t b) { return (b + 63) & ~(size_t)63; }

}  // namespace
}  // namespace pde_amd

using namespace pde_amd;

extern "C" {

size_t pde_amd_multi_workspace_bytes(int32_t n_tensors) {
  if (n_tensors < 0) return 0;
  return align64(norm_workspace(n_tensors)) + sizeof(StepHead) + (size_t)n_tensors * sizeof(Prep) + 64;
}

int pde_amd_multi_norm(const void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, int32_t norm_type,
                       float* total, float* each, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_tensors(tensors, numel, dtypes, n_tensors);
  if (st != PDE_AMD_OK) return st;
  if (!total || !workspace || norm_type < NORM_INF || norm_type > NORM_TWO) return PDE_AMD_EINVAL;
  if (workspace_bytes < pde_amd_multi_workspace_bytes(n_tensors)) return PDE_AMD_EWORKSPACE;
  return norm_any(tensors, numel, dtypes, n_tensors, norm_type, total, each, (double*)workspace, (hipStream_t)stream);
}

int pde_amd_multi_clip(void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, float max_norm,
                       const float* total, void* stream) {
  const int st = check_tensors((const void* const*)tensors, numel, dtypes, n_tensors);
  if (st != PDE_AMD_OK) return st;
  if (!total || !(max_norm >= 0.0f)) return PDE_AMD_EINVAL;
  for (int32_t at = 0; at < n_tensors;) {
    TensorList list;
    uint32_t blocks;
    at += fill(list, (const void* const*)tensors, numel, dtypes, at, n_tensors, blocks);
    if (blocks) scale_kernel<<<blocks, NT, 0, (hipStream_t)stream>>>(list, total, max_norm);
  }
  return launch_status();
}

int pde_amd_multi_norm_clip(void* const* tensors, const int64_t* numel, const int32_t* dtypes, int32_t n_tensors, int32_t norm_type,
                            float max_norm, float* total, void* workspace, size_t workspace_bytes, void* stream) {
  if (!(max_norm >= 0.0f)) return PDE_AMD_EINVAL;
  const int st = pde_amd_multi_norm((const void* const*)tensors, numel, dtypes, n_tensors, norm_type, total, nullptr, workspace,
                                    workspace_bytes, stream);
  return st != PDE_AMD_OK ? st : pde_amd_multi_clip(tensors, numel, dtypes, n_tensors, max_norm, total, stream);
}

int pde_amd_multi_adamw(const pde_amd_adamw_tensor* table, const pde_amd_adamw_tensor* table_device, const void* const* grads, int32_t n_tensors,
                        const pde_amd_adamw_group* groups, int32_t n_groups, float max_norm, int32_t skip_nonfinite,
                        const float* total_in, float* total, void* workspace, size_t workspace_bytes, void* stream) {
  if (n_tensors < 0 || n_groups < 1 || n_groups > PDE_AMD_ADAMW_MAX_GROUPS || !groups || !workspace || max_norm != max_norm) return PDE_AMD_EINVAL;
  if (n_tensors > 0 && (!table || !table_device || !grads)) return PDE_AMD_EINVAL;
  const bool need_norm = max_norm >= 0.0f || skip_nonfinite;
  if (need_norm && !total_in && !total) return PDE_AMD_EINVAL;
  if (workspace_bytes < pde_amd_multi_workspace_bytes(n_tensors)) return PDE_AMD_EWORKSPACE;
  int64_t units = 0;
  for (int32_t i = 0; i < n_tensors; ++i) {
    const pde_amd_adamw_tensor& t = table[i];
    if (t.numel < 0 || t.group < 0 || t.group >= n_groups || (t.dtype != PDE_AMD_F32 && t.dtype != PDE_AMD_BF16)) return PDE_AMD_EINVAL;
    if (t.numel > 0 && grads[i] && (!t.param || !t.exp_avg || !t.exp_avg_sq || !t.step || (t.dtype == PDE_AMD_BF16 && !t.master))) return PDE_AMD_EINVAL;
    if (t.numel > (MAX_UNITS - units) * UNIT) return PDE_AMD_ESHAPE;
    units += units_of(t.numel);
  }
  hipStream_t st = (hipStream_t)stream;
  if (need_norm && !total_in) {
    // the tensors that have a gradient, a launch's worth at a time
    double* partial = (double*)workspace;
    int count = 0;
    for (int32_t at = 0; at < n_tensors;) {
      TensorList list;
      int64_t u = 0;
      int32_t k = 0;
      for (; at < n_tensors && k < LIST; ++at) {
        if (!grads[at] || table[at].numel == 0) continue;
        list.ptr[k] = (uint64_t)(uintptr_t)grads[at];
        list.size[k] = (uint64_t)table[at].numel | ((uint64_t)table[at].dtype << 56);
        list.first[k++] = (uint32_t)u;
        u += units_of(table[at].numel);
      }
      list.first[k] = (uint32_t)u;
      list.n = k;
      uint32_t blocks;
      deal(u, list.per_block, blocks);
      if (blocks) norm_partial_kernel<NORM_TWO, false><<<blocks, NT, 0, st>>>(list, partial + count);
      count += (int)blocks;
    }
    norm_total_kernel<NORM_TWO><<<1, NT, 0, st>>>(partial, count, total);
    total_in = total;
  }
  char* rest = (char*)workspace + align64(norm_workspace(n_tensors));
  StepHead* head = (StepHead*)rest;
  Prep* prep = (Prep*)(rest + sizeof(StepHead));
  PrepArgs pa;
  pa.skip_nonfinite = skip_nonfinite ? 1 : 0;
  pa.max_norm = max_norm;
  for (int32_t g = 0; g < n_groups; ++g) pa.group[g] = groups[g];
  for (int32_t at = 0; at < n_tensors;) {
    StepList list;
    int64_t u = 0;
    int32_t k = 0;
    for (; at < n_tensors && k < STEP_LIST; ++at) {
      if (!grads[at]) continue;
      list.grad[k] = (uint64_t)(uintptr_t)grads[at];
      list.index[k] = pa.index[k] = (uint32_t)at;
      list.first[k++] = (uint32_t)u;
      u += units_of(table[at].numel);
    }
    list.first[k] = (uint32_t)u;
    list.n = pa.n = k;
    if (!k) break;
    uint32_t blocks;
    deal(u, list.per_block, blocks);
    adamw_prep_kernel<<<1, NT, 0, st>>>(pa, table_device, need_norm ? total_in : nullptr, head, prep);
    if (blocks) adamw_update_kernel<<<blocks, NT, 0, st>>>(list, table_device, head, prep);
  }
  return launch_status();
}

}  // extern "C"
