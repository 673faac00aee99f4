// Global 2-norm of many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum_t sum_i g_t[i]^2),   g_t[i] *= min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: one read of every gradient for the norm, one more read and a write when it clips.
// The tensors of a call lie anywhere and have any type and size, so the work is cut into units of kUnit
// elements numbered over all tensors, and every workgroup takes one run of consecutive units: equal shares
// whatever the sizes are, one search for the first tensor and a step to the next where a run crosses over.
// The tensors' addresses travel in the launch's arguments (kJobs of them a launch, no table in device memory to
// fill, so a launch can be captured).
//
// Squares are summed in 64 bits: fp64 has the rate of unpacked fp32 here and the pass waits for memory, so it
// costs nothing; the squares of gradients near 1e20 or 1e-25 neither overflow nor vanish.  Each workgroup leaves
// one partial sum, and one workgroup adds the partials in a fixed order: no atomics, the same bits every call.
#include "common.h"

#include <vector>

namespace dta {

constexpr int kJobs = 160;       // 160 x 20 B of arguments stay under 4 KiB
constexpr int kUnit = 8192;      // elements: 4 (2 bytes) to 16 (8 bytes) 16-byte loads a thread
constexpr int kNormGrid = 8192;  // workgroups at most (1.4 G bf16 elements: 1459 us, 1514 with 2048, 1462 with 16384)

// The norm's pass reads with non-temporal loads (6.9 TB/s, 5.4 without), except for what the Infinity Cache can hold
// until the clipping pass: the last kKeep bytes, which that pass, walking each workgroup's run backwards, meets first.
// Norm and clip together, bf16: 124 M elements 128 us, 150 with nothing kept; 1.4 G 1513, 1529 with nothing kept.
constexpr int64_t kKeep = 192 << 20;

struct NormJobs {
  int n;
  int units;               // of this launch
  int keep;                // units at the end of each workgroup's run that are read into the caches
  int start[kJobs + 1];    // first unit of each tensor
  void* p[kJobs];
  int64_t numel_type[kJobs];  // numel * 4 + type (0 f32, 1 bf16, 2 f16, 3 f64)
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
// 16-byte accesses at any element address (a gradient may be a slice at an odd offset)
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));
typedef half8 half8_u __attribute__((aligned(2)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef f64x2 f64x2_u __attribute__((aligned(8)));

template <typename T> struct Pack;
template <> struct Pack<bf16> { typedef bf16x8_u V; static constexpr int n = 8; };
template <> struct Pack<_Float16> { typedef half8_u V; static constexpr int n = 8; };
template <> struct Pack<float> { typedef f32x4_u V; static constexpr int n = 4; };
template <> struct Pack<double> { typedef f64x2_u V; static constexpr int n = 2; };

template <bool NT, typename V>
__device__ __forceinline__ V load_v(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load(static_cast<const V*>(p));
  else return *static_cast<const V*>(p);
}

template <bool NT, typename T>
__device__ __forceinline__ double sumsq_unit(const T* __restrict__ p, int64_t c0, int64_t numel) {
  constexpr int W = Pack<T>::n, STEP = 256 * W, LOADS = kUnit / STEP, U = LOADS < 4 ? LOADS : 4;
  double acc = 0.0;
  if (c0 + kUnit <= numel) {
    for (int l = 0; l < LOADS; l += U) {
      typename Pack<T>::V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = load_v<NT, typename Pack<T>::V>(p + c0 + (l + u) * STEP + threadIdx.x * W);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const double d = (double)v[u][j];
          acc = fma(d, d, acc);
        }
    }
  } else {  // a tensor's end: whole vectors, then up to W - 1 elements
    const int64_t end = numel - (numel - c0) % W;
#pragma unroll 4
    for (int64_t i = c0 + threadIdx.x * W; i < end; i += STEP) {
      const typename Pack<T>::V v = load_v<false, typename Pack<T>::V>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const double d = (double)v[j];
        acc = fma(d, d, acc);
      }
    }
    if (end + threadIdx.x < numel) {
      const double d = (double)p[end + threadIdx.x];
      acc = fma(d, d, acc);
    }
  }
  return acc;
}

// The coefficient is used in fp32 (2^-24 relative; fp64 gradients take it whole) and each product rounded to T.  Below
// fp32's normal numbers (gradients near 1e38) it would lose bits: it is held 2^64 times as large there, and `rest` takes
// the product back (exactly, or with the one rounding of a subnormal product).
struct Coef {
  double whole;
  float f, rest;
  __device__ __forceinline__ explicit Coef(double c) : whole(c) {
    const bool tiny = c < 0x1p-126;
    f = (float)(tiny ? c * 0x1p64 : c);
    rest = tiny ? 0x1p-64f : 1.f;
  }
};
template <typename T>
__device__ __forceinline__ T scaled(T x, const Coef& c) {
  if constexpr (sizeof(T) == 8) return x * c.whole;
  else return (T)((float)x * c.f * c.rest);
}
template <typename T>
__device__ __forceinline__ void scale_unit(T* __restrict__ p, int64_t c0, int64_t numel, const Coef& coef) {
  constexpr int W = Pack<T>::n, STEP = 256 * W, LOADS = kUnit / STEP, U = LOADS < 4 ? LOADS : 4;
  if (c0 + kUnit <= numel) {
    for (int l = 0; l < LOADS; l += U) {
      typename Pack<T>::V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = load_v<true, typename Pack<T>::V>(p + c0 + (l + u) * STEP + threadIdx.x * W);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[u][j] = scaled<T>(v[u][j], coef);
        __builtin_nontemporal_store(
            v[u], reinterpret_cast<typename Pack<T>::V*>(p + c0 + (l + u) * STEP + threadIdx.x * W));
      }
    }
  } else {
    const int64_t end = numel - (numel - c0) % W;
#pragma unroll 4
    for (int64_t i = c0 + threadIdx.x * W; i < end; i += STEP) {
      typename Pack<T>::V v = load_v<false, typename Pack<T>::V>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = scaled<T>(v[j], coef);
      *reinterpret_cast<typename Pack<T>::V*>(p + i) = v;
    }
    if (end + threadIdx.x < numel) p[end + threadIdx.x] = scaled<T>(p[end + threadIdx.x], coef);
  }
}

// The tensor that unit u belongs to: the last one that starts at or before it
__device__ __forceinline__ int tensor_of(const NormJobs& jobs, int u) {
  int lo = 0, hi = jobs.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (jobs.start[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// This workgroup's run of units, from its end to its start where BACK: f(pointer, type, first element, numel, whether
// the unit is one of the `keep` at the end)
template <bool BACK, typename F>
__device__ __forceinline__ void walk_units(const NormJobs& jobs, F f) {
  const int u0 = (int)((int64_t)jobs.units * blockIdx.x / gridDim.x);
  const int u1 = (int)((int64_t)jobs.units * (blockIdx.x + 1) / gridDim.x);
  if (u0 >= u1) return;
  int j = tensor_of(jobs, BACK ? u1 - 1 : u0);
  for (int i = 0; i < u1 - u0; ++i) {
    const int u = BACK ? u1 - 1 - i : u0 + i;
    if (BACK) while (u < jobs.start[j]) --j;
    else while (u >= jobs.start[j + 1]) ++j;
    const int64_t nt = jobs.numel_type[j];
    f(jobs.p[j], (int)(nt & 3), (int64_t)(u - jobs.start[j]) * kUnit, nt >> 2, u >= u1 - jobs.keep);
  }
}

template <bool NT>
__device__ __forceinline__ double sumsq_of(const void* p, int type, int64_t c0, int64_t numel) {
  if (type == 1) return sumsq_unit<NT>((const bf16*)p, c0, numel);
  if (type == 0) return sumsq_unit<NT>((const float*)p, c0, numel);
  if (type == 2) return sumsq_unit<NT>((const _Float16*)p, c0, numel);
  return sumsq_unit<NT>((const double*)p, c0, numel);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

template <int NT>
__device__ __forceinline__ double block_sum64(double v) {
  __shared__ double red[NT / 64];
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) s += red[w];
  return s;
}

__global__ void __launch_bounds__(256) grad_sumsq_kernel(NormJobs jobs, double* __restrict__ part) {
  double acc = 0.0;
  walk_units<false>(jobs, [&](void* p, int type, int64_t c0, int64_t numel, bool keep) {
    acc += keep ? sumsq_of<false>(p, type, c0, numel) : sumsq_of<true>(p, type, c0, numel);
  });
  acc = block_sum64<256>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// sumsq[0] = sum of the partials, norm[0] = its root in fp32
__global__ void __launch_bounds__(1024) grad_norm_kernel(const double* __restrict__ part, int n,
                                                         double* __restrict__ sumsq, float* __restrict__ norm) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) acc += part[i];
  acc = block_sum64<1024>(acc);
  if (threadIdx.x == 0) {
    *sumsq = acc;
    *norm = (float)sqrt(acc);
  }
}

// A norm within the bound leaves every gradient as it is: the workgroups end without touching them.  A NaN norm
// gives a NaN coefficient (not 1), an infinite one 0, as min(1, max_norm / (norm + 1e-6)) says.
__device__ __forceinline__ void clip_units(const NormJobs& jobs, double root, double max_norm) {
  const double c = max_norm / (root + 1e-6);
  if (c >= 1.0) return;
  const Coef coef(c);
  walk_units<true>(jobs, [&](void* p, int type, int64_t c0, int64_t numel, bool) {
    if (type == 1) scale_unit((bf16*)p, c0, numel, coef);
    else if (type == 0) scale_unit((float*)p, c0, numel, coef);
    else if (type == 2) scale_unit((_Float16*)p, c0, numel, coef);
    else scale_unit((double*)p, c0, numel, coef);
  });
}
__global__ void __launch_bounds__(256) grad_clip_kernel(NormJobs jobs, const double* __restrict__ sumsq,
                                                        double max_norm) {
  clip_units(jobs, sqrt(*sumsq), max_norm);
}
// For few partial sums: every workgroup adds them up itself, which spares the launch of grad_norm_kernel.  A pass in us,
// two launches / three: 30 K fp32 elements in 40 tensors 14.3 / 19.5, 2 M in 4 tensors 11.1 / 15.1, 8 M (977 partial
// sums) 15.2 / 16.4; the read of the sums grows with the square of their number, so it stops there.
constexpr int kJoined = 1024;
__global__ void __launch_bounds__(256) grad_clip_joined_kernel(NormJobs jobs, const double* __restrict__ part, int n,
                                                               float* __restrict__ norm, double max_norm) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += part[i];
  const double root = sqrt(block_sum64<256>(acc));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)root;
  clip_units(jobs, root, max_norm);
}

// Norm and clip of a small model in one launch of one workgroup (a wave a unit of kSmallUnit elements): the other forms
// are mostly launches there.  A pass in us, one launch / two: 100 elements 4.5 / 10.7, 11 K in 4 tensors (23 units)
// 7.3 / 10.7, 4 K in 64 tensors (64 units) 11.9 / 15.9, 32 K in 4 tensors (64 units) 13.1 / 11.1, or 7.6 / 10.9 where the
// norm is within the bound.
constexpr int kSmallUnit = 512, kSmallUnits = 64;

template <typename T>
__device__ __forceinline__ double small_sumsq(const T* p, int64_t c0, int64_t numel) {
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < kSmallUnit / 64; ++k) {
    const int64_t i = c0 + k * 64 + (threadIdx.x & 63);
    const double d = i < numel ? (double)p[i] : 0.0;
    acc = fma(d, d, acc);
  }
  return acc;
}
template <typename T>
__device__ __forceinline__ void small_scale(T* p, int64_t c0, int64_t numel, const Coef& coef) {
#pragma unroll
  for (int k = 0; k < kSmallUnit / 64; ++k) {
    const int64_t i = c0 + k * 64 + (threadIdx.x & 63);
    if (i < numel) p[i] = scaled<T>(p[i], coef);
  }
}

__global__ void __launch_bounds__(1024) grad_clip_small_kernel(NormJobs jobs, double max_norm,
                                                               float* __restrict__ norm) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto walk = [&](auto f) {
    for (int u = wave; u < jobs.units; u += 16) {
      const int j = tensor_of(jobs, u);
      f(jobs.p[j], (int)(jobs.numel_type[j] & 3), (int64_t)(u - jobs.start[j]) * kSmallUnit, jobs.numel_type[j] >> 2);
    }
  };
  double acc = 0.0;
  walk([&](void* p, int type, int64_t c0, int64_t numel) {
    if (type == 1) acc += small_sumsq((const bf16*)p, c0, numel);
    else if (type == 0) acc += small_sumsq((const float*)p, c0, numel);
    else if (type == 2) acc += small_sumsq((const _Float16*)p, c0, numel);
    else acc += small_sumsq((const double*)p, c0, numel);
  });
  const double root = sqrt(block_sum64<1024>(acc));
  if (threadIdx.x == 0) *norm = (float)root;
  const double c = max_norm / (root + 1e-6);
  if (c >= 1.0) return;
  const Coef coef(c);
  walk([&](void* p, int type, int64_t c0, int64_t numel) {
    if (type == 1) small_scale((bf16*)p, c0, numel, coef);
    else if (type == 0) small_scale((float*)p, c0, numel, coef);
    else if (type == 2) small_scale((_Float16*)p, c0, numel, coef);
    else small_scale((double*)p, c0, numel, coef);
  });
}

// The launches' tables for `count` tensors, in units of kUnit elements
static std::vector<NormJobs> tables(void* const* p, const int64_t* numel, const int* type, int count,
                                    int64_t unit = kUnit) {
  constexpr int64_t kMostUnits = 1 << 30;
  std::vector<NormJobs> all;
  int i = 0;
  int64_t done = 0;  // elements of tensor i that earlier launches took
  while (i < count) {
    all.emplace_back();
    NormJobs& jobs = all.back();
    int64_t units = 0, bytes = 0;
    int n = 0;
    while (i < count && n < kJobs && units < kMostUnits) {
      const int64_t left = numel[i] - done, need = (left + unit - 1) / unit;
      const int64_t take = need < kMostUnits - units ? need : kMostUnits - units;
      if (take > 0) {
        const int64_t elems = take == need ? left : take * unit;
        const int size = type[i] == 0 ? 4 : type[i] == 3 ? 8 : 2;
        jobs.p[n] = static_cast<char*>(p[i]) + done * size;
        jobs.numel_type[n] = elems * 4 + type[i];
        jobs.start[n++] = (int)units;
        units += take;
        done += elems;
        bytes += elems * size;
      }
      if (take == need) {
        ++i;
        done = 0;
      }
    }
    jobs.n = n;
    jobs.units = (int)units;
    jobs.start[n] = (int)units;
    // a workgroup's share of kKeep, in units of this launch's mean size
    jobs.keep = bytes <= kKeep ? (int)units : (int)((double)kKeep / (double)bytes * (double)units / kNormGrid);
    if (n == 0) all.pop_back();
  }
  return all;
}
static int workgroups(const NormJobs& jobs) { return jobs.units < kNormGrid ? jobs.units : kNormGrid; }

}  // namespace dta

using namespace dta;

// Partial sums that dta_grad_sumsq needs room for (doubles)
int64_t dta_grad_sumsq_parts(const int64_t* numel, int count) {
  int64_t units = 0;
  for (int i = 0; i < count; ++i) units += (numel[i] + kUnit - 1) / kUnit;
  // full tables, plus the tables that a launch's limit on units cuts short (two for each cut), plus the last
  return (count / kJobs + 2 * (units >> 30) + 1) * (units < kNormGrid ? units + 1 : kNormGrid);
}

static hipError_t partial_sums(const std::vector<NormJobs>& all, double* part, int64_t parts, int* used,
                               hipStream_t st) {
  *used = 0;
  for (const NormJobs& jobs : all) {
    const int grid = workgroups(jobs);
    if (*used + grid > parts) return hipErrorInvalidValue;
    hipLaunchKernelGGL(grad_sumsq_kernel, dim3(grid), dim3(256), 0, st, jobs, part + *used);
    DTA_HIP_CHECK(hipGetLastError());
    *used += grid;
  }
  return hipSuccess;
}
static hipError_t clip_by(const std::vector<NormJobs>& all, const double* sumsq, double max_norm, hipStream_t st) {
  for (size_t i = all.size(); i-- > 0;) {  // the last launch's gradients are the ones that are still cached
    hipLaunchKernelGGL(grad_clip_kernel, dim3(workgroups(all[i])), dim3(256), 0, st, all[i], sumsq, max_norm);
    DTA_HIP_CHECK(hipGetLastError());
  }
  return hipSuccess;
}

// sumsq (1 double), norm (1 float); part: dta_grad_sumsq_parts doubles of scratch
hipError_t dta_grad_sumsq(void* const* p, const int64_t* numel, const int* type, int count, double* part,
                          int64_t parts, double* sumsq, float* norm, hipStream_t st) {
  int used;
  DTA_HIP_CHECK(partial_sums(tables(p, numel, type, count), part, parts, &used, st));
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, st, part, used, sumsq, norm);
  return hipGetLastError();
}

hipError_t dta_grad_clip(void* const* p, const int64_t* numel, const int* type, int count, const double* sumsq,
                         double max_norm, hipStream_t st) {
  return clip_by(tables(p, numel, type, count), sumsq, max_norm, st);
}

// dta_grad_sumsq and dta_grad_clip in one
hipError_t dta_grad_clip_norm(void* const* p, const int64_t* numel, const int* type, int count, double* part,
                              int64_t parts, double* sumsq, float* norm, double max_norm, hipStream_t st) {
  const std::vector<NormJobs> all = tables(p, numel, type, count);
  int used;
  DTA_HIP_CHECK(partial_sums(all, part, parts, &used, st));
  if (all.size() == 1 && used <= kJoined) {
    hipLaunchKernelGGL(grad_clip_joined_kernel, dim3(workgroups(all[0])), dim3(256), 0, st, all[0], part, used, norm,
                       max_norm);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, st, part, used, sumsq, norm);
  DTA_HIP_CHECK(hipGetLastError());
  return clip_by(all, sumsq, max_norm, st);
}

// Whether the gradients are few enough for dta_grad_clip_small
int dta_grad_is_small(const int64_t* numel, int count) {
  int64_t units = 0;
  if (count > kJobs) return 0;
  for (int i = 0; i < count && units <= kSmallUnits; ++i) units += (numel[i] + kSmallUnit - 1) / kSmallUnit;
  return units <= kSmallUnits;
}

// dta_grad_clip_norm in one launch
hipError_t dta_grad_clip_small(void* const* p, const int64_t* numel, const int* type, int count, double max_norm,
                               float* norm, hipStream_t st) {
  if (!dta_grad_is_small(numel, count)) return hipErrorInvalidValue;
  const std::vector<NormJobs> all = tables(p, numel, type, count, kSmallUnit);
  NormJobs none{};
  hipLaunchKernelGGL(grad_clip_small_kernel, dim3(1), dim3(1024), 0, st, all.empty() ? none : all[0], max_norm, norm);
  return hipGetLastError();
}
