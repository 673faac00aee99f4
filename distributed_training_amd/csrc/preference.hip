// Losses that train a model on rewards or preferences, from its logits [B, S, V]: token log-probabilities, the
// clipped policy loss with a KL term, and the paired preference loss; forward and backward.
//
//   c = log2(e) / temperature,  M = max_j z_j,  s = sum_j 2^((z_j - M) c)
//   lp = (z_y - M) / temperature - ln s                              log-probability of the token y
//   dz_j = k ([j = y] - 2^((z_j - M) c - log2 s)),  k = dloss/dlp / temperature
//
// Three steps: every row's (M, s) (lse_partial_kernel, one pass over the logits, a row cut into pieces where there
// are few); the rows' terms and the loss (one thread a row, then one workgroup); dz (logit_grad_kernel, a second
// read of the logits and a write).  Both passes over the logits wait for memory.
//
// The row's maximum is subtracted before the multiplication by c, not folded into one fma: rows of the type's lowest
// value then keep their uniform distribution instead of overflowing.  Sums of exponentials are fp32; what follows
// per row (logarithm, ratio, KL term) and the sums over rows are fp64, since 1 - ratio, exp(d) - d - 1 and the
// difference of two sequences' sums cancel.  It is one thread's work a row: free beside V exponentials.
//
// A row whose target is ignore_index or lies outside [0, V) counts for nothing: its logits are not read (they may hold
// anything) and its gradient is written as zero.  Reductions have a fixed order: the same bits every call.
#include "common.h"

namespace dta {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
// 16-byte accesses at any element address: rows of an odd vocabulary begin anywhere
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));
typedef half8 half8_u __attribute__((aligned(2)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));

template <typename T> struct Row8;  // 8 logits as they lie in memory
template <> struct Row8<bf16> {
  bf16x8 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const bf16x8_u*>(p); }
  __device__ __forceinline__ float get(int j) const { return bf2f(v[j]); }
  __device__ __forceinline__ void set(int j, float x) { v[j] = f2bf(x); }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<bf16x8_u*>(p) = v; }
};
template <> struct Row8<_Float16> {
  half8 v;
  __device__ __forceinline__ void load(const _Float16* p) { v = *reinterpret_cast<const half8_u*>(p); }
  __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
  __device__ __forceinline__ void set(int j, float x) { v[j] = (_Float16)x; }
  __device__ __forceinline__ void store(_Float16* p) const { *reinterpret_cast<half8_u*>(p) = v; }
};
template <> struct Row8<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4_u*>(p);
    b = *reinterpret_cast<const f32x4_u*>(p + 4);
  }
  __device__ __forceinline__ float get(int j) const { return j < 4 ? a[j & 3] : b[j & 3]; }
  __device__ __forceinline__ void set(int j, float x) {
    if (j < 4) a[j & 3] = x;
    else b[j & 3] = x;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<f32x4_u*>(p) = a;
    *reinterpret_cast<f32x4_u*>(p + 4) = b;
  }
};
// the chunk [c, c + 8) of a row of V: past the end -inf on loads, left alone on stores
template <typename T>
__device__ __forceinline__ void load_chunk(Row8<T>& r, const T* x, int64_t c, int64_t V) {
  if (c + 8 <= V) {
    r.load(x + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.set(j, c + j < V ? (float)x[c + j] : -INFINITY);
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(const Row8<T>& r, T* x, int64_t c, int64_t V) {
  if (c + 8 <= V) {
    r.store(x + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < V) x[c + j] = (T)r.get(j);
  }
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// [B, S, V] logits (rows of unit inner stride) and the [B, S] per-token arrays that go with them
struct Logits {
  const void* z;
  int64_t sb, ss;  // element strides of a sequence and of a token
  const int64_t* target;
  int64_t tb, ts;
  int64_t B, S, V, ignore;
  __device__ __forceinline__ int64_t target_of(int64_t b, int64_t s) const {  // -1: the row does not count
    const int64_t t = target[b * tb + s * ts];
    return t == ignore || t < 0 || t >= V ? -1 : t;
  }
};
struct TokenArray {  // fp32 [B, S] of any strides (0: broadcast); p null where absent
  const float* p;
  int64_t sb, ss;
  __device__ __forceinline__ float at(int64_t b, int64_t s) const { return p[b * sb + s * ss]; }
};

// What the gradient needs of a row
struct RowState {
  float M, l2s, coef, pad;  // coef: dloss/dlp without the sequence's weight
};

constexpr int kLseThreads = 256;
constexpr int kSegRows = 256;  // rows of one workgroup in the passes over rows

// ------------------------------------------------------------------ (M, s) of every row
// Workgroup row * pieces + i: piece i of the row, [i * span, (i + 1) * span).  U chunks a thread are requested before
// any is used and share one rescaling of the running sum.
template <typename T>
__global__ void __launch_bounds__(kLseThreads) lse_partial_kernel(Logits L, float c, int pieces, int64_t span,
                                                                  float2* __restrict__ part) {
  constexpr int NW = kLseThreads / 64, U = sizeof(T) == 4 ? 2 : 4;
  const int64_t row = blockIdx.x / pieces;
  const int64_t b = row / L.S, s0 = row % L.S;
  if (L.target_of(b, s0) < 0) return;
  const T* x = static_cast<const T*>(L.z) + b * L.sb + s0 * L.ss;
  const int64_t begin = (int64_t)(blockIdx.x % pieces) * span, end = min(begin + span, L.V);
  float m = -INFINITY, s = 0.f;
  for (int64_t c0 = begin + threadIdx.x * 8; c0 < end; c0 += kLseThreads * 8 * U) {
    Row8<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t cc = c0 + u * kLseThreads * 8;
      if (cc < end) load_chunk(r[u], x, cc, end);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * kLseThreads * 8 < end)
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = fmaxf(mn, r[u].get(j));
    const float ms = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: the sum stays 0, not NaN
    s *= exp2_((m - ms) * c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * kLseThreads * 8 < end)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += exp2_((r[u].get(j) - ms) * c);
    m = mn;
  }
  __shared__ float sm[NW], sv[NW];
  const float wm = wave_max(m);
  const float wms = wm == -INFINITY ? 0.f : wm;
  s = wave_sum(s * exp2_((m - wms) * c));
  if ((threadIdx.x & 63) == 0) {
    sm[threadIdx.x >> 6] = wm;
    sv[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float M = sm[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, sm[w]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float S = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) S += sv[w] * exp2_((sm[w] - Ms) * c);
    part[blockIdx.x] = make_float2(M, S);
  }
}

// One thread: the row's pieces joined.  lp in fp64; a row of nothing but -inf, or with a NaN or +inf, gives NaN.
template <typename T>
__device__ __forceinline__ double join_row(const Logits& L, const float2* __restrict__ part, int pieces, int64_t row,
                                           int64_t b, int64_t s, int64_t t, float c, double inv_temp,
                                           RowState* st) {
  const float2* p = part + row * pieces;
  float M = p[0].x;
  for (int i = 1; i < pieces; ++i) M = fmaxf(M, p[i].x);
  double S = 0.0;
  for (int i = 0; i < pieces; ++i) S += (double)p[i].y * exp2_((p[i].x - M) * c);
  const double zt = (double)(float)static_cast<const T*>(L.z)[b * L.sb + s * L.ss + t];
  const double l2 = log2(S);
  st->M = M;
  st->l2s = (float)l2;
  return (zt - (double)M) * inv_temp - l2 * 0.69314718055994530942;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
template <int K>  // sums of K values over a 256-thread workgroup, in every thread
__device__ __forceinline__ void block_sums64(double (&v)[K]) {
  __shared__ double red[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = wave_sum64(v[k]);
    if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = red[k][0] + red[k][1] + red[k][2] + red[k][3];
  __syncthreads();
}

// ------------------------------------------------------------------ token log-probabilities
template <typename T>
__global__ void __launch_bounds__(256) logprob_rows_kernel(Logits L, const float2* __restrict__ part, int pieces,
                                                           float c, double inv_temp, float* __restrict__ logp,
                                                           RowState* __restrict__ rows) {
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= L.B * L.S) return;
  const int64_t b = row / L.S, s = row % L.S, t = L.target_of(b, s);
  RowState st{0.f, 0.f, 0.f, 0.f};
  double lp = 0.0;
  if (t >= 0) {
    lp = join_row<T>(L, part, pieces, row, b, s, t, c, inv_temp, &st);
    st.coef = 1.f;
  }
  logp[row] = (float)lp;
  rows[row] = st;
}

// ------------------------------------------------------------------ clipped policy loss
struct PolicyArgs {
  TokenArray old_logp, ref_logp, adv;
  double low, high, kl_coef;  // ratio bounds 1 - clip, 1 + clip_high
};

// One token: the loss term, and its slope by lp.  min(r A, clip(r) A) has slope r A except where the clipped term is the
// smaller one: A > 0 above the upper bound, A < 0 below the lower one.
__device__ __forceinline__ void policy_token(const PolicyArgs& a, int64_t b, int64_t s, double lp, double* loss,
                                             double* slope, double* kl, bool* clipped) {
  const double A = (double)a.adv.at(b, s);
  const double r = exp(lp - (double)a.old_logp.at(b, s));
  *clipped = (A > 0.0 && r > a.high) || (A < 0.0 && r < a.low);
  const double rc = *clipped ? (A > 0.0 ? a.high : a.low) : r;
  *loss = -rc * A;
  *slope = *clipped ? 0.0 : -r * A;
  *kl = 0.0;
  if (a.ref_logp.p) {
    const double d = (double)a.ref_logp.at(b, s) - lp;
    const double e = expm1(d);
    *kl = e - d;
    if (a.kl_coef != 0.0) {
      *loss += a.kl_coef * *kl;
      *slope -= a.kl_coef * e;
    }
  }
}

// Workgroup b * segs + i: kSegRows tokens of sequence b.  seg: [B * segs] sums {loss, kl, clipped, tokens}.
template <typename T>
__global__ void __launch_bounds__(kSegRows) policy_rows_kernel(Logits L, const float2* __restrict__ part, int pieces,
                                                               float c, double inv_temp, PolicyArgs a, int segs,
                                                               float* __restrict__ logp, RowState* __restrict__ rows,
                                                               double4* __restrict__ seg) {
  const int64_t b = blockIdx.x / segs, s = (int64_t)(blockIdx.x % segs) * kSegRows + threadIdx.x;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  if (s < L.S) {
    const int64_t row = b * L.S + s, t = L.target_of(b, s);
    RowState st{0.f, 0.f, 0.f, 0.f};
    double lp = 0.0;
    if (t >= 0) {
      lp = join_row<T>(L, part, pieces, row, b, s, t, c, inv_temp, &st);
      double slope;
      bool clipped;
      policy_token(a, b, s, lp, &v[0], &slope, &v[1], &clipped);
      v[2] = clipped ? 1.0 : 0.0;
      v[3] = 1.0;
      st.coef = (float)slope;
    }
    logp[row] = (float)lp;
    rows[row] = st;
  }
  block_sums64(v);
  if (threadIdx.x == 0) seg[blockIdx.x] = make_double4(v[0], v[1], v[2], v[3]);
}

// stats: {kl, clip fraction}; weight[b]: what a token of sequence b counts in the loss
__global__ void __launch_bounds__(256) policy_total_kernel(const double4* __restrict__ seg, int64_t B, int segs,
                                                           int by_sequence, double scale, float* __restrict__ loss,
                                                           float* __restrict__ stats, float* __restrict__ weight) {
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t b = threadIdx.x; b < B; b += 256) {
    double q[4] = {0.0, 0.0, 0.0, 0.0};
    for (int i = 0; i < segs; ++i) {
      const double4 x = seg[b * segs + i];
      q[0] += x.x;
      q[1] += x.y;
      q[2] += x.z;
      q[3] += x.w;
    }
    if (by_sequence) {
      const double w = 1.0 / ((q[3] > 1.0 ? q[3] : 1.0) * (double)B);
      q[0] *= w;
      weight[b] = (float)(w * scale);
    }
    for (int k = 0; k < 4; ++k) v[k] += q[k];
  }
  block_sums64(v);
  const double w = 1.0 / (v[3] > 1.0 ? v[3] : 1.0);
  if (!by_sequence)
    for (int64_t b = threadIdx.x; b < B; b += 256) weight[b] = (float)(w * scale);
  if (threadIdx.x == 0) {
    *loss = (float)(v[0] * (by_sequence ? scale : w * scale));
    stats[0] = (float)(v[1] * w);
    stats[1] = (float)(v[2] * w);
  }
}

// ------------------------------------------------------------------ paired preference loss
// seg: [B * segs] sums {log-probability, tokens}
template <typename T>
__global__ void __launch_bounds__(kSegRows) pair_rows_kernel(Logits L, const float2* __restrict__ part, int pieces,
                                                             float c, int segs, RowState* __restrict__ rows,
                                                             double2* __restrict__ seg) {
  const int64_t b = blockIdx.x / segs, s = (int64_t)(blockIdx.x % segs) * kSegRows + threadIdx.x;
  double v[2] = {0.0, 0.0};
  if (s < L.S) {
    const int64_t row = b * L.S + s, t = L.target_of(b, s);
    RowState st{0.f, 0.f, 0.f, 0.f};
    if (t >= 0) {
      v[0] = join_row<T>(L, part, pieces, row, b, s, t, c, 1.0, &st);
      v[1] = 1.0;
      st.coef = 1.f;
    }
    rows[row] = st;
  }
  block_sums64(v);
  if (threadIdx.x == 0) seg[blockIdx.x] = make_double2(v[0], v[1]);
}

// Pair p: sequences p (chosen) and p + P (rejected).  softplus(x) = max(x, 0) + log1p(exp(-|x|)).
__global__ void __launch_bounds__(256) pair_total_kernel(const double2* __restrict__ seg, int64_t P, int segs,
                                                         const float* __restrict__ ref, int64_t ref_stride,
                                                         double beta, double smoothing, int average, double scale,
                                                         float* __restrict__ loss, float* __restrict__ logp,
                                                         float* __restrict__ margin, float* __restrict__ weight) {
  double v[1] = {0.0};
  for (int64_t p = threadIdx.x; p < P; p += 256) {
    double gap[2], share[2];
    for (int side = 0; side < 2; ++side) {
      const int64_t b = p + side * P;
      double l = 0.0, n = 0.0;
      for (int i = 0; i < segs; ++i) {
        l += seg[b * segs + i].x;
        n += seg[b * segs + i].y;
      }
      share[side] = average ? 1.0 / (n > 1.0 ? n : 1.0) : 1.0;
      l *= share[side];
      logp[b] = (float)l;
      gap[side] = ref ? l - (double)ref[b * ref_stride] : l;
    }
    const double h = beta * (gap[0] - gap[1]);
    const double tail = log1p(exp(-fabs(h)));
    v[0] += (1.0 - smoothing) * (tail + (h < 0.0 ? -h : 0.0)) + smoothing * (tail + (h > 0.0 ? h : 0.0));
    margin[p] = (float)h;
    const double slope = scale * beta / (double)P * (1.0 / (1.0 + exp(-h)) - (1.0 - smoothing));
    weight[p] = (float)(slope * share[0]);
    weight[p + P] = (float)(-slope * share[1]);
  }
  block_sums64(v);
  if (threadIdx.x == 0) *loss = (float)(scale * v[0] / (double)P);
}

// ------------------------------------------------------------------ gradient of the logits
constexpr int kGradThreads = 256, kGradChunks = 4;
constexpr int kGradSpan = kGradThreads * kGradChunks * 8;  // logits of one workgroup

// k = coef * weight[b] * gout[b, s] / temperature (weight absent: 1; a scalar gout has strides 0)
template <typename T>
__global__ void __launch_bounds__(kGradThreads) logit_grad_kernel(Logits L, float c, const RowState* __restrict__ rows,
                                                                  const float* __restrict__ weight, TokenArray gout,
                                                                  float inv_temp, int spans, T* __restrict__ dz) {
  const int64_t row = blockIdx.x / spans;
  const int64_t begin = (int64_t)(blockIdx.x % spans) * kGradSpan;
  const int64_t b = row / L.S, s0 = row % L.S, t = L.target_of(b, s0);
  T* out = dz + row * L.V;
  if (t < 0) {
    Row8<T> zero;
#pragma unroll
    for (int j = 0; j < 8; ++j) zero.set(j, 0.f);
#pragma unroll
    for (int u = 0; u < kGradChunks; ++u) {
      const int64_t cc = begin + (u * kGradThreads + threadIdx.x) * 8;
      if (cc < L.V) store_chunk(zero, out, cc, L.V);
    }
    return;
  }
  const T* x = static_cast<const T*>(L.z) + b * L.sb + s0 * L.ss;
  Row8<T> r[kGradChunks];
#pragma unroll
  for (int u = 0; u < kGradChunks; ++u) {
    const int64_t cc = begin + (u * kGradThreads + threadIdx.x) * 8;
    if (cc < L.V) load_chunk(r[u], x, cc, L.V);
  }
  const RowState st = rows[row];
  const float k = st.coef * (weight ? weight[b] : 1.f) * gout.at(b, s0) * inv_temp;
#pragma unroll
  for (int u = 0; u < kGradChunks; ++u) {
    const int64_t cc = begin + (u * kGradThreads + threadIdx.x) * 8;
    if (cc < L.V) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = exp2_(fmaf(r[u].get(j) - st.M, c, -st.l2s));
        r[u].set(j, ((cc + j == t ? 1.f : 0.f) - p) * k);
      }
      store_chunk(r[u], out, cc, L.V);
    }
  }
}

// ------------------------------------------------------------------ launchers
struct LseShape {
  int pieces;
  int64_t span;
};

// Pieces of a row: enough workgroups to fill the chip where rows are few, each piece at least one round of loads
static LseShape lse_shape(int64_t N, int64_t V) {
  const int64_t least = kLseThreads * 8;
  int64_t pieces = N > 0 ? 2048 / N : 1;
  pieces = min(pieces, (V + least - 1) / least);
  if (pieces < 1) pieces = 1;
  const int64_t span = ((V + pieces - 1) / pieces + 7) / 8 * 8;
  return {(int)((V + span - 1) / span), span};
}

template <typename T>
static hipError_t lse_partial(const Logits& L, float c, const LseShape& sh, float2* part, hipStream_t st) {
  hipLaunchKernelGGL(lse_partial_kernel<T>, dim3((unsigned)(L.B * L.S * sh.pieces)), dim3(kLseThreads), 0, st, L, c,
                     sh.pieces, sh.span, part);
  return hipGetLastError();
}

static float scale_of(double temperature) { return (float)(1.44269504088896340736 / temperature); }

}  // namespace dta

#include "preference.h"

using namespace dta;

static Logits logits_of(const PrefLogits& l) {
  return {l.z, l.sb, l.ss, l.target, l.tb, l.ts, l.B, l.S, l.V, l.ignore};
}
static TokenArray array_of(const PrefTokens& t) { return {t.p, t.sb, t.ss}; }

#define DTA_BY_TYPE(type, call)                     \
  switch (type) {                                   \
    case 0: { typedef float T; call; } break;       \
    case 1: { typedef bf16 T; call; } break;        \
    case 2: { typedef _Float16 T; call; } break;    \
    default: return hipErrorInvalidValue;           \
  }

// Workgroups of the passes over the logits have to fit a launch
int dta_pref_fits(int64_t N, int64_t V) {
  const int64_t most = (int64_t)1 << 31, spans = (V + kGradSpan - 1) / kGradSpan;
  return N >= 0 && V > 0 && N < most && V < most && N * spans < most;
}
int64_t dta_pref_parts(int64_t N, int64_t V) { return N * lse_shape(N, V).pieces; }
int64_t dta_pref_segs(int64_t S) { return (S + kSegRows - 1) / kSegRows; }

hipError_t dta_pref_logprobs(const PrefLogits& l, int type, double temperature, void* part, float* logp, void* rows,
                             hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  const LseShape sh = lse_shape(N, L.V);
  const float c = scale_of(temperature);
  DTA_BY_TYPE(type, {
    DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (float2*)part, st));
    hipLaunchKernelGGL(logprob_rows_kernel<T>, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st, L, (float2*)part,
                       sh.pieces, c, 1.0 / temperature, logp, (RowState*)rows);
  })
  return hipGetLastError();
}

hipError_t dta_pref_policy(const PrefLogits& l, int type, double temperature, const PrefTokens& old_logp,
                           const PrefTokens& ref_logp, const PrefTokens& adv, double clip, double clip_high,
                           double kl_coef, int by_sequence, double scale, void* part, double* seg, float* loss,
                           float* stats, float* logp, void* rows, float* weight, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const int segs = (int)dta_pref_segs(L.S);
  if (N > 0) {
    const LseShape sh = lse_shape(N, L.V);
    const float c = scale_of(temperature);
    const PolicyArgs a{array_of(old_logp), array_of(ref_logp), array_of(adv), 1.0 - clip, 1.0 + clip_high, kl_coef};
    DTA_BY_TYPE(type, {
      DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (float2*)part, st));
      hipLaunchKernelGGL(policy_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(kSegRows), 0, st, L, (float2*)part,
                         sh.pieces, c, 1.0 / temperature, a, segs, logp, (RowState*)rows, (double4*)seg);
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(256), 0, st, (double4*)seg, L.B, segs, by_sequence, scale, loss,
                     stats, weight);
  return hipGetLastError();
}

hipError_t dta_pref_pairs(const PrefLogits& l, int type, const float* ref, int64_t ref_stride, double beta,
                          double smoothing, int average, double scale, void* part, double* seg, float* loss,
                          float* logp, float* margin, void* rows, float* weight, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const int segs = (int)dta_pref_segs(L.S);
  if (N > 0) {
    const LseShape sh = lse_shape(N, L.V);
    const float c = scale_of(1.0);
    DTA_BY_TYPE(type, {
      DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (float2*)part, st));
      hipLaunchKernelGGL(pair_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(kSegRows), 0, st, L, (float2*)part,
                         sh.pieces, c, segs, (RowState*)rows, (double2*)seg);
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(pair_total_kernel, dim3(1), dim3(256), 0, st, (double2*)seg, L.B / 2, segs, ref, ref_stride, beta,
                     smoothing, average, scale, loss, logp, margin, weight);
  return hipGetLastError();
}

hipError_t dta_pref_grad(const PrefLogits& l, int type, double temperature, const void* rows, const float* weight,
                         const PrefTokens& gout, void* dz, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  const int spans = (int)((L.V + kGradSpan - 1) / kGradSpan);
  DTA_BY_TYPE(type, {
    hipLaunchKernelGGL(logit_grad_kernel<T>, dim3((unsigned)(N * spans)), dim3(kGradThreads), 0, st, L,
                       scale_of(temperature), (const RowState*)rows, weight, array_of(gout),
                       (float)(1.0 / temperature), spans, (T*)dz);
  })
  return hipGetLastError();
}
