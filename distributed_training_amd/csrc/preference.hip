// Losses that train a model on rewards or preferences, from its logits [B, S, V]: token log-probabilities, the
// clipped policy loss with a KL term, and the paired preference loss; forward and backward.
//
//   c = log2(e) / temperature,  M = max_j z_j,  s = sum_j 2^((z_j - M) c)
//   lp = (z_y - M) / temperature - ln s                              log-probability of the token y
//   dz_j = k ([j = y] - 2^((z_j - M) c - log2 s)),  k = dloss/dlp / temperature
//
// Three steps: every row's (M, s) (lse_partial_kernel, one pass over the logits, a row cut into pieces where there
// are few); the rows' terms and the loss (one thread a row, then one workgroup); dz (logit_grad_kernel, a second
// read of the logits and a write).  Both passes over the logits wait for memory.  The policy loss of many rows takes
// one pass instead (policy_fused_kernel): all that a row's gradient needs is known once its own sum is.
//
// The row's maximum is subtracted before the multiplication by c, not folded into one fma: rows of the type's lowest
// value then keep their uniform distribution instead of overflowing.  c is held in two floats: its rounding to one
// (up to 6e-8) would shift every log-probability of a sequence the same way, and a preference pair sums hundreds.
// Sums of exponentials are fp32; what follows per row (logarithm, ratio, KL term) and the sums over rows are fp64,
// since 1 - ratio, exp(d) - d - 1 and the difference of two sequences' sums cancel.  It is one thread's work a row.
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

// The logits stream through once a pass: non-temporal accesses leave the caches to others (measured on plain
// copies of 2.1 GB: 6.1 TB/s, 5.65 without; reads 6.9, 6.1 without).
template <typename V>
__device__ __forceinline__ V load_nt(const void* p) { return __builtin_nontemporal_load(static_cast<const V*>(p)); }
template <typename V>
__device__ __forceinline__ void store_nt(V v, void* p) { __builtin_nontemporal_store(v, static_cast<V*>(p)); }
// Opaque to the compiler: a row kept in registers stays as it was loaded, not converted to fp32 (twice the registers)
template <typename V>
__device__ __forceinline__ void keep_as_is(V& v) {
  typedef int i4 __attribute__((ext_vector_type(4)));
  i4 w = __builtin_bit_cast(i4, v);
  asm volatile("" : "+v"(w));
  v = __builtin_bit_cast(V, w);
}

template <typename T> struct Row8;  // 8 logits as they lie in memory
template <> struct Row8<bf16> {
  bf16x8 v;
  __device__ __forceinline__ void load(const bf16* p) { v = load_nt<bf16x8_u>(p); }
  __device__ __forceinline__ float get(int j) const { return bf2f(v[j]); }
  __device__ __forceinline__ void set(int j, float x) { v[j] = f2bf(x); }
  __device__ __forceinline__ void store(bf16* p) const { store_nt<bf16x8_u>(v, p); }
  __device__ __forceinline__ void keep() { keep_as_is(v); }
};
template <> struct Row8<_Float16> {
  half8 v;
  __device__ __forceinline__ void load(const _Float16* p) { v = load_nt<half8_u>(p); }
  __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
  __device__ __forceinline__ void set(int j, float x) { v[j] = (_Float16)x; }
  __device__ __forceinline__ void store(_Float16* p) const { store_nt<half8_u>(v, p); }
  __device__ __forceinline__ void keep() { keep_as_is(v); }
};
template <> struct Row8<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = load_nt<f32x4_u>(p);
    b = load_nt<f32x4_u>(p + 4);
  }
  __device__ __forceinline__ float get(int j) const { return j < 4 ? a[j & 3] : b[j & 3]; }
  __device__ __forceinline__ void set(int j, float x) {
    if (j < 4) a[j & 3] = x;
    else b[j & 3] = x;
  }
  __device__ __forceinline__ void store(float* p) const {
    store_nt<f32x4_u>(a, p);
    store_nt<f32x4_u>(b, p + 4);
  }
  __device__ __forceinline__ void keep() {
    keep_as_is(a);
    keep_as_is(b);
  }
};
// the chunk [c, c + 8) of a row of V: past the end -inf on loads, left alone on stores
template <typename T>
__device__ __forceinline__ void load_chunk(Row8<T>& r, const T* x, int c, int V) {
  if (c <= V - 8) {  // (V is below 2^31 - 2^16: offsets within a row are 32-bit)
    r.load(x + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.set(j, c + j < V ? (float)x[c + j] : -INFINITY);
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(const Row8<T>& r, T* x, int c, int V) {
  if (c <= V - 8) {
    r.store(x + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < V) x[c + j] = (T)r.get(j);
  }
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

struct Scale {  // c = log2(e) / temperature in two floats, both positive (d = -inf: no inf - inf); of_exp: 2^(d c)
  float hi, lo;
  __device__ __forceinline__ float of(float d) const { return fmaf(d, hi, d * lo); }
  __device__ __forceinline__ float of_exp(float d) const { return exp2_(of(d)); }
};

// The sum of 2^((z - m) c) over 8 logits, pair by pair: the largest term (often near the whole sum) meets 3 roundings
// here, not one for each term that follows it
template <typename T>
__device__ __forceinline__ float exp_sum8(const Row8<T>& r, float m, const Scale& c) {
  float e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = c.of_exp(r.get(j) - m);
  return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
}

// [B, S, V] logits (rows of unit inner stride) and the [B, S] per-token arrays that go with them
struct Logits {
  const void* z;
  int64_t sb, ss;  // element strides of a sequence and of a token
  const int64_t* target;
  int64_t tb, ts;
  int64_t B, S, V, ignore;
  template <typename T>
  __device__ __forceinline__ const T* row(int64_t b, int64_t s) const {
    return static_cast<const T*>(z) + b * sb + s * ss;
  }
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

template <int CTRL, int ROWMASK>
__device__ __forceinline__ double dpp_mov64(double v) {  // lanes outside ROWMASK get 0
  const int2 h = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, h.x, CTRL, ROWMASK, 0xf, false),
                                              __builtin_amdgcn_update_dpp(0, h.y, CTRL, ROWMASK, 0xf, false)));
}
// wave_sum (common.h) in 64 bits: the sum in lane 63
__device__ __forceinline__ double wave_sum64_last(double v) {
  v += dpp_mov64<0xB1, 0xf>(v);
  v += dpp_mov64<0x4E, 0xf>(v);
  v += dpp_mov64<0x141, 0xf>(v);
  v += dpp_mov64<0x140, 0xf>(v);
  v += dpp_mov64<0x142, 0xa>(v);
  v += dpp_mov64<0x143, 0xc>(v);
  return v;
}

struct RowSum {  // of a row or a piece of one
  double S;
  float M, pad;
};

// A workgroup's threads together
template <int NW>
__device__ __forceinline__ RowSum block_join(float m, float s, const Scale& c) {
  __shared__ float sm[NW];
  __shared__ double sv[NW];
  const float wm = wave_max(m);
  const double ws = wave_sum64_last((double)(s * c.of_exp(m - (wm == -INFINITY ? 0.f : wm))));
  if ((threadIdx.x & 63) == 63) {
    sm[threadIdx.x >> 6] = wm;
    sv[threadIdx.x >> 6] = ws;
  }
  __syncthreads();
  float M = sm[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) M = fmaxf(M, sm[w]);
  const float Ms = M == -INFINITY ? 0.f : M;
  double S = 0.0;
#pragma unroll
  for (int w = 0; w < NW; ++w) S += sv[w] * (double)c.of_exp(sm[w] - Ms);
  return {S, M, 0.f};
}

// ------------------------------------------------------------------ (M, s) of every row
// Workgroup row * pieces + i: piece i of the row, [i * span, (i + 1) * span).  U chunks a thread are requested before
// any is used and share one rescaling of the running sum.
template <typename T>
__global__ void __launch_bounds__(kLseThreads) lse_partial_kernel(Logits L, Scale c, int pieces, int span,
                                                                  RowSum* __restrict__ part) {
  constexpr int NW = kLseThreads / 64, U = sizeof(T) == 4 ? 2 : 4;
  const int64_t row = blockIdx.x / pieces;
  const int64_t b = row / L.S, s0 = row % L.S;
  if (L.target_of(b, s0) < 0) return;
  const T* x = L.row<T>(b, s0);
  const int begin = (int)(blockIdx.x % pieces) * span, end = (int)min((int64_t)begin + span, L.V);
  float m = -INFINITY, s = 0.f;
  for (int c0 = begin + threadIdx.x * 8; c0 < end; c0 += kLseThreads * 8 * U) {
    Row8<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cc = c0 + u * kLseThreads * 8;
      if (cc < end) load_chunk(r[u], x, cc, end);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * kLseThreads * 8 < end)
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = fmaxf(mn, r[u].get(j));
    const float ms = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: the sum stays 0, not NaN
    float e = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * kLseThreads * 8 < end) e += exp_sum8(r[u], ms, c);
    s = s * c.of_exp(m - ms) + e;
    m = mn;
  }
  const RowSum all = block_join<NW>(m, s, c);
  if (threadIdx.x == 0) part[blockIdx.x] = all;
}

// Log-probability of token t from its row's (M, S), in fp64; a row of nothing but -inf, or with a NaN or +inf, gives NaN.
template <typename T>
__device__ __forceinline__ double row_logprob(const T* x, int64_t t, float M, double S, double inv_temp, float* l2s) {
  const double l2 = log2(S);
  *l2s = (float)l2;
  return ((double)(float)x[t] - (double)M) * inv_temp - l2 * 0.69314718055994530942;
}

// A group of `lanes` (a power of two, at least `pieces`) joins its row's pieces: (M, S) in every lane of the group
__device__ __forceinline__ void join_pieces(const RowSum* __restrict__ part, int pieces, int lanes, int64_t row,
                                            bool live, const Scale& c, float* M, double* S) {
  const int i = threadIdx.x & (lanes - 1);
  RowSum p{0.0, -INFINITY, 0.f};
  if (live && i < pieces) p = part[row * pieces + i];
  float m = p.M;
  for (int off = lanes >> 1; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  double s = live && i < pieces ? p.S * (double)c.of_exp(p.M - m) : 0.0;
  for (int off = lanes >> 1; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
  *M = m;
  *S = s;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
template <int K, int NW = 4>  // sums of K values over a workgroup of NW waves, in every thread
__device__ __forceinline__ void block_sums64(double (&v)[K]) {
  __shared__ double red[K][NW];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = wave_sum64(v[k]);
    if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = red[k][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v[k] += red[k][w];
  }
  __syncthreads();
}

// ------------------------------------------------------------------ token log-probabilities
// 256 / lanes rows a workgroup, here and in the other passes over rows; the group's first lane does the row
template <typename T>
__global__ void __launch_bounds__(256) logprob_rows_kernel(Logits L, const RowSum* __restrict__ part, int pieces,
                                                           int lanes, Scale c, double inv_temp,
                                                           float* __restrict__ logp, RowState* __restrict__ rows) {
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool there = row < L.B * L.S;
  const int64_t b = row / L.S, s = row % L.S, t = there ? L.target_of(b, s) : -1;
  RowState st{0.f, 0.f, 0.f, 0.f};
  double S, lp = 0.0;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (!there || (threadIdx.x & (lanes - 1))) return;
  if (t >= 0) {
    lp = row_logprob(L.row<T>(b, s), t, st.M, S, inv_temp, &st.l2s);
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

// Workgroup b * segs + i: 256 / lanes tokens of sequence b.  seg: [B * segs] sums {loss, kl, clipped, tokens}.
template <typename T>
__global__ void __launch_bounds__(256) policy_rows_kernel(Logits L, const RowSum* __restrict__ part, int pieces,
                                                          int lanes, Scale c, double inv_temp, PolicyArgs a, int segs,
                                                          float* __restrict__ logp, RowState* __restrict__ rows,
                                                          double4* __restrict__ seg) {
  const int64_t b = blockIdx.x / segs;
  const int64_t s = (int64_t)(blockIdx.x % segs) * (256 / lanes) + threadIdx.x / lanes, row = b * L.S + s;
  const int64_t t = s < L.S ? L.target_of(b, s) : -1;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  RowState st{0.f, 0.f, 0.f, 0.f};
  double S, lp = 0.0;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (s < L.S && (threadIdx.x & (lanes - 1)) == 0) {
    if (t >= 0) {
      lp = row_logprob(L.row<T>(b, s), t, st.M, S, inv_temp, &st.l2s);
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
__global__ void __launch_bounds__(256) pair_rows_kernel(Logits L, const RowSum* __restrict__ part, int pieces,
                                                        int lanes, Scale c, int segs, RowState* __restrict__ rows,
                                                        double2* __restrict__ seg) {
  const int64_t b = blockIdx.x / segs;
  const int64_t s = (int64_t)(blockIdx.x % segs) * (256 / lanes) + threadIdx.x / lanes, row = b * L.S + s;
  const int64_t t = s < L.S ? L.target_of(b, s) : -1;
  double v[2] = {0.0, 0.0};
  RowState st{0.f, 0.f, 0.f, 0.f};
  double S;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (s < L.S && (threadIdx.x & (lanes - 1)) == 0) {
    if (t >= 0) {
      v[0] = row_logprob(L.row<T>(b, s), t, st.M, S, 1.0, &st.l2s);
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

// dz of the chunks [begin, begin + CHUNKS * NT * 8) of a row that are in registers
template <typename T, int CHUNKS, int NT>
__device__ __forceinline__ void write_grad(Row8<T> (&r)[CHUNKS], T* out, int begin, int V, int t, float M,
                                           float l2s, float k, const Scale& c) {
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {
    const int cc = begin + (u * NT + (int)threadIdx.x) * 8;
    if (cc < V) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = r[u].get(j) - M, p = exp2_(fmaf(d, c.hi, fmaf(d, c.lo, -l2s)));
        r[u].set(j, ((cc + j == t ? 1.f : 0.f) - p) * k);
      }
      store_chunk(r[u], out, cc, V);
    }
  }
}
template <typename T, int CHUNKS, int NT>
__device__ __forceinline__ void write_zeros(T* out, int begin, int V) {
  Row8<T> zero;
#pragma unroll
  for (int j = 0; j < 8; ++j) zero.set(j, 0.f);
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {
    const int cc = begin + (u * NT + (int)threadIdx.x) * 8;
    if (cc < V) store_chunk(zero, out, cc, V);
  }
}

// k = coef * weight[b] * gout[b, s] / temperature (weight absent: 1; a scalar gout has strides 0).  unless_one: dz was
// written in the forward for gout = 1, so nothing is left to do where that is what came.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) logit_grad_kernel(Logits L, Scale c, const RowState* __restrict__ rows,
                                                                  const float* __restrict__ weight, TokenArray gout,
                                                                  float inv_temp, int spans, int64_t units,
                                                                  int unless_one, T* __restrict__ dz) {
  if (unless_one && *gout.p == 1.f) return;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t row = unit / spans, b = row / L.S, s0 = row % L.S;
    const int begin = (int)(unit % spans) * kGradSpan, V = (int)L.V, t = (int)L.target_of(b, s0);
    T* out = dz + row * L.V;
    if (t < 0) {
      write_zeros<T, kGradChunks, kGradThreads>(out, begin, V);
      continue;
    }
    const T* x = L.row<T>(b, s0);
    Row8<T> r[kGradChunks];
#pragma unroll
    for (int u = 0; u < kGradChunks; ++u) {
      const int cc = begin + (u * kGradThreads + (int)threadIdx.x) * 8;
      if (cc < V) load_chunk(r[u], x, cc, V);
    }
    const RowState st = rows[row];
    const float k = st.coef * (weight ? weight[b] : 1.f) * gout.at(b, s0) * inv_temp;
    write_grad<T, kGradChunks, kGradThreads>(r, out, begin, V, t, st.M, st.l2s, k, c);
  }
}

// ------------------------------------------------------------------ policy loss and gradient in one pass
// A token's weight in the loss is known before its logits are read: counted first, by one workgroup.
// weight[b] = scale / tokens, or scale / (B * tokens of b); count[0] = tokens
__global__ void __launch_bounds__(1024) policy_weight_kernel(Logits L, int by_sequence, double scale,
                                                             float* __restrict__ weight, double* __restrict__ count) {
  __shared__ double red[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int64_t all = 0;  // of this wave
  for (int64_t b = wave; b < L.B; b += 16) {
    int64_t n = 0;
    for (int64_t s = lane; s < L.S; s += 64) n += L.target_of(b, s) >= 0 ? 1 : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
    if (by_sequence && lane == 0) weight[b] = (float)(scale / ((double)(n > 1 ? n : 1) * (double)L.B));
    all += n;
  }
  if (lane == 0) red[wave] = (double)all;
  __syncthreads();
  double n = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) n += red[w];
  if (!by_sequence)
    for (int64_t b = threadIdx.x; b < L.B; b += 1024) weight[b] = (float)(scale / (n > 1.0 ? n : 1.0));
  if (threadIdx.x == 0) *count = n;
}

// One workgroup a row, the row in registers between its two uses (CHUNKS * NT * 8 logits at least V): one read and
// one write of the logits' size.  terms[row]: {weighted loss, kl, clipped}.
template <typename T, int NT, int CHUNKS, int WAVES>  // WAVES a SIMD that the registers have to leave room for
__global__ void __launch_bounds__(NT, WAVES) policy_fused_kernel(Logits L, Scale c, double inv_temp, PolicyArgs a,
                                                          const float* __restrict__ weight, float* __restrict__ logp,
                                                          RowState* __restrict__ rows, double4* __restrict__ terms,
                                                          T* __restrict__ dz) {
  const int64_t row = blockIdx.x, b = row / L.S, s0 = row % L.S;
  const int V = (int)L.V, t = (int)L.target_of(b, s0);
  T* out = dz + row * L.V;
  if (t < 0) {
    write_zeros<T, CHUNKS, NT>(out, 0, V);
    if (threadIdx.x == 0) {
      logp[row] = 0.f;
      rows[row] = RowState{0.f, 0.f, 0.f, 0.f};
      terms[row] = make_double4(0.0, 0.0, 0.0, 0.0);
    }
    return;
  }
  const T* x = L.row<T>(b, s0);
  Row8<T> r[CHUNKS];
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {  // every load in flight before any use
    const int cc = (u * NT + (int)threadIdx.x) * 8;
    if (cc < V) load_chunk(r[u], x, cc, V);
  }
  float m = -INFINITY, s = 0.f;
  constexpr int G = 2;  // chunks that share a rescaling
#pragma unroll
  for (int g = 0; g < CHUNKS; g += G) {
    float mn = m;
#pragma unroll
    for (int u = g; u < (g + G < CHUNKS ? g + G : CHUNKS); ++u)
      if ((u * NT + (int)threadIdx.x) * 8 < V)
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = fmaxf(mn, r[u].get(j));
    const float ms = mn == -INFINITY ? 0.f : mn;
    float e = 0.f;
#pragma unroll
    for (int u = g; u < (g + G < CHUNKS ? g + G : CHUNKS); ++u)
      if ((u * NT + (int)threadIdx.x) * 8 < V) e += exp_sum8(r[u], ms, c);
    s = s * c.of_exp(m - ms) + e;
    m = mn;
  }
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) r[u].keep();
  __shared__ float pass[3];
  const RowSum all = block_join<NT / 64>(m, s, c);
  if (threadIdx.x == 0) {
    RowState st{all.M, 0.f, 0.f, 0.f};
    const double lp = row_logprob(x, t, all.M, all.S, inv_temp, &st.l2s);
    double loss, slope, kl;
    bool clipped;
    policy_token(a, b, s0, lp, &loss, &slope, &kl, &clipped);
    st.coef = (float)slope;
    const float w = weight[b];
    pass[0] = st.M;
    pass[1] = st.l2s;
    pass[2] = st.coef * w * (float)inv_temp;
    logp[row] = (float)lp;
    rows[row] = st;
    terms[row] = make_double4(loss * (double)w, kl, clipped ? 1.0 : 0.0, 0.0);
  }
  __syncthreads();
  write_grad<T, CHUNKS, NT>(r, out, 0, V, t, pass[0], pass[1], pass[2], c);
}

__global__ void __launch_bounds__(1024) policy_sum_kernel(const double4* __restrict__ terms, int64_t N,
                                                          const double* __restrict__ count, float* __restrict__ loss,
                                                          float* __restrict__ stats) {
  double v[3] = {0.0, 0.0, 0.0};
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    const double4 x = terms[i];
    v[0] += x.x;
    v[1] += x.y;
    v[2] += x.z;
  }
  block_sums64<3, 16>(v);
  if (threadIdx.x == 0) {
    const double w = 1.0 / (*count > 1.0 ? *count : 1.0);
    *loss = (float)v[0];
    stats[0] = (float)(v[1] * w);
    stats[1] = (float)(v[2] * w);
  }
}

// ------------------------------------------------------------------ launchers
struct LseShape {
  int pieces, lanes, span;
};

// Pieces of a row: enough workgroups to fill the chip where rows are few, each piece at least one round of loads;
// lanes that join them: the next power of two
static LseShape lse_shape(int64_t N, int64_t V) {
  const int64_t least = kLseThreads * 8;
  int64_t pieces = N > 0 ? 2048 / N : 1;
  pieces = min(min(pieces, (V + least - 1) / least), (int64_t)kWave);
  if (pieces < 1) pieces = 1;
  const int64_t span = ((V + pieces - 1) / pieces + 7) / 8 * 8;
  pieces = (V + span - 1) / span;
  int lanes = 1;
  while (lanes < pieces) lanes *= 2;
  return {(int)pieces, lanes, (int)span};
}
static int64_t segments(int64_t S, const LseShape& sh) { return (S * sh.lanes + 255) / 256; }

template <typename T>
static hipError_t lse_partial(const Logits& L, const Scale& c, const LseShape& sh, RowSum* part, hipStream_t st) {
  hipLaunchKernelGGL(lse_partial_kernel<T>, dim3((unsigned)(L.B * L.S * sh.pieces)), dim3(kLseThreads), 0, st, L, c,
                     sh.pieces, sh.span, part);
  return hipGetLastError();
}

static Scale scale_of(double temperature) {
  const double c = 1.44269504088896340736 / temperature;
  float hi = (float)c;
  if ((double)hi >= c) hi = nextafterf(hi, 0.f);
  return {hi, (float)(c - (double)hi)};
}

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
  return N >= 0 && V > 0 && N < most && V < most - 65536 && N * spans < most;
}
int64_t dta_pref_parts(int64_t N, int64_t V) { return N * lse_shape(N, V).pieces; }
int64_t dta_pref_segs(int64_t B, int64_t S, int64_t V) { return B * segments(S, lse_shape(B * S, V)); }

hipError_t dta_pref_logprobs(const PrefLogits& l, int type, double temperature, void* part, float* logp, void* rows,
                             hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  const LseShape sh = lse_shape(N, L.V);
  const Scale c = scale_of(temperature);
  DTA_BY_TYPE(type, {
    DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
    hipLaunchKernelGGL(logprob_rows_kernel<T>, dim3((unsigned)((N * sh.lanes + 255) / 256)), dim3(256), 0, st, L,
                       (RowSum*)part, sh.pieces, sh.lanes, c, 1.0 / temperature, logp, (RowState*)rows);
  })
  return hipGetLastError();
}

static PolicyArgs policy_args(const PrefPolicy& p) {
  return {array_of(p.old_logp), array_of(p.ref_logp), array_of(p.adv), 1.0 - p.clip, 1.0 + p.clip_high, p.kl_coef};
}

hipError_t dta_pref_policy(const PrefLogits& l, int type, double temperature, const PrefPolicy& p, void* part,
                           double* seg, float* loss, float* stats, float* logp, void* rows, float* weight,
                           hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const LseShape sh = lse_shape(N, L.V);
  const int segs = (int)segments(L.S, sh);
  if (N > 0) {
    const Scale c = scale_of(temperature);
    DTA_BY_TYPE(type, {
      DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
      hipLaunchKernelGGL(policy_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(256), 0, st, L, (RowSum*)part,
                         sh.pieces, sh.lanes, c, 1.0 / temperature, policy_args(p), segs, logp, (RowState*)rows,
                         (double4*)seg);
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(256), 0, st, (double4*)seg, L.B, segs, p.by_sequence, p.scale,
                     loss, stats, weight);
  return hipGetLastError();
}

// The one-pass form: rows enough to fill the chip, and a row that fits a workgroup's registers.
int dta_pref_policy_fused(int type, int64_t N, int64_t V) {
  return N >= 512 && V <= (type == 0 ? 65536 : 131072);
}

template <typename T, int NT, int CHUNKS, int WAVES>
static void policy_fused(const Logits& L, double temperature, const PrefPolicy& p, const float* weight, float* logp,
                         void* rows, double* terms, void* dz, hipStream_t st) {
  hipLaunchKernelGGL((policy_fused_kernel<T, NT, CHUNKS, WAVES>), dim3((unsigned)(L.B * L.S)), dim3(NT), 0, st, L,
                     scale_of(temperature), 1.0 / temperature, policy_args(p), weight, logp, (RowState*)rows,
                     (double4*)terms, (T*)dz);
}

hipError_t dta_pref_policy_grad(const PrefLogits& l, int type, double temperature, const PrefPolicy& p, double* terms,
                                float* loss, float* stats, float* logp, void* rows, float* weight, void* dz,
                                hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (!dta_pref_policy_fused(type, N, L.V)) return hipErrorInvalidValue;
  double* count = terms + 4 * N;
  hipLaunchKernelGGL(policy_weight_kernel, dim3(1), dim3(1024), 0, st, L, p.by_sequence, p.scale, weight, count);
  DTA_HIP_CHECK(hipGetLastError());
#define DTA_FUSED(T, NT, CHUNKS, WAVES) \
  policy_fused<T, NT, CHUNKS, WAVES>(L, temperature, p, weight, logp, rows, terms, dz, st)
#define DTA_FUSED16(T)                                       \
  if (L.V <= 256 * 8 * 4) DTA_FUSED(T, 256, 4, 8);           \
  else if (L.V <= 256 * 8 * 8) DTA_FUSED(T, 256, 8, 5);      \
  else if (L.V <= 512 * 8 * 8) DTA_FUSED(T, 512, 8, 5);      \
  else if (L.V <= 512 * 8 * 13) DTA_FUSED(T, 512, 13, 4);    \
  else if (L.V <= 1024 * 8 * 10) DTA_FUSED(T, 1024, 10, 4);  \
  else DTA_FUSED(T, 1024, 16, 4);
  if (type == 1) {
    DTA_FUSED16(bf16)
  } else if (type == 2) {
    DTA_FUSED16(_Float16)
  } else if (L.V <= 256 * 8 * 4) {
    DTA_FUSED(float, 256, 4, 5);
  } else if (L.V <= 256 * 8 * 12) {
    DTA_FUSED(float, 256, 12, 3);
  } else if (L.V <= 512 * 8 * 13) {
    DTA_FUSED(float, 512, 13, 3);
  } else {
    DTA_FUSED(float, 1024, 8, 4);
  }
#undef DTA_FUSED16
#undef DTA_FUSED
  DTA_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(1024), 0, st, (double4*)terms, N, count, loss, stats);
  return hipGetLastError();
}

hipError_t dta_pref_pairs(const PrefLogits& l, int type, const float* ref, int64_t ref_stride, double beta,
                          double smoothing, int average, double scale, void* part, double* seg, float* loss,
                          float* logp, float* margin, void* rows, float* weight, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const LseShape sh = lse_shape(N, L.V);
  const int segs = (int)segments(L.S, sh);
  if (N > 0) {
    const Scale c = scale_of(1.0);
    DTA_BY_TYPE(type, {
      DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
      hipLaunchKernelGGL(pair_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(256), 0, st, L, (RowSum*)part,
                         sh.pieces, sh.lanes, c, segs, (RowState*)rows, (double2*)seg);
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(pair_total_kernel, dim3(1), dim3(256), 0, st, (double2*)seg, L.B / 2, segs, ref, ref_stride, beta,
                     smoothing, average, scale, loss, logp, margin, weight);
  return hipGetLastError();
}

hipError_t dta_pref_grad(const PrefLogits& l, int type, double temperature, const void* rows, const float* weight,
                         const PrefTokens& gout, int unless_one, void* dz, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  const int spans = (int)((L.V + kGradSpan - 1) / kGradSpan);
  const int64_t units = N * spans;
  // (a launch that is expected to end at once is a small one, whose workgroups walk over the rows if they have to)
  const int64_t grid = unless_one ? min(units, (int64_t)2048) : units;
  DTA_BY_TYPE(type, {
    hipLaunchKernelGGL(logit_grad_kernel<T>, dim3((unsigned)grid), dim3(kGradThreads), 0, st, L, scale_of(temperature),
                       (const RowState*)rows, weight, array_of(gout), (float)(1.0 / temperature), spans, units,
                       unless_one, (T*)dz);
  })
  return hipGetLastError();
}
