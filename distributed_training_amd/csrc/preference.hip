// Losses that train a model on rewards or preferences, from its logits [B, S, V]: token log-probabilities, the
// clipped policy loss with a KL term, and the paired preference loss; forward and backward.
//
//   c = log2(e) / temperature,  M = max_j z_j,  s = sum_j 2^((z_j - M) c)
//   lp = (z_y - M) / temperature - ln s                              log-probability of the token y
//   dz_j = k ([j = y] - 2^((z_j - M) c - log2 s)),  k = dloss/dlp / temperature
//
// Three steps: every row's (M, s) (lse_partial_kernel, one pass over the logits, a long row cut into pieces where there
// are few); the rows' terms and the loss (one thread a row, in the same kernel or after it, then one workgroup); dz
// (logit_grad_kernel, a second read of the logits and a write).  Both passes over the logits wait for memory.  The policy loss of many rows takes
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

// 16 bytes of logits as they lie in memory: neighbouring lanes take neighbouring chunks (two 16-byte halves of 8 fp32
// values a lane leave half-used cache lines between them: the gradient pass ran at 5.1 TB/s)
template <typename T> struct Packed;
template <> struct Packed<bf16> { typedef bf16x8_u V; };
template <> struct Packed<_Float16> { typedef half8_u V; };
template <> struct Packed<float> { typedef f32x4_u V; };
template <typename T>
struct Chunk {
  static constexpr int W = 16 / sizeof(T);
  typedef typename Packed<T>::V V;
  V v;
  __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
  __device__ __forceinline__ void set(int j, float x) { v[j] = (T)x; }
  // opaque to the compiler: a row kept in registers stays as it was loaded, not converted to fp32 (twice the registers)
  __device__ __forceinline__ void keep() {
    typedef int i4 __attribute__((ext_vector_type(4)));
    i4 w = __builtin_bit_cast(i4, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(V, w);
  }
  // at logit c of a row (rows are below 2^28: byte offsets are 32-bit, one register beside the row's scalar base)
  __device__ __forceinline__ void load(const T* x, int c) {
    v = load_nt<V>(reinterpret_cast<const char*>(x) + (unsigned)c * (unsigned)sizeof(T));
  }
  __device__ __forceinline__ void store(T* x, int c) const {
    store_nt<V>(v, reinterpret_cast<char*>(x) + (unsigned)c * (unsigned)sizeof(T));
  }
};
// A row of V is V / W whole chunks and up to W - 1 logits behind them, which the workgroup's first lanes take one each
// (handled in every chunk instead, the one-pass kernel grew past the instruction cache).
template <typename T>
__device__ __forceinline__ int whole(int V) { return V & ~(Chunk<T>::W - 1); }

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

struct Scale {  // c = log2(e) / temperature in two floats, both positive (d = -inf: no inf - inf); of_exp: 2^(d c)
  float hi, lo;
  __device__ __forceinline__ float of(float d) const { return fmaf(d, hi, d * lo); }
  __device__ __forceinline__ float of_exp(float d) const { return exp2_(of(d)); }
};

// The sum of 2^((z - m) c) over a chunk, pair by pair: the largest term (often near the whole sum) meets 2 or 3
// roundings here, not one for each term that follows it
template <typename T>
__device__ __forceinline__ float exp_sum(const Chunk<T>& r, float m, const Scale& c) {
  float e[Chunk<T>::W];
#pragma unroll
  for (int j = 0; j < Chunk<T>::W; ++j) e[j] = c.of_exp(r.get(j) - m);
#pragma unroll
  for (int n = Chunk<T>::W / 2; n > 0; n >>= 1)
#pragma unroll
    for (int j = 0; j < n; ++j) e[j] += e[j + n];
  return e[0];
}

// (m, s) with one more logit (-inf: none)
__device__ __forceinline__ void add_one(float x, const Scale& c, float* m, float* s) {
  const float mn = fmaxf(*m, x), ms = mn == -INFINITY ? 0.f : mn;
  *s = *s * c.of_exp(*m - ms) + c.of_exp(x - ms);
  *m = mn;
}

// [B, S, V] logits (rows of unit inner stride) and the [B, S] per-token arrays that go with them
struct Logits {
  const void* z;
  int64_t sb, ss;  // element strides of a sequence and of a token
  const int64_t* target;
  int64_t tb, ts;
  int64_t B, S, V, ignore;
  // rows are counted in 32 bits (B * S is below 2^31): a 64-bit division is a hundred instructions
  __device__ __forceinline__ int64_t sequence_of(unsigned row) const { return row / (unsigned)S; }
  __device__ __forceinline__ int64_t token_of(unsigned row) const { return row % (unsigned)S; }
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

// What the gradient needs of a row.  coef: dloss/dlp without the sequence's weight; with the weight, the gradient that
// arrives and 1 / temperature it is multiplied in 64 bits and rounded to fp32 once, as the product k.
struct RowState {
  float M, l2s;
  double coef;
};

// A row is one workgroup's, or, where it is short (NT = 64), one wave's: four rows in a workgroup of 256 threads, which
// share nothing and wait for nothing.  A short row in a workgroup of its own left most lanes idle and was bound by the
// rate at which workgroups start.
template <int NT> constexpr int kRows = NT == 64 ? 4 : 1;
template <int NT>
__device__ __forceinline__ int thread_of() { return NT == 64 ? (int)threadIdx.x & 63 : (int)threadIdx.x; }
template <int NT>
__device__ __forceinline__ unsigned group_of() {  // among all groups of NT threads
  return NT == 64 ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
}

constexpr int kLseThreads = 256, kLongThreads = 1024;

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

// A row's threads together
template <int NW>
__device__ __forceinline__ RowSum block_join(float m, float s, const Scale& c) {
  if constexpr (NW == 1) {
    const float wm = wave_max(m);
    const double ws = wave_sum64_last((double)(s * c.of_exp(m - (wm == -INFINITY ? 0.f : wm))));
    return {__shfl(ws, 63, kWave), wm, 0.f};
  }
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
// Log-probability of the token with logit zt from its row's (M, S), in fp64; a row of nothing but -inf, or with a NaN or
// +inf, gives NaN.
__device__ __forceinline__ double row_logprob(float zt, float M, double S, double inv_temp, float* l2s) {
  const double l2 = log2(S);
  *l2s = (float)l2;
  return ((double)zt - (double)M) * inv_temp - l2 * 0.69314718055994530942;
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

// f(b, sums of sequence b's segments) for every sequence, by one workgroup of kTotalThreads: a thread a sequence where they
// have few segments, else a wave or several a sequence
constexpr int kTotalThreads = 1024;
template <int K, typename F>
__device__ __forceinline__ void for_each_sequence(const double* __restrict__ seg, int64_t B, int segs, F f) {
  constexpr int NW = kTotalThreads / 64;
  double q[K];
  if (segs <= 16) {
    for (int64_t b = threadIdx.x; b < B; b += kTotalThreads) {
#pragma unroll
      for (int k = 0; k < K; ++k) q[k] = 0.0;
      for (int i = 0; i < segs; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) q[k] += seg[(b * segs + i) * K + k];
      f(b, q);
    }
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, each = B > 0 && B < NW ? NW / (int)B : 1;
  __shared__ double part[NW][K];
  for (int64_t b = wave / each; b < B; b += NW / each) {  // (each > 1: at most once)
#pragma unroll
    for (int k = 0; k < K; ++k) q[k] = 0.0;
#pragma unroll 8
    for (int i = wave % each * 64 + lane; i < segs; i += each * 64)
#pragma unroll
      for (int k = 0; k < K; ++k) q[k] += seg[(b * segs + i) * K + k];
#pragma unroll
    for (int k = 0; k < K; ++k) q[k] = wave_sum64(q[k]);
    if (lane == 0) {
      if (each == 1) f(b, q);
#pragma unroll
      for (int k = 0; k < K; ++k) part[wave][k] = q[k];
    }
  }
  if (each == 1) return;
  __syncthreads();
  if (threadIdx.x < B) {
#pragma unroll
    for (int k = 0; k < K; ++k) q[k] = 0.0;
    for (int w = 0; w < each; ++w)
#pragma unroll
      for (int k = 0; k < K; ++k) q[k] += part[threadIdx.x * each + w][k];
    f(threadIdx.x, q);
  }
}

// ------------------------------------------------------------------ token log-probabilities
// 256 / lanes rows a workgroup, here and in the other passes over rows; the group's first lane does the row
template <typename T>
__global__ void __launch_bounds__(256) logprob_rows_kernel(Logits L, const RowSum* __restrict__ part, int pieces,
                                                           int lanes, Scale c, double inv_temp,
                                                           float* __restrict__ logp, RowState* __restrict__ rows) {
  const unsigned row = blockIdx.x * (256u / lanes) + threadIdx.x / lanes;
  const bool there = row < L.B * L.S;
  const int64_t b = L.sequence_of(row), s = L.token_of(row), t = there ? L.target_of(b, s) : -1;
  RowState st{0.f, 0.f, 0.0};
  double S, lp = 0.0;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (!there || (threadIdx.x & (lanes - 1))) return;
  if (t >= 0) {
    lp = row_logprob((float)L.row<T>(b, s)[t], st.M, S, inv_temp, &st.l2s);
    st.coef = 1.0;
  }
  logp[row] = (float)lp;
  rows[row] = st;
}

// ------------------------------------------------------------------ clipped policy loss
struct PolicyArgs {
  TokenArray old_logp, ref_logp, adv;
  double low, high, kl_coef;  // ratio bounds 1 - clip, 1 + clip_high
};

// A value that is the same in every lane, in a scalar register
__device__ __forceinline__ float scalar(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
__device__ __forceinline__ double scalar(double x) {
  const int2 h = __builtin_bit_cast(int2, x);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readfirstlane(h.x), __builtin_amdgcn_readfirstlane(h.y)));
}

struct TokenInputs {
  float old_logp, ref_logp, adv;
  bool has_ref;
  TokenInputs() = default;
  __device__ __forceinline__ void to_scalar() {
    old_logp = scalar(old_logp);
    ref_logp = scalar(ref_logp);
    adv = scalar(adv);
  }
  __device__ __forceinline__ TokenInputs(const PolicyArgs& a, int64_t b, int64_t s)
      : old_logp(a.old_logp.at(b, s)), ref_logp(a.ref_logp.p ? a.ref_logp.at(b, s) : 0.f), adv(a.adv.at(b, s)),
        has_ref(a.ref_logp.p != nullptr) {}
};

// One token: the loss term, and its slope by lp.  min(r A, clip(r) A) has slope r A except where the clipped term is the
// smaller one: A > 0 above the upper bound, A < 0 below the lower one.  r = exp(lp - old), q = exp(ref - lp).  The KL term
// q - 1 - d keeps 52 bits below 1, of which a small d leaves few in d^2 / 2: below 2^-7 it is the series' first five terms
// (the next is d^5 / 2520 of the first: 2^-46), and q - 1 is d more than that.
__device__ __forceinline__ void policy_token(const PolicyArgs& a, const TokenInputs& in, double lp, double r, double q,
                                             double* loss, double* slope, double* kl, bool* clipped) {
  const double A = (double)in.adv;
  *clipped = (A > 0.0 && r > a.high) || (A < 0.0 && r < a.low);
  const double rc = *clipped ? (A > 0.0 ? a.high : a.low) : r;
  *loss = -rc * A;
  *slope = *clipped ? 0.0 : -r * A;
  *kl = 0.0;
  if (in.has_ref) {
    const double d = (double)in.ref_logp - lp;
    const bool small = fabs(d) < 0x1p-7;
    *kl = small ? d * d * (1.0 / 2 + d * (1.0 / 6 + d * (1.0 / 24 + d * (1.0 / 120 + d * (1.0 / 720))))) : q - 1.0 - d;
    const double e = small ? d + *kl : q - 1.0;
    if (a.kl_coef != 0.0) {
      *loss += a.kl_coef * *kl;
      *slope -= a.kl_coef * e;
    }
  }
}

// Group row * pieces + i: piece i of the row, [i * span, (i + 1) * span).  U chunks a thread are requested before
// any is used and share one rescaling of the running sum.  Bound by the read: 6.7 TB/s at 8192 x 50304 bf16 (123 us), 6.9
// at 1999 x 128256 fp32 (148 us).
// What follows for rows of one piece is worked out here as well, which spares a launch: their log-probabilities, terms of
// the policy loss (seg: a double4 a row, as policy_rows_kernel's), or terms of the pairs (a double2 a row).
enum Then { kPieces, kLogprobs, kPolicy, kPairs };
template <typename T, int NT, Then THEN>
__global__ void __launch_bounds__(NT * kRows<NT>) lse_partial_kernel(Logits L, Scale c, int pieces, int span,
                                                                  RowSum* __restrict__ part, double inv_temp,
                                                                  PolicyArgs a, float* __restrict__ logp,
                                                                  RowState* __restrict__ rows,
                                                                  void* __restrict__ seg) {
  constexpr bool WHOLE = NT == 64 || THEN != kPieces;
  constexpr int NW = NT / 64, U = 4, W = Chunk<T>::W, STEP = NT * W;
  const unsigned group = group_of<NT>();
  if (NT == 64 && group >= L.B * L.S) return;
  const unsigned row = WHOLE ? group : group / (unsigned)pieces;
  const int64_t b = L.sequence_of(row), s0 = L.token_of(row);
  const int tid = thread_of<NT>(), t = (int)L.target_of(b, s0);
  if (t < 0) {
    if (THEN == kPieces || tid != 0) return;
    if (THEN == kLogprobs || THEN == kPolicy) logp[row] = 0.f;
    rows[row] = RowState{0.f, 0.f, 0.0};
    if (THEN == kPolicy) static_cast<double4*>(seg)[row] = make_double4(0.0, 0.0, 0.0, 0.0);
    if (THEN == kPairs) static_cast<double2*>(seg)[row] = make_double2(0.0, 0.0);
    return;
  }
  const T* x = L.row<T>(b, s0);
  const int V = (int)L.V, begin = WHOLE ? 0 : (int)(group % (unsigned)pieces) * span;
  const int end = WHOLE ? whole<T>(V) : min(begin + span, whole<T>(V));
  const float zt = THEN != kPieces ? (float)x[t] : 0.f;
  TokenInputs in{};
  if (THEN == kPolicy) in = TokenInputs(a, b, s0);
  float m = -INFINITY, s = 0.f;
  for (int c0 = begin + tid * W; c0 < end; c0 += STEP * U) {
    Chunk<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * STEP < end) r[u].load(x, c0 + u * STEP);
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * STEP < end)
#pragma unroll
        for (int j = 0; j < W; ++j) mn = fmaxf(mn, r[u].get(j));
    const float ms = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: the sum stays 0, not NaN
    float e = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * STEP < end) e += exp_sum(r[u], ms, c);
    s = s * c.of_exp(m - ms) + e;
    m = mn;
  }
  if (begin + span >= V && tid < V - whole<T>(V)) add_one((float)x[whole<T>(V) + tid], c, &m, &s);
  const RowSum all = block_join<NW>(m, s, c);
  if (tid != 0) return;
  if (THEN == kPieces) {
    part[group] = all;
    return;
  }
  RowState st{all.M, 0.f, 1.0};
  const double lp = row_logprob(zt, all.M, all.S, inv_temp, &st.l2s);
  if (THEN == kPolicy) {
    double loss, slope, kl;
    bool clipped;
    policy_token(a, in, lp, exp(lp - (double)in.old_logp), in.has_ref ? exp((double)in.ref_logp - lp) : 1.0, &loss, &slope, &kl, &clipped);
    st.coef = slope;
    static_cast<double4*>(seg)[row] = make_double4(loss, kl, clipped ? 1.0 : 0.0, 1.0);
  }
  if (THEN == kPairs) static_cast<double2*>(seg)[row] = make_double2(lp, 1.0);
  if (THEN == kLogprobs || THEN == kPolicy) logp[row] = (float)lp;
  rows[row] = st;
}

// Workgroup b * segs + i: 256 / lanes tokens of sequence b.  seg: [B * segs] sums {loss, kl, clipped, tokens}.
template <typename T>
__global__ void __launch_bounds__(256) policy_rows_kernel(Logits L, const RowSum* __restrict__ part, int pieces,
                                                          int lanes, Scale c, double inv_temp, PolicyArgs a, int segs,
                                                          float* __restrict__ logp, RowState* __restrict__ rows,
                                                          double4* __restrict__ seg) {
  const int64_t b = blockIdx.x / (unsigned)segs;
  const int64_t s = (int64_t)(blockIdx.x % (unsigned)segs) * (256 / lanes) + threadIdx.x / lanes, row = b * L.S + s;
  const int64_t t = s < L.S ? L.target_of(b, s) : -1;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  RowState st{0.f, 0.f, 0.0};
  double S, lp = 0.0;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (s < L.S && (threadIdx.x & (lanes - 1)) == 0) {
    if (t >= 0) {
      lp = row_logprob((float)L.row<T>(b, s)[t], st.M, S, inv_temp, &st.l2s);
      double slope;
      bool clipped;
      const TokenInputs in(a, b, s);
      policy_token(a, in, lp, exp(lp - (double)in.old_logp), in.has_ref ? exp((double)in.ref_logp - lp) : 1.0, &v[0], &slope, &v[1], &clipped);
      v[2] = clipped ? 1.0 : 0.0;
      v[3] = 1.0;
      st.coef = slope;
    }
    logp[row] = (float)lp;
    rows[row] = st;
  }
  block_sums64(v);
  if (threadIdx.x == 0) seg[blockIdx.x] = make_double4(v[0], v[1], v[2], v[3]);
}

// stats: {kl, clip fraction}; weight[b]: what a token of sequence b counts in the loss
__global__ void __launch_bounds__(kTotalThreads) policy_total_kernel(const double* __restrict__ seg, int64_t B, int segs,
                                                           int by_sequence, double scale, float* __restrict__ loss,
                                                           float* __restrict__ stats, double* __restrict__ weight) {
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for_each_sequence<4>(seg, B, segs, [&](int64_t b, double (&q)[4]) {
    if (by_sequence) {
      const double w = 1.0 / ((q[3] > 1.0 ? q[3] : 1.0) * (double)B);
      q[0] *= w;
      weight[b] = w * scale;
    }
    for (int k = 0; k < 4; ++k) v[k] += q[k];
  });
  block_sums64<4, kTotalThreads / 64>(v);
  const double w = 1.0 / (v[3] > 1.0 ? v[3] : 1.0);
  if (!by_sequence)
    for (int64_t b = threadIdx.x; b < B; b += kTotalThreads) weight[b] = w * scale;
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
  const int64_t b = blockIdx.x / (unsigned)segs;
  const int64_t s = (int64_t)(blockIdx.x % (unsigned)segs) * (256 / lanes) + threadIdx.x / lanes, row = b * L.S + s;
  const int64_t t = s < L.S ? L.target_of(b, s) : -1;
  double v[2] = {0.0, 0.0};
  RowState st{0.f, 0.f, 0.0};
  double S;
  join_pieces(part, pieces, lanes, row, t >= 0, c, &st.M, &S);
  if (s < L.S && (threadIdx.x & (lanes - 1)) == 0) {
    if (t >= 0) {
      v[0] = row_logprob((float)L.row<T>(b, s)[t], st.M, S, 1.0, &st.l2s);
      v[1] = 1.0;
      st.coef = 1.0;
    }
    rows[row] = st;
  }
  block_sums64(v);
  if (threadIdx.x == 0) seg[blockIdx.x] = make_double2(v[0], v[1]);
}

// Pair p: sequences p (chosen) and p + P (rejected).  softplus(x) = max(x, 0) + log1p(exp(-|x|)).  total: [2 P] scratch.
__global__ void __launch_bounds__(kTotalThreads) pair_total_kernel(const double* __restrict__ seg, int64_t P, int segs,
                                                         const float* __restrict__ ref, int64_t ref_stride,
                                                         double beta, double smoothing, int average, double scale,
                                                         double2* __restrict__ total, float* __restrict__ loss,
                                                         float* __restrict__ logp, float* __restrict__ margin,
                                                         double* __restrict__ weight) {
  for_each_sequence<2>(seg, 2 * P, segs, [&](int64_t b, double (&q)[2]) {
    const double share = average ? 1.0 / (q[1] > 1.0 ? q[1] : 1.0) : 1.0;
    logp[b] = (float)(q[0] * share);
    total[b] = make_double2(q[0] * share, share);
  });
  __syncthreads();
  double v[1] = {0.0};
  for (int64_t p = threadIdx.x; p < P; p += kTotalThreads) {
    const double2 yes = total[p], no = total[p + P];
    const double r = ref ? (double)ref[p * ref_stride] - (double)ref[(p + P) * ref_stride] : 0.0;
    const double h = beta * (yes.x - no.x - r);
    const double tail = log1p(exp(-fabs(h)));
    v[0] += (1.0 - smoothing) * (tail + (h < 0.0 ? -h : 0.0)) + smoothing * (tail + (h > 0.0 ? h : 0.0));
    margin[p] = (float)h;
    const double slope = scale * beta / (double)P * (1.0 / (1.0 + exp(-h)) - (1.0 - smoothing));
    weight[p] = slope * yes.y;
    weight[p + P] = -slope * no.y;
  }
  block_sums64<1, kTotalThreads / 64>(v);
  if (threadIdx.x == 0) *loss = (float)(scale * v[0] / (double)P);
}

// ------------------------------------------------------------------ gradient of the logits
constexpr int kGradThreads = 256, kGradChunks = 4;
template <typename T, int NT = kGradThreads> constexpr int kGradSpan = NT * kGradChunks * Chunk<T>::W;  // logits of a unit

// -k 2^((z - M) c - log2 s): dz without the k that the target's logit gets on top
__device__ __forceinline__ float grad_of(float z, float M, float l2s, float k, const Scale& c) {
  const float d = z - M;
  return exp2_(fmaf(d, c.hi, fmaf(d, c.lo, -l2s))) * -k;
}
// dz of the whole chunks [begin, begin + CHUNKS * NT * W) of a row that are in registers
template <typename T, int CHUNKS, int NT>
__device__ __forceinline__ void write_grad(Chunk<T> (&r)[CHUNKS], T* out, int begin, int V, float M, float l2s, float k,
                                           const Scale& c) {
  constexpr int W = Chunk<T>::W;
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {
    const int cc = begin + (u * NT + thread_of<NT>()) * W;
    if (cc < whole<T>(V)) {
#pragma unroll
      for (int j = 0; j < W; ++j) r[u].set(j, grad_of(r[u].get(j), M, l2s, k, c));
      r[u].store(out, cc);
    }
    __builtin_amdgcn_sched_barrier(0);  // one chunk's fp32 values at a time: registers
  }
}
// The target's logit once more, with its k: one value a row, where a comparison in every element would be a sixth of the
// pass's arithmetic.  By the lane that wrote its chunk, so that the two stores are in order.
template <typename T, int NT>
__device__ __forceinline__ void write_target(T* out, int V, int t, float zt, float M, float l2s, float k, const Scale& c) {
  const int owner = t < whole<T>(V) ? t / Chunk<T>::W % NT : t - whole<T>(V);
  if (thread_of<NT>() == owner) {
    const float d = zt - M;
    out[t] = (T)((1.f - exp2_(fmaf(d, c.hi, fmaf(d, c.lo, -l2s)))) * k);
  }
}
template <typename T, int CHUNKS, int NT>
__device__ __forceinline__ void write_zeros(T* out, int begin, int V) {
  Chunk<T> zero;
#pragma unroll
  for (int j = 0; j < Chunk<T>::W; ++j) zero.set(j, 0.f);
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {
    const int cc = begin + (u * NT + thread_of<NT>()) * Chunk<T>::W;
    if (cc < whole<T>(V)) zero.store(out, cc);
  }
}

// k = coef * weight[b] * gout[b, s] / temperature (weight absent: 1; a scalar gout has strides 0).  unless_one: dz was
// written in the forward for gout = 1, so nothing is left to do where that is what came.  Bound by the read and the write:
// 6.4 TB/s at 8192 x 50304 bf16 (256 us), 6.2 at 1999 x 128256 fp32 (332 us).  The forward reads with non-temporal loads,
// so that this read finds nothing cached, in whatever order it walks the rows.
template <typename T, int NT>
__global__ void __launch_bounds__(kGradThreads) logit_grad_kernel(Logits L, Scale c, const RowState* __restrict__ rows,
                                                                  const double* __restrict__ weight, TokenArray gout,
                                                                  double inv_temp, int spans, int64_t units,
                                                                  int unless_one, T* __restrict__ dz) {
  if (unless_one && *gout.p == 1.f) return;
  for (int64_t u = group_of<NT>(); u < units; u += gridDim.x * kRows<NT>) {
    const unsigned unit = (unsigned)u, row = unit / (unsigned)spans;  // (units are below 2^31)
    const int64_t b = L.sequence_of(row), s0 = L.token_of(row);
    const int begin = (int)(unit % (unsigned)spans) * kGradSpan<T, NT>, V = (int)L.V, t = (int)L.target_of(b, s0);
    // the lane's logit behind the last whole chunk, where it has one and the span reaches there
    const int last = whole<T>(V) + thread_of<NT>();
    const bool tail = last < V && whole<T>(V) - begin < kGradSpan<T, NT> && whole<T>(V) >= begin;
    T* out = dz + (int64_t)row * L.V;
    if (t < 0) {
      write_zeros<T, kGradChunks, NT>(out, begin, V);
      if (tail) out[last] = (T)0.f;
      continue;
    }
    const T* x = L.row<T>(b, s0);
    Chunk<T> r[kGradChunks];
#pragma unroll
    for (int u = 0; u < kGradChunks; ++u) {
      const int cc = begin + (u * NT + thread_of<NT>()) * Chunk<T>::W;
      if (cc < whole<T>(V)) r[u].load(x, cc);
    }
    const RowState st = rows[row];
    const float k = (float)(st.coef * (weight ? weight[b] : 1.0) * (double)gout.at(b, s0) * inv_temp);
    write_grad<T, kGradChunks, NT>(r, out, begin, V, st.M, st.l2s, k, c);
    if (tail) out[last] = (T)grad_of((float)x[last], st.M, st.l2s, k, c);
    if (t >= begin && t - begin < kGradSpan<T, NT>)
      write_target<T, NT>(out, V, t, (float)x[t], st.M, st.l2s, k, c);
  }
}

// ------------------------------------------------------------------ policy loss and gradient in one pass
// A token's weight in the loss is known before its logits are read: counted first, by one workgroup.
// weight[b] = scale / tokens, or scale / (B * tokens of b); count[0] = tokens
__global__ void __launch_bounds__(1024) policy_weight_kernel(Logits L, int by_sequence, double scale,
                                                             double* __restrict__ weight, double* __restrict__ count) {
  const int lane = threadIdx.x & 63;
  double v[1] = {0.0};  // of this thread
  if (by_sequence && L.B >= 16) {  // a wave a sequence
    for (int64_t b = threadIdx.x >> 6; b < L.B; b += 16) {
      int n = 0;
      for (int64_t s = lane; s < L.S; s += 64) n += L.target_of(b, s) >= 0 ? 1 : 0;
      v[0] += (double)n;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
      if (lane == 0) weight[b] = scale / ((double)(n > 1 ? n : 1) * (double)L.B);
    }
  } else if (by_sequence) {  // all of them a sequence
    for (int64_t b = 0; b < L.B; ++b) {
      double n[1] = {0.0};
      for (int64_t s = threadIdx.x; s < L.S; s += 1024) n[0] += L.target_of(b, s) >= 0 ? 1.0 : 0.0;
      v[0] += n[0];
      block_sums64<1, 16>(n);
      if (threadIdx.x == 0) weight[b] = scale / ((n[0] > 1.0 ? n[0] : 1.0) * (double)L.B);
    }
  } else {
    int n = 0;
    const unsigned N = (unsigned)(L.B * L.S);
    if (L.tb == L.S * L.ts || L.B == 1) {  // one stride over all of them: no division for each
#pragma unroll 8
      for (unsigned i = threadIdx.x; i < N; i += 1024) n += L.target_of(0, i) >= 0 ? 1 : 0;
    } else {
#pragma unroll 8
      for (unsigned i = threadIdx.x; i < N; i += 1024) n += L.target_of(L.sequence_of(i), L.token_of(i)) >= 0 ? 1 : 0;
    }
    v[0] = (double)n;
  }
  block_sums64<1, 16>(v);
  if (!by_sequence)
    for (int64_t b = threadIdx.x; b < L.B; b += 1024) weight[b] = scale / (v[0] > 1.0 ? v[0] : 1.0);
  if (threadIdx.x == 0) *count = v[0];
}

// What a row adds to the loss (times the row's weight), and its KL term (never below 0), whose sign says that the token is
// clipped
struct PolicyTerms {
  double loss, kl;
};

// Running (m, s) of a thread over its chunks of a row
template <typename T, int NT, int N>
__device__ __forceinline__ void add_chunks(Chunk<T> (&r)[N], int V, const Scale& c, float* m, float* s) {
  constexpr int W = Chunk<T>::W, G = 16 / W;  // G chunks share a rescaling
#pragma unroll
  for (int g = 0; g < N; g += G) {
    float mn = *m;
#pragma unroll
    for (int u = g; u < (g + G < N ? g + G : N); ++u)
      if ((u * NT + thread_of<NT>()) * W < whole<T>(V))
#pragma unroll
        for (int j = 0; j < W; ++j) mn = fmaxf(mn, r[u].get(j));
    const float ms = mn == -INFINITY ? 0.f : mn;
    float e = 0.f;
#pragma unroll
    for (int u = g; u < (g + G < N ? g + G : N); ++u)
      if ((u * NT + thread_of<NT>()) * W < whole<T>(V)) e += exp_sum(r[u], ms, c);
    *s = *s * c.of_exp(*m - ms) + e;
    *m = mn;
    __builtin_amdgcn_sched_barrier(0);  // one group's fp32 values at a time: registers
  }
#pragma unroll
  for (int u = 0; u < N; ++u) r[u].keep();
}

// One workgroup a row, the row in registers between its two uses (NT * CHUNKS chunks, at least the row's): one read and
// one write of the logits' size.  It ran at 4.6-5.1 TB/s until less arithmetic
// and fewer registers a row brought 5.5-5.9 of the copy's 6.1 (8192 x 50304 bf16, 3/4 of the rows counting: 260 us); what is
// left is mostly the time that a row's terms keep its workgroup waiting.
template <typename T, int NT, int CHUNKS, int WAVES>  // WAVES a SIMD that the registers leave room for
__global__ void __launch_bounds__(NT * kRows<NT>, WAVES) policy_fused_kernel(Logits L, Scale c, double inv_temp, PolicyArgs a,
                                                                 const double* __restrict__ weight,
                                                                 float* __restrict__ logp, RowState* __restrict__ rows,
                                                                 PolicyTerms* __restrict__ terms, T* __restrict__ dz) {
  const unsigned group = group_of<NT>();
  if (NT == 64 && group >= L.B * L.S) return;
  const int64_t row = group, b = L.sequence_of(group), s0 = L.token_of(group);
  const int tid = thread_of<NT>(), V = (int)L.V, t = (int)L.target_of(b, s0), last = whole<T>(V) + tid;
  T* out = dz + row * L.V;
  if (t < 0) {
    write_zeros<T, CHUNKS, NT>(out, 0, V);
    if (last < V) out[last] = (T)0.f;
    if (tid == 0) {
      logp[row] = 0.f;
      rows[row] = RowState{0.f, 0.f, 0.0};
      terms[row] = {0.0, 0.0};
    }
    return;
  }
  const T* x = L.row<T>(b, s0);
  // what the row's terms need is requested first: thread 0 works on them while all the others wait
  TokenInputs in(a, b, s0);
  float zt = (float)x[t];
  double w = weight[b];
  const float tail = last < V ? (float)x[last] : -INFINITY;
  Chunk<T> r[CHUNKS];
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u) {  // every load in flight before any use
    const int cc = (u * NT + tid) * Chunk<T>::W;
    if (cc < whole<T>(V)) r[u].load(x, cc);
  }
  in.to_scalar();
  zt = scalar(zt);
  w = scalar(w);
  float m = -INFINITY, s = 0.f;
  add_chunks<T, NT>(r, V, c, &m, &s);
  add_one(tail, c, &m, &s);
  const RowSum all = block_join<NT / 64>(m, s, c);
  const float M = scalar(all.M);
  float l2s = 0.f, k = 0.f;
  if (tid < 64) {  // the first wave: the same in all lanes but for the exponential, r in the even ones, q in the odd ones
    const double lp = row_logprob(zt, M, all.S, inv_temp, &l2s);
    const double d = tid & 1 ? (double)in.ref_logp - lp : lp - (double)in.old_logp, e = exp(d);
    double loss, slope, kl;
    bool clipped;
    policy_token(a, in, lp, __shfl(e, 0, kWave), __shfl(e, 1, kWave), &loss, &slope, &kl, &clipped);
    k = (float)(slope * w * inv_temp);
    if (tid == 0) {
      logp[row] = (float)lp;
      rows[row] = RowState{M, l2s, slope};
      terms[row] = {loss * w, copysign(kl, clipped ? -1.0 : 1.0)};
    }
  }
  if constexpr (NT == 64) {  // the wave's first lane has them
    l2s = scalar(l2s);
    k = scalar(k);
  } else {
    __shared__ float pass[2];
    if (tid == 0) {
      pass[0] = l2s;
      pass[1] = k;
    }
    __syncthreads();
    l2s = scalar(pass[0]);
    k = scalar(pass[1]);
  }
  write_grad<T, CHUNKS, NT>(r, out, 0, V, M, l2s, k, c);
  if (last < V) out[last] = (T)grad_of(tail, M, l2s, k, c);
  write_target<T, NT>(out, V, t, zt, M, l2s, k, c);
}

__global__ void __launch_bounds__(1024) policy_sum_kernel(const PolicyTerms* __restrict__ terms, int64_t N,
                                                          const double* __restrict__ count, float* __restrict__ loss,
                                                          float* __restrict__ stats) {
  double v[3] = {0.0, 0.0, 0.0};
#pragma unroll 8
  for (unsigned i = threadIdx.x; i < (unsigned)N; i += 1024) {
    const PolicyTerms x = terms[i];
    v[0] += x.loss;
    v[1] += fabs(x.kl);
    v[2] += signbit(x.kl) ? 1.0 : 0.0;
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

// Pieces of a row, for the few and long rows that are cut at all (in_one_piece): up to 1024 workgroups, each piece at least
// 8192 logits; lanes that join them: the next power of two.  Log-probabilities, bf16, in us with pieces of at least 2048 /
// 8192 / 16384 logits: 1 row of 70001 5.7 / 5.7 / 6.2, 16 of 128256 7.2 / 6.8 / 7.4, 64 of 128256 8.6 / 8.6 / 8.9, 16 of
// 600001 10.7 / 10.7 / 10.3; the policy loss with its gradient, 16 rows of 70001 17.4 / 16.6 / 16.8.
static LseShape lse_shape(int64_t N, int64_t V) {
  const int64_t least = 8192;
  int64_t pieces = N > 0 ? 1024 / N : 1;
  pieces = min(min(pieces, (V + least - 1) / least), (int64_t)kWave);
  if (pieces < 1) pieces = 1;
  const int64_t span = ((V + pieces - 1) / pieces + 7) / 8 * 8;
  pieces = (V + span - 1) / span;
  int lanes = 1;
  while (lanes < pieces) lanes *= 2;
  return {(int)pieces, lanes, (int)span};
}
static int64_t segments(int64_t S, const LseShape& sh) { return (S * sh.lanes + 255) / 256; }

// A wave a row, in the sums and in the gradient: short rows, enough of them.  Sums of rows in us, workgroup / wave a row:
// bf16, 24000 rows of 1003 32.0 / 16.1, of 2000 34.8 / 20.6, of 4000 40.8 / 31.7; 2000 rows of 1003 4.8 / 4.0, of 4000
// 6.1 / 6.0, 500 rows of 1003 3.4 / 3.6, of 4000 3.6 / 4.8; fp32, 24000 rows of 2000 34.2 / 29.6, of 4000 61.0 / 57.7, but
// 4000 of them 9.7 / 11.5.  Gradient, 24000 rows: bf16 of 1003 40.0 / 21.9, of 2000 43.4 / 33.8, fp32 of 1003 42.9 / 35.1.
constexpr int64_t kWaveRows = 2000;
template <typename T>
static bool wave_sums(const Logits& L) { return L.B * L.S >= kWaveRows && L.V <= 2 * kGradSpan<T, 64>; }
template <typename T>
static bool wave_grads(const Logits& L) { return L.B * L.S >= kWaveRows && L.V <= kGradSpan<T, 64>; }

// 1024 threads for a row read in one piece: long rows.  In us, 256 threads / 1024: bf16, 8000 rows of 32000 78 / 86, of 50304
// 121 / 127, of 70000 177 / 166, of 128256 304 / 296; fp32, of 50304 233 / 232, of 70000 341 / 317, of 128256 595 / 584.
// (Of 2^22 rows and more 256 again: a launch takes fewer than 2^32 threads.)
static bool long_rows(const Logits& L) { return L.V > 60000 && L.B * L.S < (1 << 22); }
// Few rows: 1024 threads a row in one launch rather than pieces and a second launch to join them,
// unless the row is too long for that.  Pieces / one, bf16: 64 rows of 16000 5.1 / 4.3 us, of 50304 6.3 / 6.6 (with the
// host 8.8 / 6.7), of 128256 8.6 / 11.5; 16 of 70001 6.3 / 7.9; 1 of 600001 6.9 / 37.5; 128 of 128256 11.6 / 11.6, 255 15.4
// / 13.4.
static bool in_one_piece(int64_t N, int64_t V) { return lse_shape(N, V).pieces == 1 || V <= 65536 || N >= 256; }
// The losses' terms by row, in the rows' own kernel, and added up by one workgroup: few rows, where a launch less counts (a
// pass over pairs of 132 rows of 50257 62 -> 56.5 us, policy of 64 rows of 1003 64 -> 57.7).  With many the sums cost more than
// the launch: pairs of 24000 rows of 1000 28.0 us in two kernels, 23.7 in three.
constexpr int64_t kTermRows = 4096;
static bool terms_by_row(int64_t N, int64_t V) { return in_one_piece(N, V) && N <= kTermRows; }

template <typename T, int NT, Then THEN>
static void launch_lse(const Logits& L, const Scale& c, int pieces, int span, RowSum* part, double inv_temp,
                       const PolicyArgs& a, float* logp, void* rows, void* seg, hipStream_t st) {
  const int64_t groups = L.B * L.S * pieces;
  hipLaunchKernelGGL((lse_partial_kernel<T, NT, THEN>), dim3((unsigned)((groups + kRows<NT> - 1) / kRows<NT>)),
                     dim3(NT * kRows<NT>), 0, st, L, c, pieces, span, part, inv_temp, a, logp, (RowState*)rows, seg);
}

template <typename T>
static hipError_t lse_partial(const Logits& L, const Scale& c, const LseShape& sh, RowSum* part, hipStream_t st) {
  const PolicyArgs a{};
  if (wave_sums<T>(L)) launch_lse<T, 64, kPieces>(L, c, 1, sh.span, part, 0.0, a, nullptr, nullptr, nullptr, st);
  else if (sh.pieces == 1 && long_rows(L))
    launch_lse<T, kLongThreads, kPieces>(L, c, 1, sh.span, part, 0.0, a, nullptr, nullptr, nullptr, st);
  else launch_lse<T, kLseThreads, kPieces>(L, c, sh.pieces, sh.span, part, 0.0, a, nullptr, nullptr, nullptr, st);
  return hipGetLastError();
}

// Rows in one piece with what follows for each
template <typename T, Then THEN>
static hipError_t lse_then(const Logits& L, const Scale& c, const LseShape& sh, double inv_temp, const PolicyArgs& a,
                           float* logp, void* rows, void* seg, hipStream_t st) {
  const int all = (int)L.V;
  if (wave_sums<T>(L)) launch_lse<T, 64, THEN>(L, c, 1, all, nullptr, inv_temp, a, logp, rows, seg, st);
  else if (sh.pieces > 1 || long_rows(L))
    launch_lse<T, kLongThreads, THEN>(L, c, 1, all, nullptr, inv_temp, a, logp, rows, seg, st);
  else launch_lse<T, kLseThreads, THEN>(L, c, 1, all, nullptr, inv_temp, a, logp, rows, seg, st);
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

#define DTA_BY_TYPE(type, ...)                        \
  switch (type) {                                     \
    case 0: { typedef float T; __VA_ARGS__; } break;  \
    case 1: { typedef bf16 T; __VA_ARGS__; } break;   \
    case 2: { typedef _Float16 T; __VA_ARGS__; } break; \
    default: return hipErrorInvalidValue;             \
  }

// A launch takes fewer than 2^32 threads, and the row passes give a row a workgroup of 256 (1024 only to fewer than 2^22
// rows); units are counted in 32 bits
constexpr int64_t kMostGroups = ((int64_t)1 << 24) - 1;
int dta_pref_fits(int64_t N, int64_t V) {
  const int64_t spans = (V + kGradSpan<float> - 1) / kGradSpan<float>;
  return N >= 0 && V > 0 && N <= kMostGroups && V < ((int64_t)1 << 28) && N * spans < ((int64_t)1 << 31);
}
int64_t dta_pref_parts(int64_t N, int64_t V) { return N * lse_shape(N, V).pieces; }
static int segs_of(int64_t B, int64_t S, int64_t V) {
  return (int)(terms_by_row(B * S, V) ? S : segments(S, lse_shape(B * S, V)));
}
int64_t dta_pref_segs(int64_t B, int64_t S, int64_t V) { return B * segs_of(B, S, V); }

hipError_t dta_pref_logprobs(const PrefLogits& l, int type, double temperature, void* part, float* logp, void* rows,
                             hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  const LseShape sh = lse_shape(N, L.V);
  const Scale c = scale_of(temperature);
  DTA_BY_TYPE(type, {
    const double inv = 1.0 / temperature;
    if (in_one_piece(N, L.V)) return lse_then<T, kLogprobs>(L, c, sh, inv, PolicyArgs{}, logp, rows, nullptr, st);
    DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
    hipLaunchKernelGGL(logprob_rows_kernel<T>, dim3((unsigned)((N * sh.lanes + 255) / 256)), dim3(256), 0, st, L,
                       (RowSum*)part, sh.pieces, sh.lanes, c, inv, logp, (RowState*)rows);
  })
  return hipGetLastError();
}

static PolicyArgs policy_args(const PrefPolicy& p) {
  return {array_of(p.old_logp), array_of(p.ref_logp), array_of(p.adv), 1.0 - p.clip, 1.0 + p.clip_high, p.kl_coef};
}

hipError_t dta_pref_policy(const PrefLogits& l, int type, double temperature, const PrefPolicy& p, void* part,
                           double* seg, float* loss, float* stats, float* logp, void* rows, double* weight,
                           hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const LseShape sh = lse_shape(N, L.V);
  const int segs = segs_of(L.B, L.S, L.V);
  if (N > 0) {
    const Scale c = scale_of(temperature);
    DTA_BY_TYPE(type, {
      if (terms_by_row(N, L.V)) {
        DTA_HIP_CHECK((lse_then<T, kPolicy>(L, c, sh, 1.0 / temperature, policy_args(p), logp, rows, seg, st)));
      } else {
        DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
        hipLaunchKernelGGL(policy_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(256), 0, st, L, (RowSum*)part,
                           sh.pieces, sh.lanes, c, 1.0 / temperature, policy_args(p), segs, logp, (RowState*)rows,
                           (double4*)seg);
      }
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(kTotalThreads), 0, st, seg, L.B, segs, p.by_sequence, p.scale,
                     loss, stats, weight);
  return hipGetLastError();
}

// The one-pass form: rows enough to fill half the chip, and a row that fits a workgroup's registers.  bf16, in us, one pass /
// several: 64 rows of 50304 18.2 / 17.8, of 128256 26.7 / 22.4; 128 rows 18.4 / 21.2 and 27.5 / 30.9; 2048 rows 85 / 110
// and 202 / 258.
int dta_pref_policy_fused(int type, int64_t N, int64_t V) {
  return N >= 128 && N < (1 << 22) && V <= (type == 0 ? 65536 : 131072);  // (workgroups of up to 1024 threads)
}

template <typename T, int NT, int CHUNKS, int WAVES>
static void policy_fused(const Logits& L, double temperature, const PrefPolicy& p, const double* weight, float* logp,
                         void* rows, void* terms, void* dz, hipStream_t st) {
  hipLaunchKernelGGL((policy_fused_kernel<T, NT, CHUNKS, WAVES>), dim3((unsigned)((L.B * L.S + kRows<NT> - 1) / kRows<NT>)),
                     dim3(NT * kRows<NT>), 0, st, L,
                     scale_of(temperature), 1.0 / temperature, policy_args(p), weight, logp, (RowState*)rows,
                     (PolicyTerms*)terms, (T*)dz);
}

hipError_t dta_pref_policy_grad(const PrefLogits& l, int type, double temperature, const PrefPolicy& p, void* terms,
                                float* loss, float* stats, float* logp, void* rows, double* weight, void* dz,
                                hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (!dta_pref_policy_fused(type, N, L.V)) return hipErrorInvalidValue;
  double* count = (double*)((PolicyTerms*)terms + N);
  hipLaunchKernelGGL(policy_weight_kernel, dim3(1), dim3(1024), 0, st, L, p.by_sequence, p.scale, weight, count);
  DTA_HIP_CHECK(hipGetLastError());
  // Threads and 16-byte chunks a thread by the row's size: as many rows on a CU as its registers hold, few lanes idle.
  // Each form / the next one, in us of the kernel, bf16 (fp16's layout; fp32 in brackets):
  //   64 x 2   24000 rows of 1021 31.5 / 32.6, 8000 of 500 12.6 / 13.1 (24000 of 509 24.3 / 24.3)
  //   64 x 4   24000 of 2045 42.4 / 60.8, 2000 9.4 / 11.0, 128 7.4 / 6.5 (24000 of 1021 39.4 / 49.5)
  //   256 x 2  24000 of 4093 78.4 / 82.8 (2045: 68.4 / 68.6)
  //   256 x 4  24000 of 4608 82.0 / 118, of 8189 151 / 160 (2304: 73.7 / 97.6; 4093: 136 / 131)
  //   512 x 4  24000 of 9216 159 / 237, of 16381 318 / 349 (4608: 143 / 193)
  //   1024 x 4 24000 of 18432 337 / 342, 512 12.4 / 13.8 (512 of 9216 10.6 / 12.3)
  //   1024 x 7 13481 of 35840 318 / 318, a pass over 8192 of 50304, 3/4 counting, 275 / 279 (14211 of 17000 334 / 345); its 64
  //            registers spill 9, at 4 waves a SIMD without spilling 367 where 8 waves took 279
  //   512 x 16 8278 of 58368 346 / 379, 7373 of 65533 403 / 449 (29184: 349 / 336; 512 of them 22.1 / 27.6)
  //   1024 x 10 7149 of 67584 356 / 375, 5898 of 81917 458 / 469 (33792: 326 / 332)
  //   1024 x 16 the rest; 1024 x 13 in between gained 2.4 % at most (5685 of 84992 364 / 373) and is left out
#define DTA_FUSED(T, NT, CHUNKS, WAVES) \
  policy_fused<T, NT, CHUNKS, WAVES>(L, temperature, p, weight, logp, rows, terms, dz, st)
#define DTA_FUSED_ANY(T, W)                                   \
  if (L.V <= W * 64 * 2) DTA_FUSED(T, 64, 2, 8);              \
  else if (L.V <= W * 64 * 4) DTA_FUSED(T, 64, 4, 8);         \
  else if (L.V <= W * 256 * 2) DTA_FUSED(T, 256, 2, 8);       \
  else if (L.V <= W * 256 * 4) DTA_FUSED(T, 256, 4, 8);       \
  else if (L.V <= W * 512 * 4) DTA_FUSED(T, 512, 4, 8);       \
  else if (L.V <= W * 1024 * 4) DTA_FUSED(T, 1024, 4, 8);     \
  else if (L.V <= W * 1024 * 7) DTA_FUSED(T, 1024, 7, 8);     \
  else if (L.V <= W * 512 * 16) DTA_FUSED(T, 512, 16, 4);     \
  else if (L.V <= W * 1024 * 10) DTA_FUSED(T, 1024, 10, 4);   \
  else DTA_FUSED(T, 1024, 16, 4);
  if (type == 1) {
    DTA_FUSED_ANY(bf16, 8)
  } else if (type == 2) {
    DTA_FUSED_ANY(_Float16, 8)
  } else {
    DTA_FUSED_ANY(float, 4)
  }
#undef DTA_FUSED_ANY
#undef DTA_FUSED
  DTA_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(1024), 0, st, (PolicyTerms*)terms, N, count, loss, stats);
  return hipGetLastError();
}

hipError_t dta_pref_pairs(const PrefLogits& l, int type, const float* ref, int64_t ref_stride, double beta,
                          double smoothing, int average, double scale, void* part, double* seg, float* loss,
                          float* logp, float* margin, void* rows, double* weight, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  const LseShape sh = lse_shape(N, L.V);
  const int segs = segs_of(L.B, L.S, L.V);
  if (N > 0) {
    const Scale c = scale_of(1.0);
    DTA_BY_TYPE(type, {
      if (terms_by_row(N, L.V)) {
        DTA_HIP_CHECK((lse_then<T, kPairs>(L, c, sh, 1.0, PolicyArgs{}, nullptr, rows, seg, st)));
      } else {
        DTA_HIP_CHECK(lse_partial<T>(L, c, sh, (RowSum*)part, st));
        hipLaunchKernelGGL(pair_rows_kernel<T>, dim3((unsigned)(L.B * segs)), dim3(256), 0, st, L, (RowSum*)part,
                           sh.pieces, sh.lanes, c, segs, (RowState*)rows, (double2*)seg);
      }
    })
    DTA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(pair_total_kernel, dim3(1), dim3(kTotalThreads), 0, st, seg, L.B / 2, segs, ref, ref_stride, beta, smoothing,
                     average, scale, (double2*)seg + L.B * segs, loss, logp, margin, weight);
  return hipGetLastError();
}

hipError_t dta_pref_grad(const PrefLogits& l, int type, double temperature, const void* rows, const double* weight,
                         const PrefTokens& gout, int unless_one, void* dz, hipStream_t st) {
  const Logits L = logits_of(l);
  const int64_t N = L.B * L.S;
  if (N == 0) return hipSuccess;
  DTA_BY_TYPE(type, {
    const double inv = 1.0 / temperature;
    // (a launch that is expected to end at once is a small one, whose workgroups walk over the rows if they have to)
    const int64_t most = unless_one ? 2048 : kMostGroups;
    if (wave_grads<T>(L)) {
      hipLaunchKernelGGL((logit_grad_kernel<T, 64>), dim3((unsigned)min((N + 3) / 4, most)), dim3(kGradThreads), 0, st, L,
                         scale_of(temperature), (const RowState*)rows, weight, array_of(gout), inv, 1, N, unless_one,
                         (T*)dz);
    } else {
      const int spans = (int)((L.V + kGradSpan<T> - 1) / kGradSpan<T>);
      hipLaunchKernelGGL((logit_grad_kernel<T, kGradThreads>), dim3((unsigned)min(N * spans, most)), dim3(kGradThreads), 0,
                         st, L, scale_of(temperature), (const RowState*)rows, weight, array_of(gout), inv, spans,
                         N * spans, unless_one, (T*)dz);
    }
  })
  return hipGetLastError();
}
