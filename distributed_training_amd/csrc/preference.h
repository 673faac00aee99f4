// Launchers of preference.hip, called from bindings_pref.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dta {
struct PrefLogits {  // logits [B, S, V] of unit inner stride, targets [B, S]
  const void* z;
  int64_t sb, ss;
  const int64_t* target;
  int64_t tb, ts;
  int64_t B, S, V, ignore;
};
struct PrefTokens {  // fp32 [B, S], strides in elements (0: broadcast); p null where absent
  const float* p;
  int64_t sb, ss;
};
struct PrefPolicy {
  PrefTokens old_logp, ref_logp, adv;
  double clip, clip_high, kl_coef, scale;
  int by_sequence;
};
}  // namespace dta

// type: 0 f32, 1 bf16, 2 f16.  Scratch and state: part (dta_pref_parts x 16 bytes), seg (dta_pref_segs double4; pairs:
// dta_pref_segs + B double2), terms (16 B S + 8 bytes), rows (16 bytes a row), weight (B doubles).
int dta_pref_fits(int64_t N, int64_t V);
int64_t dta_pref_parts(int64_t N, int64_t V);
int64_t dta_pref_segs(int64_t B, int64_t S, int64_t V);
hipError_t dta_pref_logprobs(const dta::PrefLogits&, int type, double temperature, void* part, float* logp, void* rows,
                             hipStream_t);
hipError_t dta_pref_policy(const dta::PrefLogits&, int type, double temperature, const dta::PrefPolicy&, void* part,
                           double* seg, float* loss, float* stats, float* logp, void* rows, double* weight, hipStream_t);
// the loss with the gradient of the logits for a loss gradient of 1, in one pass; for sizes that dta_pref_policy_fused takes
int dta_pref_policy_fused(int type, int64_t N, int64_t V);
hipError_t dta_pref_policy_grad(const dta::PrefLogits&, int type, double temperature, const dta::PrefPolicy&,
                                void* terms, float* loss, float* stats, float* logp, void* rows, double* weight,
                                void* dz, hipStream_t);
hipError_t dta_pref_pairs(const dta::PrefLogits&, int type, const float* ref, int64_t ref_stride, double beta,
                          double smoothing, int average, double scale, void* part, double* seg, float* loss,
                          float* logp, float* margin, void* rows, double* weight, hipStream_t);
// unless_one: dz holds the gradient for gout = 1 already; rewritten only where the (scalar) gout is another
hipError_t dta_pref_grad(const dta::PrefLogits&, int type, double temperature, const void* rows, const double* weight,
                         const dta::PrefTokens& gout, int unless_one, void* dz, hipStream_t);
