// Python bindings, third translation unit: the preference-training operators (csrc/preference.hip) and the
// gradient norm over many tensors (csrc/grad_norm.hip), registered into the same _C module by dta_register_pref.
//
// Every entry point checks device / dtype / shape / strides on the host before enqueueing, runs on its tensors'
// device whatever the current one is, and takes its scratch from the caching allocator on the stream it uses.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <cmath>
#include <vector>

#include "preference.h"

int64_t dta_grad_sumsq_parts(const int64_t*, int);
hipError_t dta_grad_sumsq(void* const*, const int64_t*, const int*, int, double*, int64_t, double*, float*,
                          hipStream_t);
hipError_t dta_grad_clip(void* const*, const int64_t*, const int*, int, const double*, double, hipStream_t);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<torch::Tensor>;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void ok(hipError_t e, const char* what) { TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e)); }

hipStream_t stream_on(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int float_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kHalf: return 2;
    case torch::kFloat64: return 3;
    default: return -1;
  }
}

// ------------------------------------------------------------------ preference losses
// logits [B, S, V] or [N, V] (one sequence of N tokens), unit inner stride; target int64 of the leading shape
dta::PrefLogits logits_arg(const Tensor& z, const Tensor& target, int64_t ignore, int* type) {
  TORCH_CHECK(z.is_cuda() && target.is_cuda() && z.device() == target.device(),
              "logits and target must be on the same GPU");
  TORCH_CHECK(z.dim() == 2 || z.dim() == 3, "logits must be [N, V] or [B, S, V]");
  TORCH_CHECK(target.dim() == z.dim() - 1 && target.sizes() == z.sizes().slice(0, z.dim() - 1),
              "target must have the logits' shape without the vocabulary");
  TORCH_CHECK_TYPE(target.scalar_type() == torch::kInt64, "target must be int64");
  *type = float_type(z);
  TORCH_CHECK_TYPE(*type >= 0 && *type <= 2, "logits must be float32, bfloat16 or float16");
  const bool flat = z.dim() == 2;
  dta::PrefLogits l{};
  l.V = z.size(-1);
  l.S = z.size(-2);
  l.B = flat ? 1 : z.size(0);
  TORCH_CHECK(l.V >= 1, "logits must have a vocabulary");
  TORCH_CHECK(l.V == 1 || z.stride(-1) == 1, "logits must have unit inner stride");
  TORCH_CHECK(dta_pref_fits(l.B * l.S, l.V), "logits: too many rows for one launch");
  l.z = z.data_ptr();
  l.ss = z.stride(-2);
  l.sb = flat ? 0 : z.stride(0);
  l.target = target.data_ptr<int64_t>();
  l.ts = target.stride(-1);
  l.tb = flat ? 0 : target.stride(0);
  l.ignore = ignore;
  return l;
}

// A per-token fp32 array; per_sequence: [B] stands for each token of its sequence
dta::PrefTokens tokens_arg(const OptTensor& t, const Tensor& target, const char* name, bool per_sequence = false) {
  if (!has(t)) return {nullptr, 0, 0};
  TORCH_CHECK(t->device() == target.device(), name, " must be on the logits' GPU");
  TORCH_CHECK_TYPE(t->scalar_type() == torch::kFloat32, name, " must be float32");
  const bool flat = target.dim() == 1;
  if (per_sequence && !flat && t->dim() == 1) {
    TORCH_CHECK(t->size(0) == target.size(0), name, " must be [B] or [B, S]");
    return {t->data_ptr<float>(), t->stride(0), 0};
  }
  TORCH_CHECK(t->sizes() == target.sizes(), name, per_sequence ? " must be [B] or [B, S]" : " must have target's shape");
  return {t->data_ptr<float>(), flat ? 0 : t->stride(0), t->stride(-1)};
}

void temperature_arg(double t) {
  TORCH_CHECK_VALUE(std::isfinite(t) && t > 0.0, "temperature must be positive and finite");
}

// -> log-probabilities of target's shape, row state
std::vector<Tensor> pref_logprobs(Tensor logits, Tensor target, int64_t ignore_index, double temperature) {
  int type;
  const auto l = logits_arg(logits, target, ignore_index, &type);
  temperature_arg(temperature);
  const at::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const int64_t N = l.B * l.S;
  Tensor logp = torch::empty(target.sizes(), f32), rows = torch::empty({N, 4}, f32);
  Tensor part = torch::empty({dta_pref_parts(N, l.V), 2}, f32);
  ok(dta_pref_logprobs(l, type, temperature, part.data_ptr(), logp.data_ptr<float>(), rows.data_ptr(),
                       stream_on(logits)),
     "token_logprobs");
  return {logp, rows};
}

// -> loss, {kl, clip fraction}, log-probabilities, row state, sequence weights
std::vector<Tensor> pref_policy(Tensor logits, Tensor target, Tensor old_logp, Tensor advantages, OptTensor ref_logp,
                                double clip, double clip_high, double kl_coef, bool by_sequence, int64_t ignore_index,
                                double temperature, double scale) {
  int type;
  const auto l = logits_arg(logits, target, ignore_index, &type);
  temperature_arg(temperature);
  const auto old_a = tokens_arg(old_logp, target, "old_logp"), ref_a = tokens_arg(ref_logp, target, "ref_logp");
  const auto adv_a = tokens_arg(advantages, target, "advantages", true);
  const at::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const int64_t N = l.B * l.S;
  Tensor loss = torch::empty({}, f32), stats = torch::empty({2}, f32);
  Tensor logp = torch::empty(target.sizes(), f32), rows = torch::empty({N, 4}, f32);
  Tensor weight = torch::empty({l.B}, f32), part = torch::empty({dta_pref_parts(N, l.V), 2}, f32);
  Tensor seg = torch::empty({l.B * dta_pref_segs(l.S), 4}, f32.dtype(torch::kFloat64));
  ok(dta_pref_policy(l, type, temperature, old_a, ref_a, adv_a, clip, clip_high, kl_coef, by_sequence, scale,
                     part.data_ptr(), seg.data_ptr<double>(), loss.data_ptr<float>(), stats.data_ptr<float>(),
                     logp.data_ptr<float>(), rows.data_ptr(), weight.data_ptr<float>(), stream_on(logits)),
     "policy_loss");
  return {loss, stats, logp, rows, weight};
}

// -> loss, sequence log-probabilities [B], margins [B / 2], row state, sequence weights
std::vector<Tensor> pref_pairs(Tensor logits, Tensor target, OptTensor ref_logp, double beta, double smoothing,
                               bool average, int64_t ignore_index, double scale) {
  int type;
  TORCH_CHECK(logits.dim() == 3, "logits must be [2 * pairs, S, V]");
  const auto l = logits_arg(logits, target, ignore_index, &type);
  TORCH_CHECK(l.B >= 2 && l.B % 2 == 0, "logits must hold the chosen sequences, then as many rejected ones");
  const float* ref = nullptr;
  int64_t ref_stride = 0;
  if (has(ref_logp)) {
    TORCH_CHECK(ref_logp->device() == logits.device(), "ref_logp must be on the logits' GPU");
    TORCH_CHECK_TYPE(ref_logp->scalar_type() == torch::kFloat32, "ref_logp must be float32");
    TORCH_CHECK(ref_logp->dim() == 1 && ref_logp->size(0) == l.B, "ref_logp must be [2 * pairs]");
    ref = ref_logp->data_ptr<float>();
    ref_stride = ref_logp->stride(0);
  }
  const at::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(torch::kFloat32);
  const int64_t N = l.B * l.S;
  Tensor loss = torch::empty({}, f32), logp = torch::empty({l.B}, f32), margin = torch::empty({l.B / 2}, f32);
  Tensor rows = torch::empty({N, 4}, f32), weight = torch::empty({l.B}, f32);
  Tensor part = torch::empty({dta_pref_parts(N, l.V), 2}, f32);
  Tensor seg = torch::empty({l.B * dta_pref_segs(l.S), 2}, f32.dtype(torch::kFloat64));
  ok(dta_pref_pairs(l, type, ref, ref_stride, beta, smoothing, average, scale, part.data_ptr(), seg.data_ptr<double>(),
                    loss.data_ptr<float>(), logp.data_ptr<float>(), margin.data_ptr<float>(), rows.data_ptr(),
                    weight.data_ptr<float>(), stream_on(logits)),
     "preference_loss");
  return {loss, logp, margin, rows, weight};
}

// gout: a scalar, or one gradient a token (target's shape)
Tensor pref_grad(Tensor logits, Tensor target, Tensor rows, OptTensor weight, Tensor gout, int64_t ignore_index,
                 double temperature) {
  int type;
  const auto l = logits_arg(logits, target, ignore_index, &type);
  temperature_arg(temperature);
  const int64_t N = l.B * l.S;
  TORCH_CHECK(rows.device() == logits.device() && rows.scalar_type() == torch::kFloat32 && rows.is_contiguous() &&
                  rows.numel() == 4 * N,
              "row state: f32 [N, 4]");
  const float* w = nullptr;
  if (has(weight)) {
    TORCH_CHECK(weight->device() == logits.device() && weight->scalar_type() == torch::kFloat32 &&
                    weight->is_contiguous() && weight->numel() == l.B,
                "sequence weights: f32 [B]");
    w = weight->data_ptr<float>();
  }
  dta::PrefTokens g{};
  if (gout.dim() == 0) {
    TORCH_CHECK(gout.device() == logits.device() && gout.scalar_type() == torch::kFloat32, "gradient: f32 scalar");
    g = {gout.data_ptr<float>(), 0, 0};
  } else {
    g = tokens_arg(gout, target, "gradient");
  }
  const at::DeviceGuard guard(logits.device());
  Tensor dz = torch::empty(logits.sizes(), logits.options());
  ok(dta_pref_grad(l, type, temperature, rows.data_ptr(), w, g, dz.data_ptr(), stream_on(logits)), "logits gradient");
  return dz;
}

// ------------------------------------------------------------------ gradient norm
struct GradList {
  std::vector<void*> p;
  std::vector<int64_t> numel;
  std::vector<int> type;
};

GradList grads_arg(const std::vector<Tensor>& ts) {
  GradList g;
  TORCH_CHECK(!ts.empty(), "no tensors");
  g.p.reserve(ts.size());
  g.numel.reserve(ts.size());
  g.type.reserve(ts.size());
  for (const auto& t : ts) {
    TORCH_CHECK(t.is_cuda() && t.device() == ts[0].device(), "gradients must be on one GPU");
    const int type = float_type(t);
    TORCH_CHECK_TYPE(type >= 0, "gradients must be float32, bfloat16, float16 or float64");
    TORCH_CHECK(t.is_non_overlapping_and_dense(), "gradients must be dense in memory");
    g.p.push_back(t.data_ptr());
    g.numel.push_back(t.numel());
    g.type.push_back(type);
  }
  return g;
}

// -> sum of squares (f64 scalar), norm (f32 scalar)
std::vector<Tensor> grad_sumsq(std::vector<Tensor> grads) {
  const GradList g = grads_arg(grads);
  const at::DeviceGuard guard(grads[0].device());
  const int n = (int)grads.size();
  const auto f64 = torch::TensorOptions().device(grads[0].device()).dtype(torch::kFloat64);
  const int64_t parts = dta_grad_sumsq_parts(g.numel.data(), n);
  Tensor part = torch::empty({parts}, f64), sumsq = torch::empty({}, f64);
  Tensor norm = torch::empty({}, f64.dtype(torch::kFloat32));
  ok(dta_grad_sumsq(g.p.data(), g.numel.data(), g.type.data(), n, part.data_ptr<double>(), parts,
                    sumsq.data_ptr<double>(), norm.data_ptr<float>(), stream_on(grads[0])),
     "grad_sumsq");
  return {sumsq, norm};
}

void grad_clip_(std::vector<Tensor> grads, Tensor sumsq, double max_norm) {
  const GradList g = grads_arg(grads);
  TORCH_CHECK(sumsq.device() == grads[0].device() && sumsq.scalar_type() == torch::kFloat64 && sumsq.numel() == 1,
              "sumsq: f64 scalar on the gradients' GPU");
  const at::DeviceGuard guard(grads[0].device());
  ok(dta_grad_clip(g.p.data(), g.numel.data(), g.type.data(), (int)grads.size(), sumsq.data_ptr<double>(), max_norm,
                   stream_on(grads[0])),
     "grad_clip");
}

}  // namespace

void dta_register_pref(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("pref_logprobs", &pref_logprobs, py::arg("logits"), py::arg("target"), py::arg("ignore_index"),
        py::arg("temperature"));
  m.def("pref_policy", &pref_policy, py::arg("logits"), py::arg("target"), py::arg("old_logp"), py::arg("advantages"),
        py::arg("ref_logp"), py::arg("clip"), py::arg("clip_high"), py::arg("kl_coef"), py::arg("by_sequence"),
        py::arg("ignore_index"), py::arg("temperature"), py::arg("scale"));
  m.def("pref_pairs", &pref_pairs, py::arg("logits"), py::arg("target"), py::arg("ref_logp"), py::arg("beta"),
        py::arg("smoothing"), py::arg("average"), py::arg("ignore_index"), py::arg("scale"));
  m.def("pref_grad", &pref_grad, py::arg("logits"), py::arg("target"), py::arg("rows"), py::arg("weight"),
        py::arg("gout"), py::arg("ignore_index"), py::arg("temperature"));
  m.def("grad_sumsq", &grad_sumsq, py::arg("grads"));
  m.def("grad_clip_", &grad_clip_, py::arg("grads"), py::arg("sumsq"), py::arg("max_norm"));
}
