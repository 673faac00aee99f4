// Python bindings, third translation unit: the preference-training operators (csrc/preference.hip) and the
// gradient norm over many tensors (csrc/grad_norm.hip), registered into the same _C module by dta_register_pref.
//
// Every entry point checks device / dtype / shape / strides on the host before enqueueing, runs on its tensors'
// device whatever the current one is, and takes its scratch from the caching allocator on the stream it uses.  The
// losses are autograd functions here rather than in Python: a small batch's pass is all host time.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <cmath>
#include <algorithm>
#include <functional>
#include <vector>

#include "preference.h"

int64_t dta_grad_sumsq_parts(const int64_t*, int);
hipError_t dta_grad_sumsq(void* const*, const int64_t*, const int*, int, double*, int64_t, double*, float*,
                          hipStream_t);
hipError_t dta_grad_clip(void* const*, const int64_t*, const int*, int, const double*, double, hipStream_t);
hipError_t dta_grad_clip_norm(void* const*, const int64_t*, const int*, int, double*, int64_t, double*, float*, double,
                              hipStream_t);
int dta_grad_is_small(const int64_t*, int);
hipError_t dta_grad_clip_small(void* const*, const int64_t*, const int*, int, double, float*, hipStream_t);

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<torch::Tensor>;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void ok(hipError_t e, const char* what) { TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e)); }

hipStream_t stream_on(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// 0 while nothing is being captured on the stream
unsigned long long capture_of(hipStream_t st) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  ok(hipStreamGetCaptureInfo(st, &status, &id), "hipStreamGetCaptureInfo");
  return status == hipStreamCaptureStatusNone ? 0 : id;
}

int float_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kHalf: return 2;
    case torch::kFloat64: return 3;
    default: return -1;
  }
}

// ------------------------------------------------------------------ arguments
// logits [B, S, V] or [N, V] (one sequence of N tokens), unit inner stride; target int64 of the leading shape
dta::PrefLogits logits_arg(const Tensor& z, const Tensor& target, int64_t ignore, int* type) {
  TORCH_CHECK_TYPE(z.defined() && target.defined(), "logits and target must be tensors");
  TORCH_CHECK_VALUE(z.is_cuda(), "logits must be on a GPU (got ", z.device(), ")");
  TORCH_CHECK_VALUE(z.dim() == 2 || z.dim() == 3, "logits must be [N, V] or [B, S, V] (got ", z.sizes(), ")");
  TORCH_CHECK_VALUE(target.sizes() == z.sizes().slice(0, z.dim() - 1), "target must be ",
                    z.sizes().slice(0, z.dim() - 1), " (got ", target.sizes(), ")");
  TORCH_CHECK_VALUE(target.device() == z.device(), "target is on ", target.device(), ", logits on ", z.device());
  TORCH_CHECK_TYPE(target.scalar_type() == torch::kInt64, "target must be int64 (got ", target.scalar_type(), ")");
  *type = float_type(z);
  TORCH_CHECK_TYPE(*type >= 0 && *type <= 2, "GPU logits must be bfloat16, float16 or float32 (got ",
                   z.scalar_type(), ")");
  const bool flat = z.dim() == 2;
  dta::PrefLogits l{};
  l.V = z.size(-1);
  l.S = z.size(-2);
  l.B = flat ? 1 : z.size(0);
  TORCH_CHECK_VALUE(l.V >= 1, "logits must have a vocabulary");
  TORCH_CHECK_VALUE(l.V == 1 || z.stride(-1) == 1, "logits must have unit inner stride");
  TORCH_CHECK_VALUE(dta_pref_fits(l.B * l.S, l.V), "logits: too many rows for one launch");
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
dta::PrefTokens tokens_arg(const Tensor& t, const Tensor& target, const char* name, bool per_sequence = false) {
  TORCH_CHECK_TYPE(t.defined(), name, " must be a tensor");
  const bool flat = target.dim() == 1;
  const bool one_each = per_sequence && !flat && t.dim() == 1 && t.size(0) == target.size(0);
  TORCH_CHECK_VALUE(one_each || t.sizes() == target.sizes(), name, " must be ", target.sizes(),
                    per_sequence && !flat ? " or one a sequence" : "", " (got ", t.sizes(), ")");
  TORCH_CHECK_VALUE(t.device() == target.device(), name, " is on ", t.device(), ", logits on ", target.device());
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kFloat32, name, " must be float32 (got ", t.scalar_type(), ")");
  if (one_each) return {t.data_ptr<float>(), t.stride(0), 0};
  return {t.data_ptr<float>(), flat ? 0 : t.stride(0), t.stride(-1)};
}

Tensor unit_stride(const Tensor& z) {
  return z.defined() && z.dim() >= 2 && z.size(-1) != 1 && z.stride(-1) != 1 ? z.contiguous() : z;
}

// Inputs that carry no gradient, whatever they came from
Tensor fixed(const Tensor& t) { return t.defined() && t.requires_grad() ? t.detach() : t; }
OptTensor fixed(const OptTensor& t) { return has(t) ? OptTensor(fixed(*t)) : t; }

bool wants_grad(const Tensor& z) { return torch::GradMode::is_enabled() && z.requires_grad(); }

// One allocation of scratch and state: sections of `bytes`, each 256-byte aligned
struct Arena {
  int64_t size = 0;
  Tensor t;
  int64_t add(int64_t bytes) {
    const int64_t at = size;
    size += (bytes + 255) / 256 * 256;
    return at;
  }
  void make(const Tensor& like) { t = torch::empty({size > 0 ? size : 1}, like.options().dtype(torch::kUInt8)); }
  char* at(int64_t off) const { return static_cast<char*>(t.data_ptr()) + off; }
};

// ------------------------------------------------------------------ gradient of the logits
// state: [rows: 16 N bytes, rounded up to 256][sequence weights]
int64_t weight_at(int64_t N) { return (16 * N + 255) / 256 * 256; }

void logits_grad(const Tensor& z, const Tensor& target, const Tensor& state, bool weighted, const Tensor& g,
                 int64_t ignore, double temperature, bool unless_one, const Tensor& dz) {
  int type;
  const auto l = logits_arg(z, target, ignore, &type);
  const Tensor gf = g.scalar_type() == torch::kFloat32 ? g : g.to(torch::kFloat32);
  const dta::PrefTokens gout = gf.dim() == 0 ? dta::PrefTokens{gf.data_ptr<float>(), 0, 0}
                                             : tokens_arg(gf, target, "gradient");
  TORCH_CHECK(gf.device() == z.device(), "gradient is on ", gf.device(), ", logits on ", z.device());
  char* s = static_cast<char*>(state.data_ptr());
  ok(dta_pref_grad(l, type, temperature, s, weighted ? reinterpret_cast<double*>(s + weight_at(l.B * l.S)) : nullptr,
                   gout, unless_one, dz.data_ptr(), stream_on(z)),
     "logits gradient");
}

// A backward under create_graph: its gradient stands in the graph behind the logits and the gradient that arrived, so that
// whoever differentiates it again (by way of either) is refused, not handed a result that lacks a term
struct DifferentiatedOnce : torch::autograd::Function<DifferentiatedOnce> {
  static Tensor forward(AutogradContext*, const Tensor& dz, const Tensor&, const Tensor&) { return dz.detach(); }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "the preference losses can be differentiated once: no second derivative through them");
  }
};
Tensor once(const Tensor& dz, const Tensor& z, const Tensor& g) {
  return torch::GradMode::is_enabled() ? DifferentiatedOnce::apply(dz, z, g) : dz;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& target, int64_t ignore,
                        double temperature) {
    int type;
    const auto l = logits_arg(z, target, ignore, &type);
    const at::DeviceGuard guard(z.device());
    const int64_t N = l.B * l.S;
    Arena a;
    const int64_t rows = a.add(16 * N), part = a.add(16 * dta_pref_parts(N, l.V));
    a.make(z);
    Tensor logp = torch::empty(target.sizes(), z.options().dtype(torch::kFloat32));
    ok(dta_pref_logprobs(l, type, temperature, a.at(part), logp.data_ptr<float>(), a.at(rows), stream_on(z)),
       "token_logprobs");
    ctx->save_for_backward({z, target, a.t});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["temperature"] = temperature;
    return logp;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &target = saved[1];
    const at::DeviceGuard guard(z.device());
    Tensor dz = torch::empty(z.sizes(), z.options());
    logits_grad(z, target, saved[2], false, grads[0], ctx->saved_data["ignore"].toInt(),
                ctx->saved_data["temperature"].toDouble(), false, dz);
    return {once(dz, z, grads[0]), Tensor(), Tensor(), Tensor()};
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& target, const Tensor& old_logp,
                               const Tensor& advantages, const OptTensor& ref_logp, double clip, double clip_high,
                               double kl_coef, bool by_sequence, int64_t ignore, double temperature, double scale,
                               bool grad) {
    int type;
    const auto l = logits_arg(z, target, ignore, &type);
    dta::PrefPolicy p{};
    p.old_logp = tokens_arg(old_logp, target, "old_logp");
    if (has(ref_logp)) p.ref_logp = tokens_arg(*ref_logp, target, "ref_logp");
    p.adv = tokens_arg(advantages, target, "advantages", true);
    p.clip = clip;
    p.clip_high = clip_high;
    p.kl_coef = kl_coef;
    p.scale = scale;
    p.by_sequence = by_sequence;
    const at::DeviceGuard guard(z.device());
    const hipStream_t st = stream_on(z);
    const int64_t N = l.B * l.S;
    const bool fused = grad && dta_pref_policy_fused(type, N, l.V);
    Arena a;
    const int64_t rows = a.add(16 * N), weight = a.add(8 * l.B);
    const int64_t part = a.add(fused ? 16 * N + 8 : 16 * dta_pref_parts(N, l.V));
    const int64_t seg = a.add(fused ? 0 : 32 * dta_pref_segs(l.B, l.S, l.V));
    a.make(z);
    const auto f32 = z.options().dtype(torch::kFloat32);
    Tensor loss = torch::empty({}, f32), stats = torch::empty({2}, f32), logp = torch::empty(target.sizes(), f32);
    if (fused) {
      Tensor dz = torch::empty(z.sizes(), z.options());
      ok(dta_pref_policy_grad(l, type, temperature, p, a.at(part), loss.data_ptr<float>(),
                              stats.data_ptr<float>(), logp.data_ptr<float>(), a.at(rows),
                              reinterpret_cast<double*>(a.at(weight)), dz.data_ptr(), st),
         "policy_loss");
      ctx->saved_data["dz"] = dz;
      ctx->saved_data["capture"] = (int64_t)capture_of(st);
    } else {
      ok(dta_pref_policy(l, type, temperature, p, a.at(part), reinterpret_cast<double*>(a.at(seg)),
                         loss.data_ptr<float>(), stats.data_ptr<float>(), logp.data_ptr<float>(), a.at(rows),
                         reinterpret_cast<double*>(a.at(weight)), st),
         "policy_loss");
    }
    ctx->save_for_backward({z, target, a.t});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    Tensor kl = stats[0], clipped = stats[1];
    ctx->mark_non_differentiable({logp, kl, clipped});
    return {loss, logp, kl, clipped};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list none(13);
    if (!grads[0].defined()) return none;
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &target = saved[1];
    const at::DeviceGuard guard(z.device());
    // The gradient that the forward wrote for a loss gradient of 1 goes to the first backward, which rewrites it where
    // another came; a second backward over a retained graph writes its own.  So does one that is captured into a graph
    // without its forward: a replay would find what its caller has made of the buffer since.
    Tensor dz;
    auto& data = ctx->saved_data;
    const auto it = data.find("dz");
    if (it != data.end()) {
      if (data["capture"].toInt() == (int64_t)capture_of(stream_on(z))) dz = it->second.toTensor();
      data.erase("dz");
    }
    const bool written = dz.defined();
    if (!written) dz = torch::empty(z.sizes(), z.options());
    logits_grad(z, target, saved[2], true, grads[0], data["ignore"].toInt(), data["temperature"].toDouble(), written,
                dz);
    none[0] = once(dz, z, grads[0]);
    return none;
  }
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& target, const OptTensor& ref_logp,
                               double beta, double smoothing, bool average, int64_t ignore, double scale) {
    int type;
    const auto l = logits_arg(z, target, ignore, &type);
    TORCH_CHECK_VALUE(z.dim() == 3 && l.B >= 2 && l.B % 2 == 0,
                      "logits must be [2 P, S, V]: P chosen sequences, then as many rejected ones (got ", z.sizes(),
                      ")");
    const float* ref = nullptr;
    int64_t ref_stride = 0;
    if (has(ref_logp)) {
      TORCH_CHECK_VALUE(ref_logp->dim() == 1 && ref_logp->size(0) == l.B, "ref_logp must be [", l.B, "] (got ",
                        ref_logp->sizes(), ")");
      TORCH_CHECK_VALUE(ref_logp->device() == z.device(), "ref_logp is on ", ref_logp->device(), ", logits on ",
                        z.device());
      TORCH_CHECK_TYPE(ref_logp->scalar_type() == torch::kFloat32, "ref_logp must be float32 (got ",
                       ref_logp->scalar_type(), ")");
      ref = ref_logp->data_ptr<float>();
      ref_stride = ref_logp->stride(0);
    }
    const at::DeviceGuard guard(z.device());
    const int64_t N = l.B * l.S;
    Arena a;
    const int64_t rows = a.add(16 * N), weight = a.add(8 * l.B), part = a.add(16 * dta_pref_parts(N, l.V));
    const int64_t seg = a.add(16 * (dta_pref_segs(l.B, l.S, l.V) + l.B));
    a.make(z);
    const auto f32 = z.options().dtype(torch::kFloat32);
    Tensor loss = torch::empty({}, f32), logp = torch::empty({l.B}, f32), margin = torch::empty({l.B / 2}, f32);
    ok(dta_pref_pairs(l, type, ref, ref_stride, beta, smoothing, average, scale, a.at(part),
                      reinterpret_cast<double*>(a.at(seg)), loss.data_ptr<float>(), logp.data_ptr<float>(),
                      margin.data_ptr<float>(), a.at(rows), reinterpret_cast<double*>(a.at(weight)), stream_on(z)),
       "preference_loss");
    ctx->save_for_backward({z, target, a.t});
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({logp, margin});
    return {loss, logp, margin};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list none(8);
    if (!grads[0].defined()) return none;
    const auto saved = ctx->get_saved_variables();
    const at::DeviceGuard guard(saved[0].device());
    Tensor dz = torch::empty(saved[0].sizes(), saved[0].options());
    logits_grad(saved[0], saved[1], saved[2], true, grads[0], ctx->saved_data["ignore"].toInt(), 1.0, false, dz);
    none[0] = once(dz, saved[0], grads[0]);
    return none;
  }
};

Tensor token_logprobs(const Tensor& logits, const Tensor& target, int64_t ignore_index, double temperature) {
  return TokenLogprobs::apply(unit_stride(logits), target, ignore_index, temperature);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& target,
                                                       const Tensor& old_logp, const Tensor& advantages,
                                                       const OptTensor& ref_logp, double clip, double clip_high,
                                                       double kl_coef, bool by_sequence, int64_t ignore_index,
                                                       double temperature, double scale) {
  const Tensor z = unit_stride(logits);
  const auto r = PolicyLoss::apply(z, target, fixed(old_logp), fixed(advantages), fixed(ref_logp), clip, clip_high, kl_coef, by_sequence,
                                   ignore_index, temperature, scale, z.defined() && wants_grad(z));
  return {r[0], r[1], r[2], r[3]};
}

std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& target,
                                                   const OptTensor& ref_logp, double beta, double smoothing,
                                                   bool average, int64_t ignore_index, double scale) {
  const auto r = PreferenceLoss::apply(unit_stride(logits), target, fixed(ref_logp), beta, smoothing, average, ignore_index,
                                       scale);
  return {r[0], r[1], r[2]};
}

// ------------------------------------------------------------------ gradient norm
struct GradList {
  std::vector<void*> p;
  std::vector<int64_t> numel;
  std::vector<int> type;
  void add(const Tensor& t, int type_) {
    p.push_back(t.data_ptr());
    numel.push_back(t.numel());
    type.push_back(type_);
  }
  int64_t bytes(size_t i) const { return numel[i] * (type[i] == 0 ? 4 : type[i] == 3 ? 8 : 2); }
  // Memory that is listed twice is kept once (two parameters may share a gradient): scaled twice it would depend on
  // which workgroup comes first.  Gradients that share a part are refused for the same reason.
  void drop_repeats() {
    std::vector<size_t> order;
    for (size_t i = 0; i < p.size(); ++i)
      if (numel[i] > 0) order.push_back(i);
    std::sort(order.begin(), order.end(), [&](size_t a, size_t b) { return std::less<void*>()(p[a], p[b]); });
    bool any = false;
    for (size_t k = 1, last = 0; k < order.size(); ++k) {
      const size_t i = order[k], j = order[last];
      if (p[i] == p[j] && numel[i] == numel[j] && type[i] == type[j]) {
        numel[i] = 0;
        any = true;
        continue;
      }
      TORCH_CHECK_VALUE(static_cast<char*>(p[j]) + bytes(j) <= static_cast<char*>(p[i]),
                        "gradients overlap in memory without being the same");
      last = k;
    }
    if (!any) return;
    size_t n = 0;
    for (size_t i = 0; i < p.size(); ++i) {
      if (numel[i] == 0) continue;
      p[n] = p[i];
      numel[n] = numel[i];
      type[n++] = type[i];
    }
    p.resize(n);
    numel.resize(n);
    type.resize(n);
  }
};

GradList grads_arg(const std::vector<Tensor>& ts) {
  GradList g;
  TORCH_CHECK(!ts.empty(), "no tensors");
  for (const auto& t : ts) {
    TORCH_CHECK(t.is_cuda() && t.device() == ts[0].device(), "gradients must be on one GPU");
    const int type = float_type(t);
    TORCH_CHECK_TYPE(type >= 0, "gradients must be float32, bfloat16, float16 or float64");
    TORCH_CHECK(t.is_non_overlapping_and_dense(), "gradients must be dense in memory");
    g.add(t, type);
  }
  return g;
}

// -> sum of squares (f64 scalar), norm (f32 scalar)
std::tuple<Tensor, Tensor> sumsq_of(const GradList& g, c10::Device device, hipStream_t st) {
  const auto f64 = torch::TensorOptions().device(device).dtype(torch::kFloat64);
  const int n = (int)g.p.size();
  const int64_t parts = dta_grad_sumsq_parts(g.numel.data(), n);
  Tensor part = torch::empty({parts}, f64), sumsq = torch::empty({}, f64);
  Tensor norm = torch::empty({}, f64.dtype(torch::kFloat32));
  ok(dta_grad_sumsq(g.p.data(), g.numel.data(), g.type.data(), n, part.data_ptr<double>(), parts,
                    sumsq.data_ptr<double>(), norm.data_ptr<float>(), st),
     "grad_sumsq");
  return {sumsq, norm};
}

std::tuple<Tensor, Tensor> grad_sumsq(const std::vector<Tensor>& grads) {
  const GradList g = grads_arg(grads);
  const at::DeviceGuard guard(grads[0].device());
  return sumsq_of(g, grads[0].device(), stream_on(grads[0]));
}

void grad_clip_(const std::vector<Tensor>& grads, const Tensor& sumsq, double max_norm) {
  GradList g = grads_arg(grads);
  g.drop_repeats();
  TORCH_CHECK(sumsq.device() == grads[0].device() && sumsq.scalar_type() == torch::kFloat64 && sumsq.numel() == 1,
              "sumsq: f64 scalar on the gradients' GPU");
  const at::DeviceGuard guard(grads[0].device());
  for (const auto& t : grads) t.unsafeGetTensorImpl()->bump_version();  // (refuses inference tensors)
  ok(dta_grad_clip(g.p.data(), g.numel.data(), g.type.data(), (int)g.p.size(), sumsq.data_ptr<double>(), max_norm,
                   stream_on(grads[0])),
     "grad_clip");
}

// Norm and clip of gradients on one device: the norm (f32 scalar)
Tensor clip_all(const GradList& g, c10::Device device, double max_norm) {
  const at::DeviceGuard guard(device);
  const hipStream_t st = c10::hip::getCurrentHIPStream(device.index()).stream();
  const int n = (int)g.p.size();
  Tensor norm = torch::empty({}, torch::TensorOptions().device(device).dtype(torch::kFloat32));
  if (dta_grad_is_small(g.numel.data(), n)) {
    ok(dta_grad_clip_small(g.p.data(), g.numel.data(), g.type.data(), n, max_norm, norm.data_ptr<float>(), st),
       "grad_clip");
    return norm;
  }
  const int64_t parts = dta_grad_sumsq_parts(g.numel.data(), n);
  Tensor part = torch::empty({parts + 1}, norm.options().dtype(torch::kFloat64));
  double* scratch = part.data_ptr<double>();
  ok(dta_grad_clip_norm(g.p.data(), g.numel.data(), g.type.data(), n, scratch + 1, parts, scratch,
                        norm.data_ptr<float>(), max_norm, st),
     "grad_clip");
  return norm;
}

Tensor clip_grads_(const std::vector<Tensor>& grads, double max_norm) {
  GradList g = grads_arg(grads);
  g.drop_repeats();
  for (const auto& t : grads) t.unsafeGetTensorImpl()->bump_version();  // (refuses inference tensors)
  return clip_all(g, grads[0].device(), max_norm);
}

// The whole of clip_grad_norm_ for parameters whose gradients all lie dense on one GPU: the norm, or None where they
// do not (ops/optim.py then takes them one device and one layout at a time).
OptTensor clip_params_(const std::vector<Tensor>& params, double max_norm) {
  GradList g;
  std::vector<Tensor> grads;
  for (const auto& p : params) {
    const Tensor& t = p.grad();
    if (!t.defined()) continue;
    if (t.layout() != torch::kStrided || !t.is_cuda() || (!grads.empty() && t.device() != grads[0].device()) ||
        float_type(t) < 0 || !t.is_non_overlapping_and_dense())
      return c10::nullopt;
    g.add(t, float_type(t));
    grads.push_back(t);
  }
  if (grads.empty()) return c10::nullopt;
  g.drop_repeats();  // a parameter listed twice, or a gradient that two share, counts and is clipped once
  for (const auto& t : grads) t.unsafeGetTensorImpl()->bump_version();  // (refuses inference tensors)
  return clip_all(g, grads[0].device(), max_norm);
}

}  // namespace

void dta_register_pref(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("target"), py::arg("ignore_index"),
        py::arg("temperature"));
  m.def("policy_loss", &policy_loss, py::arg("logits"), py::arg("target"), py::arg("old_logp"), py::arg("advantages"),
        py::arg("ref_logp"), py::arg("clip"), py::arg("clip_high"), py::arg("kl_coef"), py::arg("by_sequence"),
        py::arg("ignore_index"), py::arg("temperature"), py::arg("scale"));
  m.def("preference_loss", &preference_loss, py::arg("logits"), py::arg("target"), py::arg("ref_logp"),
        py::arg("beta"), py::arg("smoothing"), py::arg("average"), py::arg("ignore_index"), py::arg("scale"));
  m.def("grad_sumsq", &grad_sumsq, py::arg("grads"));
  m.def("grad_clip_", &grad_clip_, py::arg("grads"), py::arg("sumsq"), py::arg("max_norm"));
  m.def("clip_grads_", &clip_grads_, py::arg("grads"), py::arg("max_norm"));
  m.def("clip_params_", &clip_params_, py::arg("params"), py::arg("max_norm"));
}
