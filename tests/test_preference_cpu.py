"""ops/preference.py and the gradient-norm functions of ops/optim.py on CPU tensors: the plain math against 64-bit
forms and against differences, the refusals, and torch's own clip."""
import math

import pytest
import torch

from distributed_training_amd.ops import optim, preference
from tests import preference_oracle as oracle


def _inputs(B=4, S=5, V=11, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, S, V, generator=g, dtype=torch.float64) * 2
    target = torch.randint(V, (B, S), generator=g)
    target[0, :2] = -100
    target[1] = -100  # a sequence without tokens
    lp, _ = oracle.logprobs64(z, target)
    old = lp + 0.3 * torch.randn(B, S, generator=g, dtype=torch.float64)
    ref = lp + 0.3 * torch.randn(B, S, generator=g, dtype=torch.float64)
    adv = torch.randn(B, S, generator=g, dtype=torch.float64)
    return z.to(dtype), target, old, ref, adv


def _against_differences(f, z, points=12, step=1e-5):
    z = z.clone().requires_grad_()
    (grad,) = torch.autograd.grad(f(z), z)
    flat = z.detach().reshape(-1)
    for i in torch.linspace(0, flat.numel() - 1, points).long().tolist():
        hi, lo = flat.clone(), flat.clone()
        hi[i] += step
        lo[i] -= step
        with torch.no_grad():
            d = (f(hi.view_as(z)) - f(lo.view_as(z))) / (2 * step)
        # central difference: step^2 / 6 times a third derivative of order 1, plus 2^-52 |f| / step
        assert abs(float(d) - float(grad.reshape(-1)[i])) < 1e-8 + 1e-6 * abs(float(d))


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs(temperature):
    z, target, *_ = _inputs()
    lp = preference.token_logprobs(z, target, temperature=temperature)
    want, _ = oracle.logprobs64(z, target, temperature=temperature)
    torch.testing.assert_close(lp, want, rtol=1e-12, atol=1e-12)
    w = torch.randn(target.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    _against_differences(lambda x: (preference.token_logprobs(x, target, temperature=temperature) * w).sum(), z)
    lp32 = preference.token_logprobs(z.float(), target, temperature=temperature)
    assert lp32.dtype == torch.float32


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kl,high,per_sequence", [(0.0, None, True), (0.1, 0.28, False)])
def test_policy_loss(reduction, kl, high, per_sequence):
    z, target, old, ref, adv = _inputs()
    adv = adv[:, 0] if per_sequence else adv
    kw = dict(clip_high=high, kl_coef=kl, reduction=reduction, scale=0.5)
    out = preference.policy_loss(z, target, old, adv, ref, **kw)
    loss, lp, mean_kl, clipped = oracle.policy64(z, target, old, adv, ref, **kw)
    assert 0 < float(clipped) < 1  # both sides of the clip occur
    for got, want in ((out.loss, loss), (out.logp, lp), (out.kl, mean_kl), (out.clip_fraction, clipped)):
        torch.testing.assert_close(got, want.to(got.dtype), rtol=1e-10, atol=1e-12)
    _against_differences(lambda x: preference.policy_loss(x, target, old, adv, ref, **kw).loss, z)


@pytest.mark.parametrize("smoothing,average,use_ref", [(0.0, False, True), (0.2, True, False), (0.5, False, False)])
def test_preference_loss(smoothing, average, use_ref):
    z, target, *_ = _inputs()
    ref = torch.linspace(-9, -4, 4, dtype=torch.float64) if use_ref else None
    kw = dict(beta=0.3, label_smoothing=smoothing, average=average, scale=2.0)
    out = preference.preference_loss(z, target, ref, **kw)
    for got, want in zip(out, oracle.pairs64(z, target, ref, **kw)):
        torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-12)
    _against_differences(lambda x: preference.preference_loss(x, target, ref, **kw).loss, z)


def test_positions_that_do_not_count():
    """Their logits, and what else is given for them, may hold anything; targets outside the vocabulary count as ignored."""
    z, target, old, ref, adv = _inputs(dtype=torch.float32)
    old, ref, adv = old.float(), ref.float(), adv.float()
    dead = target == -100
    target[0, 0], target[0, 1] = 11, -7
    for t, fill in ((z, float("nan")), (old, float("inf")), (ref, float("nan")), (adv, float("-inf"))):
        t[dead] = fill
    z.requires_grad_()
    out = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1)
    pair = preference.preference_loss(z, target)
    lp = preference.token_logprobs(z, target)
    for loss in (out.loss, pair.loss, lp.sum()):
        (grad,) = torch.autograd.grad(loss, z)
        assert torch.isfinite(loss) and torch.isfinite(grad).all()
        assert (grad[dead] == 0).all() and (grad[~dead] != 0).any()
    assert (lp[dead] == 0).all()


def test_nothing_counts_and_nothing_there():
    z = torch.randn(2, 3, 5, requires_grad=True)
    target = torch.full((2, 3), -100)
    zero = torch.zeros(2, 3)
    for reduction in ("token", "sequence"):
        out = preference.policy_loss(z, target, zero, zero, zero, kl_coef=0.1, reduction=reduction)
        assert out.loss.item() == 0 and float(out.kl) == 0 and float(out.clip_fraction) == 0
        assert (torch.autograd.grad(out.loss, z)[0] == 0).all()
    out = preference.preference_loss(z, target)
    assert abs(float(out.loss) - math.log(2)) < 1e-6 and (out.margin == 0).all()
    empty = preference.policy_loss(torch.randn(2, 0, 5), torch.zeros(2, 0, dtype=torch.long), torch.zeros(2, 0), torch.zeros(2))
    assert float(empty.loss) == 0 and empty.logp.shape == (2, 0)
    assert preference.token_logprobs(torch.randn(0, 5), torch.zeros(0, dtype=torch.long)).shape == (0,)


def test_refusals():
    z, target, old, ref, adv = _inputs(dtype=torch.float32)
    old, ref, adv = old.float(), ref.float(), adv.float()
    P, T, R = preference.policy_loss, preference.token_logprobs, preference.preference_loss
    with pytest.raises(ValueError, match="logits must be"):
        T(z[0, 0], target[0, 0])
    with pytest.raises(ValueError, match="target must be"):
        T(z, target[:, :-1])
    with pytest.raises(ValueError, match="vocabulary"):
        T(z[..., :0], target)
    with pytest.raises(TypeError, match="int64"):
        T(z, target.int())
    with pytest.raises(TypeError, match="floating"):
        T(z.long(), target)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        for t in (bad, 1e-7, 1e7):
            with pytest.raises(ValueError, match="temperature"):
                T(z, target, temperature=t)
            with pytest.raises(ValueError, match="temperature"):
                P(z, target, old, adv, temperature=t)
        with pytest.raises(ValueError, match="beta"):
            R(z, target, beta=bad)
    with pytest.raises(ValueError, match="old_logp must be"):
        P(z, target, old[0], adv)
    with pytest.raises(TypeError, match="old_logp must be float32"):
        P(z, target, old.bfloat16(), adv)
    with pytest.raises(ValueError, match="advantages must be"):
        P(z, target, old, adv[:, :1])
    with pytest.raises(ValueError, match="kl_coef needs ref_logp"):
        P(z, target, old, adv, kl_coef=0.1)
    with pytest.raises(ValueError, match="kl_coef must be"):
        P(z, target, old, adv, ref, kl_coef=-0.1)
    with pytest.raises(ValueError, match="clip must be"):
        P(z, target, old, adv, clip=float("nan"))
    with pytest.raises(ValueError, match="clip_high must be"):
        P(z, target, old, adv, clip_high=-0.1)
    with pytest.raises(ValueError, match="scale"):
        P(z, target, old, adv, scale=float("inf"))
    with pytest.raises(ValueError, match="reduction must be"):
        P(z, target, old, adv, reduction="sum")
    with pytest.raises(ValueError, match="needs logits"):
        P(z[0], target[0], old[0], adv[0], reduction="sequence")
    with pytest.raises(ValueError, match="chosen"):
        R(z[:3], target[:3])
    with pytest.raises(ValueError, match="chosen"):
        R(z[0], target[0])
    with pytest.raises(ValueError, match="ref_logp must be"):
        R(z, target, ref)
    with pytest.raises(ValueError, match="label_smoothing"):
        R(z, target, label_smoothing=1.1)


def test_native_entry_points_refuse_host_tensors():
    """The bindings check their tensors themselves, before anything is enqueued."""
    from distributed_training_amd.ops import native

    C = native()
    z, target, old, ref, adv = _inputs(dtype=torch.float32)
    old, adv = old.float(), adv.float()
    with pytest.raises(ValueError, match="on a GPU"):
        C.token_logprobs(z, target, -100, 1.0)
    with pytest.raises(ValueError, match="on a GPU"):
        C.policy_loss(z, target, old, adv, None, 0.2, 0.2, 0.0, False, -100, 1.0, 1.0)
    with pytest.raises(ValueError, match="on a GPU"):
        C.preference_loss(z, target, None, 0.1, 0.0, False, -100, 1.0)
    with pytest.raises(TypeError):
        C.token_logprobs(z, None, -100, 1.0)
    with pytest.raises(RuntimeError, match="one GPU"):
        C.grad_sumsq([z])
    with pytest.raises(RuntimeError, match="no tensors"):
        C.grad_sumsq([])


# ------------------------------------------------------------------ gradient norm
def _params(shapes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    params = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.zeros(s, dtype=dtypes[i % len(dtypes)]))
        p.grad = (torch.randn(s, generator=g) * scale).to(p.dtype)
        params.append(p)
    return params


@pytest.mark.parametrize("max_norm", [0.5, 1e6, 0.0])
def test_clip_grad_norm_as_torch(max_norm):
    shapes = [(3, 5), (7,), (), (2, 0), (33, 9)]
    ours, torchs = _params(shapes, [torch.float32]), _params(shapes, [torch.float32])
    ours.append(torch.nn.Parameter(torch.zeros(4)))  # no gradient
    got = optim.clip_grad_norm_(iter(ours), max_norm)
    want = torch.nn.utils.clip_grad_norm_(torchs, max_norm)
    # torch sums in fp32: 312 terms and two roots, under 2^-24 * 64 relative
    torch.testing.assert_close(got, want, rtol=64 * 2.0 ** -24, atol=0)
    for a, b in zip(ours, torchs):
        torch.testing.assert_close(a.grad, b.grad, rtol=64 * 2.0 ** -24, atol=0)


def test_clip_grad_norm_mixed_strided_and_repeated():
    params = _params([(6, 4), (5,), (8, 3)], [torch.float32, torch.bfloat16, torch.float64])
    wide = torch.randn(6, 9)
    params[0].grad = wide[:, 2:6]  # gaps between its rows
    before = [p.grad.double().clone() for p in params]
    norm = math.sqrt(sum(float(b.square().sum()) for b in before))
    got = optim.clip_grad_norm_(params + params[:1], 0.25)  # one listed twice counts once
    assert abs(float(got) - norm) < 2e-7 * norm
    for p, b in zip(params, before):
        want = b * (0.25 / (norm + 1e-6))
        assert ((p.grad.double() - want).abs() <= want.abs() * (oracle.half_step(p.dtype) + 2.0 ** -23)).all()
    assert (wide[:, :2] != 0).all() and torch.equal(params[0].grad, wide[:, 2:6])


def test_norm_of_extremes_and_nonfinite():
    assert float(optim.global_norm([])) == 0
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0
    big = torch.full((100,), 1e25)
    assert abs(float(optim.global_norm(big)) / 1e26 - 1) < 1e-6  # squares beyond fp32
    assert abs(float(optim.global_norm([big * 0 + 1e-30])) / 1e-29 - 1) < 1e-6
    for bad in (float("nan"), float("inf")):
        (p,) = _params([(5,)], [torch.float32])
        p.grad[2] = bad
        with pytest.raises(RuntimeError, match="cannot be clipped"):
            optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        q = torch.nn.Parameter(torch.zeros(5))
        q.grad = p.grad.clone()
        optim.clip_grad_norm_(p, 1.0)
        torch.nn.utils.clip_grad_norm_(q, 1.0)
        torch.testing.assert_close(p.grad, q.grad, equal_nan=True)


def test_norm_refusals():
    (p,) = _params([(5,)], [torch.float32])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grad_norm_(p, bad)
    with pytest.raises(TypeError, match="gradient norm"):
        optim.global_norm([torch.ones(3, dtype=torch.long)])
    with pytest.raises(TypeError, match="gradient norm"):
        optim.global_norm([torch.eye(3).to_sparse()])


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_clip_of_complex_gradients(dtype):
    """A complex parameter's gradient counts with its modulus, beside real ones, as torch's clip has it; also a strided one and a
    conjugate view, of which torch's refuses the latter."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(6, 7, dtype=dtype, generator=g)
    grads = [z[:, 2:5].clone(), z[:, 1:3], z[:2].clone(), torch.randn(5, generator=g)]
    params, theirs = [], []
    for x in grads:
        for found, grad in ((params, x.clone(memory_format=torch.preserve_format)), (theirs, x.clone())):
            found.append(torch.nn.Parameter(torch.zeros(x.shape, dtype=x.dtype)))
            found[-1].grad = grad
    wide = z.clone()
    params[1].grad = wide[:, 1:3]  # gaps between its rows
    params[2].grad = params[2].grad.conj()
    assert params[2].grad.is_conj()
    want = torch.nn.utils.clip_grad_norm_(theirs, 0.5)
    norm = optim.clip_grad_norm_(params + params[:1], 0.5)
    # torch's fp32 sums: 61 terms and their roots
    torch.testing.assert_close(norm.double(), want.double(), rtol=64 * 2.0 ** -24, atol=0)
    for k, (p, q) in enumerate(zip(params, theirs)):
        grad = p.grad.conj() if k == 2 else p.grad
        torch.testing.assert_close(grad, q.grad, rtol=64 * 2.0 ** -24, atol=0)
    assert torch.equal(wide[:, 3:], z[:, 3:]) and torch.equal(wide[:, :1], z[:, :1])
    with pytest.raises(TypeError, match="gradient norm"):
        optim.global_norm([z.to_sparse()])


def test_the_trainer_clips_complex_gradients():
    """The trainer's clip over a plain module takes what torch's took."""
    from types import SimpleNamespace

    from distributed_training_amd.engine.trainer import Trainer

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.ones(3, 2, dtype=torch.complex64) * (1 - 2j))
            self.b = torch.nn.Parameter(torch.ones(2))

        def forward(self, x):
            return (x.to(self.w.dtype) @ self.w).abs() + self.b

    x, y = torch.linspace(-1, 1, 12).view(4, 3), torch.zeros(4, 2)
    nets = Net(), Net()
    torch.nn.functional.mse_loss(nets[1](x), y).backward()
    norm = torch.nn.utils.clip_grad_norm_(nets[1].parameters(), 0.1)
    assert float(norm) > 0.1
    torch.optim.SGD(nets[1].parameters(), lr=1.0).step()
    trainer = SimpleNamespace(optimizer=torch.optim.SGD(nets[0].parameters(), lr=1.0), model=nets[0],
                              config=SimpleNamespace(loss="mse", grad_clip=0.1), _loss_fn=torch.nn.functional.mse_loss)
    Trainer._run_batch_eager(trainer, x, y)
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        # torch's fp32 norm of 8 numbers, and the step's own subtraction
        torch.testing.assert_close(a, b, rtol=16 * 2.0 ** -24, atol=16 * 2.0 ** -24 * 0.1)


def test_per_token_inputs_are_fp32_on_every_device():
    """What the GPU refuses (fp64 per-token inputs beside fp32 or 16-bit logits) the CPU refuses too; fp64 logits, which only the
    CPU takes, come with either."""
    z, target, old, ref, adv = _inputs()
    P, R = preference.policy_loss, preference.preference_loss
    for dtype in (torch.float32, torch.bfloat16):
        x = z.to(dtype)
        P(x, target, old.float(), adv.float(), ref.float())
        for bad in ([old, adv.float(), ref.float()], [old.float(), adv, ref.float()], [old.float(), adv.float(), ref],
                    [old.float(), adv[:, 0], ref.float()]):
            with pytest.raises(TypeError, match="must be float32"):
                P(x, target, *bad)
        R(x, target, ref[:, 0].float())
        with pytest.raises(TypeError, match="ref_logp must be float32"):
            R(x, target, ref[:, 0])
    a, b = P(z, target, old.float(), adv.float(), ref.float()), P(z, target, old, adv, ref)
    assert a.loss.dtype == b.loss.dtype == torch.float64
    R(z[:, :0], target[:, :0], ref[:, 0])


def test_norm_on_the_host_takes_no_copies():
    """Host-resident gradients (offloaded shards) are as large as the model: the norm's fp64 squares are taken piece by piece."""
    import resource

    g = torch.empty(1 << 27).fill_(0.0)  # 512 MB in memory; whole fp64 copies would take 1 GB each
    g[5], g[-1] = 3.0, 4.0
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    norm = optim.clip_grads_([g], 2.5)
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 128 << 10  # KiB
    coef = 2.5 / (5.0 + 1e-6)  # (rounded to fp32, and the products)
    assert float(norm) == 5.0
    assert abs(float(g[5]) / (3.0 * coef) - 1) <= 2.0 ** -23 and abs(float(g[-1]) / (4.0 * coef) - 1) <= 2.0 ** -23
    n = (1 << 18) * 2 + 3  # pieces and a remainder, strided, fp64 (read as it is, not squared in place)
    for t in (torch.randn(n, generator=torch.Generator().manual_seed(0)), torch.randn(n, 2).double()[:, 1]):
        keep = t.clone()
        want = math.sqrt(float(t.double().square().sum()))
        assert abs(float(optim.global_norm(t)) - want) <= 2.0 ** -23 * want and torch.equal(t, keep)


def test_a_coefficient_below_fp32():
    """Gradients near 1e37 clipped to a norm near 1 and below: the coefficient leaves fp32's normal numbers, the products do not.
    (fp32 coefficient and product, the sum of squares in 64 bits: 2^-24 each, and half a step of the type.)"""
    for dtype in (torch.float32, torch.bfloat16, torch.float64):
        for n in (100, 300007):
            base = (torch.rand(n, generator=torch.Generator().manual_seed(n)) + 0.5) * 1e37
            p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device="cpu"))
            before = base.to(dtype).to("cpu")
            norm = math.sqrt(float(before.double().square().sum()))
            for max_norm in (1.0, 1e-4):
                p.grad = before.clone()
                optim.clip_grad_norm_(p, max_norm)
                want = before.double() * (max_norm / (norm + 1e-6))
                step = 2.0 ** -40 if dtype == torch.float64 else oracle.half_step(dtype) * 1.01 + 3 * 2.0 ** -24
                assert ((p.grad.double() - want).abs() <= want * step).all(), (dtype, n, max_norm)
