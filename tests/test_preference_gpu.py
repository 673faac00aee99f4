"""gfx950 kernels of ops/preference.py against 64-bit forms: sizes from one token, every type, rows at any address and
stride, positions that do not count, extreme logits, streams and captured graphs."""
import math

import pytest
import torch
import torch.utils.checkpoint

from distributed_training_amd.ops import preference
from tests import preference_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(B, S, V, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(B, S, V, generator=g) * spread).to(dtype).to(DEV)
    target = torch.randint(V, (B, S), generator=g).to(DEV)
    lp, _ = oracle.logprobs64(z.double(), target)
    old = (lp.cpu() - torch.randn(B, S, generator=g).mul(8).round() / 32 - 1 / 64).float().to(DEV)
    ref = (lp.cpu() + torch.randn(B, S, generator=g).mul(0.3)).float().to(DEV)
    adv = torch.randn(B, S, generator=g).to(DEV)
    if S > 2:
        target[0, : S // 3] = -100
    if B > 2:
        target[2] = -100  # a sequence without tokens
    return z, target, old, ref, adv


def _grad_near(got, want, p, k, k_err, e, dtype):
    """|got - want|: one rounding to the type, the probability's relative error ``e`` (oracle.stat_error) times its
    coefficient, and the coefficient's own error ``k_err`` (fp32 products: 4 u; the slope's dependence on lp: given)."""
    assert got.dtype == dtype and got.shape == want.shape
    k, k_err = k.abs().unsqueeze(-1), k_err.unsqueeze(-1)
    onehot_minus_p = (want / torch.where(k > 0, k, torch.ones_like(k))).abs()
    tol = want.abs() * oracle.half_step(dtype) * 1.01 + k * p * e + (k_err + k * 4 * 2.0 ** -24) * onehot_minus_p * 1.01
    off = (got.double() - want).abs() - (tol + oracle.smallest(dtype) * 1.01 + 2.0 ** -149)
    assert (off <= 0).all(), f"off by {float(off.max())} beyond the tolerance at {int(off.argmax())}"


SHAPES = [(1, 1, 1), (1, 1, 2), (2, 1, 7), (1, 3, 8), (2, 5, 9), (4, 3, 63), (3, 7, 257), (2, 4, 1003), (2, 3, 2048),
          (2, 2, 2049), (1, 2, 8191), (2, 2, 8193), (2, 5, 50257), (1, 3, 128256), (2, 300, 33), (1, 1025, 520),
          (2, 700, 4099)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,V", SHAPES)
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs(B, S, V, dtype, temperature):
    z, target, *_ = _case(B, S, V, dtype, seed=B * S + V)
    w = torch.randn(B, S, generator=torch.Generator().manual_seed(1)).to(DEV)
    z.requires_grad_()
    lp = preference.token_logprobs(z, target, temperature=temperature)
    (grad,) = torch.autograd.grad(lp, z, w)
    z64 = z.detach().double().requires_grad_()
    want, live = oracle.logprobs64(z64, target, temperature=temperature)
    (gwant,) = torch.autograd.grad(want, z64, w.double())
    e = oracle.stat_error(z64.detach(), temperature)
    want = want.detach()
    assert ((lp.detach().double() - want).abs() <= e + want.abs() * 2.0 ** -24).all()
    assert (lp[~live] == 0).all() and (grad[~live] == 0).all()
    k = w.double() / temperature * live
    _grad_near(grad, gwant, torch.softmax(z64.detach() / temperature, -1), k, torch.zeros_like(k), e, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,V", [(1, 1, 1), (2, 5, 9), (4, 3, 63), (3, 7, 257), (2, 4, 1003), (4, 2, 8193), (2, 5, 50257),
                                   (4, 2, 128256), (3, 300, 33), (2, 700, 4099), (1, 512, 1), (3, 257, 8192), (2, 300, 16383),
                                   (1, 520, 24577), (1, 515, 32767), (2, 257, 50257), (1, 512, 53248), (1, 514, 65535),
                                   (1, 513, 70001), (4, 130, 128256), (1, 5000, 33), (20, 40, 65), (17, 30, 1100),
                                   (600, 1, 4200), (3, 200, 60001)])
@pytest.mark.parametrize("kl,high,reduction,scale", [(0.0, None, "token", 1.0), (0.1, 0.28, "sequence", 0.25)])
def test_policy_loss(B, S, V, dtype, kl, high, reduction, scale):
    z, target, old, ref, adv = _case(B, S, V, dtype, seed=B + S + V)
    per_sequence = reduction == "sequence"
    A = adv[:, 0] if per_sequence else adv
    kw = dict(clip_high=high, kl_coef=kl, reduction=reduction, scale=scale)
    z.requires_grad_()
    out = preference.policy_loss(z, target, old, A, ref, **kw)
    (grad,) = torch.autograd.grad(out.loss, z)
    z64 = z.detach().double().requires_grad_()
    loss, lp, mean_kl, clipped = oracle.policy64(z64, target, old, A, ref, **kw)
    lp64 = lp.detach()
    (gwant,) = torch.autograd.grad(loss, z64)
    live = (target != -100).double()
    e = oracle.stat_error(z64.detach())
    A64 = (A.unsqueeze(1) if per_sequence else A).double().expand(B, S)
    ratio, d = torch.exp(lp64 - old.double()), torch.where(live > 0, ref.double() - lp64, torch.zeros_like(lp64))
    n = live.sum().clamp(min=1)
    weight = live / n if reduction == "token" else live / live.sum(1, keepdim=True).clamp(min=1) / B
    # d/dlp of a token's term is at most r |A| + kl |1 - exp(d)|, of its slope r |A| + kl exp(d)
    bend = (ratio * A64.abs() + kl * d.exp()) * weight * scale
    steep = (ratio * A64.abs() + kl * torch.expm1(d).abs()) * weight * scale
    assert abs(float(out.loss.detach()) - float(loss.detach())) <= float((steep * e).sum()) * 1.01 + abs(float(loss.detach())) * 2.0 ** -24
    assert ((out.logp.double() - lp64).abs() <= e + lp64.abs() * 2.0 ** -24).all()
    kl_tol = float(((torch.expm1(d).abs() + e) * live * e).sum() / n) * 1.01 + abs(float(mean_kl)) * 2.0 ** -24
    assert abs(float(out.kl) - float(mean_kl)) <= kl_tol
    assert abs(float(out.clip_fraction) - float(clipped)) <= 2.0 ** -24
    # the token's coefficient as autograd has it: the target's gradient is k (1 - p)
    stopped = ((A64 > 0) & (ratio > 1 + (0.2 if high is None else high))) | ((A64 < 0) & (ratio < 0.8))
    k = (torch.where(stopped, 0.0, -ratio * A64) - kl * torch.expm1(d)) * weight * scale
    _grad_near(grad, gwant, torch.softmax(z64.detach(), -1), torch.where(live > 0, k, 0.0), bend * e, e, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,V", [(2, 1, 1), (2, 5, 9), (4, 3, 63), (6, 7, 257), (4, 2, 8193), (4, 5, 50257), (2, 3, 128256),
                                   (4, 300, 33), (2, 700, 4099), (2, 4500, 17), (300, 2, 40)])
@pytest.mark.parametrize("smoothing,average,use_ref", [(0.0, False, True), (0.1, True, False)])
def test_preference_loss(B, S, V, dtype, smoothing, average, use_ref):
    z, target, *_ = _case(B, S, V, dtype, seed=B + S + V)
    L64 = oracle.pairs64(z.double(), target, None, average=average)[1]
    g = torch.Generator().manual_seed(3)
    ref = (L64.cpu() + torch.randn(B, generator=g)).float().to(DEV) if use_ref else None
    kw = dict(beta=0.7, label_smoothing=smoothing, average=average, scale=1.5)
    z.requires_grad_()
    out = preference.preference_loss(z, target, ref, **kw)
    (grad,) = torch.autograd.grad(out.loss, z)
    z64 = z.detach().double().requires_grad_()
    loss, L, h = oracle.pairs64(z64, target, ref, **kw)
    (gwant,) = torch.autograd.grad(loss, z64)
    live = (target != -100).double()
    L, h, loss = L.detach(), h.detach(), loss.detach()
    share = live / live.sum(1, keepdim=True).clamp(min=1) if average else live
    e = oracle.stat_error(z64.detach())
    eL = (share * e).sum(1)
    P = B // 2
    eh = 0.7 * (eL[:P] + eL[P:])
    u = 2.0 ** -24
    assert ((out.logp.double() - L).abs() <= eL + L.abs() * u).all()
    assert ((out.margin.double() - h).abs() <= eh + h.abs() * u).all()
    assert abs(float(out.loss.detach()) - float(loss)) <= 1.5 * float(eh.mean()) * 1.01 + abs(float(loss)) * u
    slope = 1.5 * 0.7 / P * (torch.sigmoid(h) - (1 - smoothing))
    bend = 1.5 * 0.7 / P * 0.25 * eh * 1.01
    k = torch.cat([slope, -slope]).unsqueeze(1) * share
    _grad_near(grad, gwant, torch.softmax(z64.detach(), -1), k, torch.cat([bend, bend]).unsqueeze(1) * share, e, dtype)


def _all_three(z, target, old, ref, adv, **kw):
    """Losses, statistics and gradients of the three operators on one set of inputs."""
    z = z.detach().requires_grad_()
    a = preference.token_logprobs(z, target, **kw)
    b = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1, **kw)
    got = [a.detach(), b.loss.detach(), b.logp, b.kl, b.clip_fraction]
    got += [torch.autograd.grad(a, z, torch.ones_like(a))[0], torch.autograd.grad(b.loss, z)[0]]
    if z.dim() == 3 and z.shape[0] % 2 == 0:
        c = preference.preference_loss(z, target)
        got += [c.loss.detach(), c.logp, c.margin, torch.autograd.grad(c.loss, z)[0]]
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,V", [(6, 1003), (6, 1008), (131, 1003)])
def test_layouts(S, V, dtype):
    """Rows of a padded vocabulary, every second sequence, shifted tokens, a buffer at an odd address, a transposed
    vocabulary, [N, V] logits, broadcast and transposed per-token arrays: the same bits as the contiguous call."""
    B = 4
    z, target, old, ref, adv = _case(B, S, V, dtype)
    want = _all_three(z, target, old, ref, adv)
    padded = torch.full((B, S, V + 13), float("nan"), device=DEV, dtype=dtype)
    padded[..., 5:V + 5] = z
    odd = torch.empty(B * S * V + 3, device=DEV, dtype=dtype)[3:].view(B, S, V)
    odd.copy_(z)
    spaced = torch.full((2 * B, S + 1, V), float("nan"), device=DEV, dtype=dtype)
    spaced[::2, 1:] = z
    turned = z.transpose(1, 2).contiguous().transpose(1, 2)
    ttarget = target.t().contiguous().t()
    told = torch.stack([old, old], -1)[..., 1]
    for other in (padded[..., 5:V + 5], odd, spaced[::2, 1:], turned):
        for x, y in zip(_all_three(other, ttarget, told, ref.t().contiguous().t(), adv), want):
            assert torch.equal(x, y)
    flat = _all_three(z.view(B * S, V), target.view(-1), old.view(-1), ref.view(-1), adv.view(-1))
    for x, y in zip(flat, want):
        assert torch.equal(x.reshape(-1), y.reshape(-1))
    row_adv = adv[:, :1]
    x = preference.policy_loss(z, target, old, row_adv.expand(B, S))
    y = preference.policy_loss(z, target, old, row_adv[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(x, y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 2100, 50304])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.5, 1.4426950408889634])  # log2(e) / temperature rounds down, up, is 1
def test_extreme_logits(V, dtype, temperature):
    """Rows with masked (-inf, lowest) entries, of nothing but the lowest value, of nothing but -inf, with a NaN or +inf:
    what log_softmax says of each; a target that is masked has log-probability -inf."""
    low = torch.finfo(dtype).min
    z = torch.randn(1, 7, V, generator=torch.Generator().manual_seed(0)).to(dtype).to(DEV)
    target = torch.full((1, 7), V - 1, device=DEV)
    z[0, 0, : V // 2] = float("-inf")
    z[0, 1, : V // 2] = low
    z[0, 2] = low
    z[0, 3] = float("-inf")
    z[0, 4, 1] = float("nan")
    z[0, 5, 2] = float("inf")
    z[0, 6, V - 1] = float("-inf")
    z.requires_grad_()
    lp = preference.token_logprobs(z, target, temperature=temperature)
    (grad,) = torch.autograd.grad(lp.sum(), z)
    z64 = z.detach().double().requires_grad_()
    want = torch.log_softmax(z64 / temperature, -1)[..., V - 1]
    (gwant,) = torch.autograd.grad(want.sum(), z64)
    # (unit-normal rows: the exponents reach under 12 nats, as stat_error counts them for the ordinary row 6)
    e = oracle.stat_error(z64.detach()[:, 6:, :-1], temperature) + 2.0 ** -24 * 64
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(lp), torch.isnan(want)) and torch.equal(torch.isinf(lp), torch.isinf(want))
    assert ((lp.double() - want).abs()[fine] <= e + want.abs()[fine] * 2.0 ** -24).all()
    for row in (0, 1, 2, 6):
        off = (grad[0, row].double() - gwant[0, row]).abs()
        assert (off <= gwant[0, row].abs() * (oracle.half_step(dtype) * 1.01 + 4 * 2.0 ** -24) + e + oracle.smallest(dtype) * 1.01).all()
    for row in (3, 4, 5):
        assert torch.isnan(grad[0, row]).all() == torch.isnan(gwant[0, row]).all()


@pytest.mark.parametrize("S", [9, 200])
def test_positions_that_do_not_count(S):
    """Not read: NaN there reaches nothing; targets outside the vocabulary are positions that do not count."""
    z, target, old, ref, adv = _case(4, S, 777, torch.bfloat16)
    target[target == 5] = 6
    dead = target == -100
    assert dead.any()
    want = _all_three(z, target, old, ref, adv)
    target[0, 0], target[0, 1], target[0, 2] = 777, -7, 2 ** 40
    for t in (z, old, ref, adv):
        t[dead] = float("nan")
    for x, y in zip(_all_three(z, target, old, ref, adv), want):
        assert torch.equal(x, y)
    moved = torch.where(target == -100, 5, target)  # another ignore_index
    for x, y in zip(_all_three(z, moved, old, ref, adv, ignore_index=5)[:7], want[:7]):
        assert torch.equal(x, y)


def test_nothing_counts_and_nothing_there():
    z = torch.randn(2, 3, 50, device=DEV, requires_grad=True)
    target = torch.full((2, 3), -100, device=DEV)
    nan = torch.full((2, 3), float("nan"), device=DEV)
    for reduction in ("token", "sequence"):
        out = preference.policy_loss(z, target, nan, nan, nan, kl_coef=0.1, reduction=reduction)
        assert out.loss.item() == 0 and out.kl.item() == 0 and out.clip_fraction.item() == 0
        assert (torch.autograd.grad(out.loss, z)[0] == 0).all()
    for x, t in ((z, target), (torch.randn(2, 0, 50, device=DEV, requires_grad=True), target[:, :0])):
        out = preference.preference_loss(x, t)
        assert abs(out.loss.item() - math.log(2)) < 1e-6 and (out.margin == 0).all()
        assert (torch.autograd.grad(out.loss, x)[0] == 0).all()
    for shape in ((2, 0, 50), (0, 50)):
        z = torch.randn(shape, device=DEV, requires_grad=True)
        target = torch.zeros(shape[:-1], dtype=torch.long, device=DEV)
        none = torch.zeros(shape[:-1], device=DEV)
        lp = preference.token_logprobs(z, target)
        out = preference.policy_loss(z, target, none, none)
        assert lp.shape == target.shape and out.loss.item() == 0
        assert torch.autograd.grad(out.loss + lp.sum(), z)[0].shape == z.shape


@pytest.mark.parametrize("B,S,V", [(1, 5000, 33), (4, 130, 2003), (2, 300, 50257)])
def test_policy_loss_without_gradient(B, S, V):
    """The forward alone (several passes, no gradient) against the forward with one: each within its bound of the definition."""
    z, target, old, ref, adv = _case(B, S, V, torch.bfloat16)
    e = oracle.stat_error(z.double())
    with torch.no_grad():
        a = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1)
    b = preference.policy_loss(z.clone().requires_grad_(), target, old, adv, ref, kl_coef=0.1)
    live = target != -100
    n = live.sum()
    steep = ((torch.exp(a.logp - old) * adv.abs() + 0.1 * torch.expm1(ref - a.logp).abs()) * live).double().sum() / n
    assert (a.logp - b.logp).abs().max() <= 2 * e + 2.0 ** -23 * a.logp.abs().max()
    assert abs(float(a.loss) - float(b.loss.detach())) <= float(steep) * 2.1 * e + 2.0 ** -23 * abs(float(a.loss))
    assert a.clip_fraction == b.clip_fraction and not a.loss.requires_grad and b.loss.requires_grad


def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements: the last sequence's values and gradients are those of its own call."""
    B, S, V = 4, 4200, 128256
    assert B * S * V > 2 ** 31
    z = torch.zeros(B, S, V, device=DEV, dtype=torch.bfloat16)
    z[-1].normal_(0, 2, generator=torch.Generator(device=DEV).manual_seed(0))
    target = torch.full((B, S), -100, device=DEV)
    target[-1] = torch.randint(V, (S,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    old = torch.full((B, S), -11.5, device=DEV)
    adv = torch.linspace(-1, 1, S, device=DEV).expand(B, S)
    z.requires_grad_()
    out = preference.policy_loss(z, target, old, adv)
    (grad,) = torch.autograd.grad(out.loss, z)
    tail = z.detach()[-1:].clone().requires_grad_()
    want = preference.policy_loss(tail, target[-1:], old[-1:], adv[-1:])
    (gwant,) = torch.autograd.grad(want.loss, tail)
    assert torch.equal(out.loss, want.loss) and torch.equal(out.logp[-1:], want.logp)
    assert torch.equal(grad[-1:], gwant)
    assert not grad[0].any() and not grad[2].any()


@pytest.mark.parametrize("S", [6, 150])  # few rows, and enough for the policy loss's one-pass form
def test_backward_twice_scaled_and_other_uses(S):
    """A retained graph's second backward, a scaled loss, a leaf that accumulates: each as the formula says."""
    z, target, old, ref, adv = _case(4, S, 1003, torch.float32)
    z.requires_grad_()
    for make in (lambda: preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1).loss,
                 lambda: preference.preference_loss(z, target).loss,
                 lambda: preference.token_logprobs(z, target).mean()):
        (g1,) = torch.autograd.grad(make(), z)
        loss = make()
        (a,) = torch.autograd.grad(loss, z, retain_graph=True)
        a.zero_()  # what backward returned belongs to the caller
        (b,) = torch.autograd.grad(loss, z, retain_graph=True)
        (c,) = torch.autograd.grad(loss * 4.0, z)
        assert torch.equal(b, g1) and torch.equal(c, 4.0 * g1)
        z.grad = None
        make().backward()
        (make() * 0.5).backward()
        torch.testing.assert_close(z.grad, 1.5 * g1, rtol=2.0 ** -22, atol=2.0 ** -149)
        z.grad = None
    scaled = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1, scale=0.25)
    full = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1)
    assert torch.equal(scaled.loss, 0.25 * full.loss)
    assert torch.equal(torch.autograd.grad(scaled.loss, z)[0], 0.25 * torch.autograd.grad(full.loss, z)[0])
    with torch.no_grad():
        assert torch.equal(preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1).loss, full.loss)
    with pytest.raises(RuntimeError):  # no second derivatives
        (g,) = torch.autograd.grad(preference.preference_loss(z, target).loss, z, create_graph=True)
        g.sum().backward()
    loss = preference.preference_loss(z.clone(), target).loss
    y = z.clone()
    loss = preference.policy_loss(y, target, old, adv).loss
    y.mul_(2.0)  # the logits changed since the forward: autograd says so
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("S", [40, 140])
def test_same_bits_every_call_and_other_streams(S):
    z, target, old, ref, adv = _case(4, S, 9973, torch.bfloat16)
    want = _all_three(z, target, old, ref, adv)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 2:  # two streams at once
        with torch.cuda.stream(s):
            got.append(_all_three(z, target, old, ref, adv))
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(x, y) for x, y in zip(other, want))


@pytest.mark.parametrize("shape", [(4, 12, 5003), (4, 130, 2003)])
def test_captured_and_replayed(shape):
    """Forward and backward of the three operators in one graph, replayed on new inputs between eager calls."""
    fixed = [t.clone() for t in _case(*shape, torch.bfloat16)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _all_three(*fixed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _all_three(*fixed)
    for seed in range(1, 5):
        new = _case(*shape, torch.bfloat16, seed=seed)
        want = _all_three(*new)
        for f, n in zip(fixed, new):
            f.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        del want, new


@pytest.mark.parametrize("S", [6, 150])
def test_under_inference_mode_hooks_and_checkpoints(S):
    """Scoring under inference_mode, inputs that happen to require a gradient, saved tensors kept on the host, a loss that a
    checkpoint recomputes: the same bits as the plain call."""
    z, target, old, ref, adv = _case(4, S, 1003, torch.bfloat16)
    want = _all_three(z, target, old, ref, adv)
    with torch.inference_mode():
        assert torch.equal(preference.token_logprobs(z * 1.0, target), want[0])
        assert torch.equal(preference.preference_loss(z * 1.0, target).logp, want[8])
    loose = [t.clone().requires_grad_() for t in (old, ref, adv)]
    assert not preference.policy_loss(z, target, loose[0], loose[2], loose[1]).loss.requires_grad
    for x, y in zip(_all_three(z, target, loose[0], loose[1], loose[2]), want):
        assert torch.equal(x, y)
    with torch.autograd.graph.save_on_cpu():
        for x, y in zip(_all_three(z, target, old, ref, adv), want):
            assert torch.equal(x, y)
    leaf = z.clone().requires_grad_()
    loss = torch.utils.checkpoint.checkpoint(
        lambda x: preference.policy_loss(x * 1.0, target, old, adv, ref, kl_coef=0.1).loss, leaf, use_reentrant=False)
    loss.backward()
    assert torch.equal(loss.detach(), want[1]) and torch.equal(leaf.grad, want[6])


def test_refusals_on_the_device():
    z, target, old, ref, adv = _case(2, 3, 50, torch.float32)
    with pytest.raises(TypeError, match="GPU logits"):
        preference.token_logprobs(z.double(), target)
    with pytest.raises(ValueError, match="logits on"):
        preference.token_logprobs(z, target.cpu())
    with pytest.raises(ValueError, match="logits on"):
        preference.policy_loss(z, target, old.cpu(), adv)
    with pytest.raises(TypeError, match="float32"):
        preference.policy_loss(z, target, old, adv.double())
    with pytest.raises(ValueError, match="logits on"):
        preference.preference_loss(z, target, torch.zeros(2))


def test_many_rows_of_a_tiny_vocabulary():
    """The passes take up to 2^24 - 1 rows, the one-pass policy loss up to 2^22 - 1; one more is refused, or done in several
    passes."""
    N = 2 ** 24
    z = torch.zeros(N, 2, device=DEV, dtype=torch.bfloat16)
    z[:, 1] = 1.0
    target = torch.ones(N, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="too many rows"):
        preference.token_logprobs(z, target)
    z = z[:-1].requires_grad_()
    lp = preference.token_logprobs(z, target[:-1])
    want = -math.log1p(math.exp(-1.0))
    assert float((lp.detach() - want).abs().max()) < 1e-6
    (g,) = torch.autograd.grad(lp.sum(), z)
    assert float((g.double() - torch.tensor([-1.0, 1.0], device=DEV) * (1 - math.exp(want))).abs().max()) < 2 ** -10
    for n in (2 ** 22 - 1, 2 ** 22):
        x = z.detach()[:n].requires_grad_()
        old, adv = torch.full((n,), want, device=DEV), torch.ones(n, device=DEV)
        out = preference.policy_loss(x, target[:n], old, adv)
        assert abs(float(out.loss.detach()) + 1.0) < 1e-6 and float(out.clip_fraction) == 0.0
        out.loss.backward()
        # k = -1 / n times [-(1 - p), 1 - p], rounded to bf16
        slope = (1 - math.exp(want)) / n
        assert float((x.grad.double() - torch.tensor([slope, -slope], device=DEV, dtype=torch.float64)).abs().max()) <= slope * 2 ** -7


def test_a_preference_step_end_to_end():
    """A reference model scores, the policy under the DDP engine is trained on pairs and on rewards, gradients are
    clipped, the optimizer steps: the run of operators as a training program has them, its gradients against the same
    run with the losses in 64 bits."""
    from distributed_training_amd.models.gpt2 import GPT2, GPT2Config
    from distributed_training_amd.ops.optim import FusedAdamW
    from distributed_training_amd.parallel.comm import RcclComm
    from distributed_training_amd.parallel.ddp import DistributedDataParallel

    torch.manual_seed(0)
    dev = torch.device(DEV, 0)
    model = GPT2(GPT2Config(n_layer=2, n_head=2, n_embd=128, vocab_size=1000, block_size=64)).to(dev)
    w = DistributedDataParallel(model, comm=RcclComm(0, 1, dev), device=dev, param_dtype=torch.bfloat16)
    opt = FusedAdamW(w.parameters(), lr=1e-3)
    idx = torch.randint(1000, (4, 64), device=DEV)
    target = torch.roll(idx, -1, 1)
    target[:, :8] = -100
    target[:, -1] = -100
    adv = torch.tensor([1.0, -0.5, 0.8, -1.2], device=DEV)
    with torch.no_grad():
        ref_tok = preference.token_logprobs(w(idx), target)

    def loss_of(logits, exact):
        if exact:
            z = logits.double()
            return (oracle.policy64(z, target, ref_tok + 0.1, adv, ref_tok, kl_coef=0.05)[0]
                    + oracle.pairs64(z, target, ref_tok.sum(1))[0]).float()
        return (preference.policy_loss(logits, target, ref_tok + 0.1, adv, ref_tok, kl_coef=0.05).loss
                + preference.preference_loss(logits, target, ref_tok.sum(1)).loss)

    for step in range(2):
        grads = []
        for exact in (True, False):
            w.zero_grad(set_to_none=True)
            loss_of(w(idx), exact).backward()
            torch.cuda.synchronize()
            grads.append([p.grad.double().clone() for p in w.parameters()])
        for a, b in zip(*grads):
            # the logit gradients of the two losses are rounded to bf16 before their sum is (half a step each, 2^-9 of a
            # term), and what follows rounds at each of the 2 layers' 8 products and norms: a few of those steps in norm
            assert (a - b).norm() <= 16 * 2.0 ** -9 * a.norm() + 1e-6
        want = math.sqrt(sum(float(g.square().sum()) for g in grads[1]))
        norm = w.clip_grad_norm_(0.1)
        assert want > 0.1 and abs(float(norm) - want) <= 2.0 ** -23 * want
        for p, g in zip(w.parameters(), grads[1]):
            g = g * (0.1 / (want + 1e-6))
            assert ((p.grad.double() - g).abs() <= g.abs() * (oracle.half_step(p.grad.dtype) + 2.0 ** -22)).all()
        opt.step()
    assert all(torch.isfinite(p).all() for p in w.parameters())


@pytest.mark.parametrize("V", [2100, 50304])
def test_extreme_logits_in_one_pass(V):
    """The policy loss's one-pass form on rows with -inf and lowest entries agrees with the form for few rows, and a row that
    is NaN by the definition makes its own gradient NaN and no other's."""
    z = torch.randn(1, 600, V, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    target = torch.full((1, 600), V - 1, device=DEV)
    z[0, 0, : V // 2] = float("-inf")
    z[0, 1, : V // 2] = torch.finfo(torch.bfloat16).min
    z[0, 2] = torch.finfo(torch.bfloat16).min
    old, adv = torch.full((1, 600), -8.0, device=DEV), torch.ones(1, 600, device=DEV)
    few = slice(0, 40)

    def grads(z, n, scale):
        z = z.detach().requires_grad_()
        out = preference.policy_loss(z, target[:, :n], old[:, :n], adv[:, :n], clip_high=1e9, scale=scale)
        return out.logp, torch.autograd.grad(out.loss, z)[0]

    lp, g = grads(z, 600, 600.0)
    lp_few, g_few = grads(z[:, few], 40, 40.0)
    e = oracle.stat_error(z[:, 3:].double())
    assert torch.isfinite(g).all()
    assert ((lp[:, few] - lp_few).abs() <= 2 * e + lp_few.abs() * 2.0 ** -23).all()
    assert ((g[:, few].double() - g_few.double()).abs() <= g_few.double().abs() * 2.0 ** -7 + 4 * e * math.exp(8.0)).all()
    z[0, 3], z[0, 4, 7], z[0, 5, 9] = float("-inf"), float("nan"), float("inf")
    lp, g = grads(z, 600, 600.0)
    assert torch.isnan(lp[0, 3:6]).all() and torch.isnan(g[0, 3:6]).all()
    assert torch.isfinite(lp[0, 6:]).all() and torch.isfinite(g[0, 6:]).all() and torch.isfinite(g[0, :3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 7, 8, 9, 63, 512, 513, 1024, 1025, 2047, 2048, 2049, 4096, 4097])
def test_short_rows(V, dtype):
    """From 2000 rows on a short row is one wave's: the operators at the sizes around its limits, rows not in fours."""
    test_token_logprobs(3, 667, V, dtype, 0.7)
    test_policy_loss(3, 667, V, dtype, 0.1, 0.28, "sequence", 0.25)
    test_preference_loss(2, 1001, V, dtype, 0.1, True, False)


@pytest.mark.parametrize("S,V", [(1, 40), (16, 513), (17, 40), (40, 8193), (300, 65)])
@pytest.mark.parametrize("B", [1, 2, 3, 5, 12, 15, 16, 17, 40])
def test_sums_over_sequences(B, S, V):
    """Terms by row, added up by waves: sequences shorter and longer than a thread takes, fewer and more than the waves."""
    test_policy_loss_without_gradient(B, S, V)
    test_policy_loss(B, S, V, torch.bfloat16, 0.1, 0.28, "sequence", 0.25)
    if B % 2 == 0:
        test_preference_loss(B, S, V, torch.float32, 0.1, True, False)


def test_more_rows_than_terms_by_row():
    for B, S in ((2, 2048), (2, 2049), (128, 32), (2, 33000), (4100, 2), (1, 70001)):
        test_policy_loss_without_gradient(B, S, 9)
        if B % 2 == 0:
            test_preference_loss(B, S, 9, torch.bfloat16, 0.0, False, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [900, 2000, 4000])
def test_extreme_logits_in_short_rows(V, dtype):
    """Rows of -inf, of the type's lowest value, of NaN and inf, of strided logits: a wave a row as a workgroup a row."""
    N = 2003
    wide = torch.randn(N, V + 5, generator=torch.Generator().manual_seed(V)).to(dtype).to(DEV)
    z = wide[:, 3:3 + V]
    target = torch.randint(V, (N,), generator=torch.Generator().manual_seed(1)).to(DEV)
    target[7], target[8], target[2002] = -100, V, -1
    low = torch.finfo(dtype).min
    z[0, : V - 1], z[1], z[2, : V // 2], z[3] = float("-inf"), low, low, float("-inf")
    z[4, 5], z[5, V - 1], z[7], z[2002] = float("nan"), float("inf"), float("nan"), float("nan")
    target[0] = V - 1
    got = []
    for n in (N, 40):
        x = z[:n].detach().requires_grad_()
        lp = preference.token_logprobs(x, target[:n], temperature=0.7)
        got.append((lp.detach(), torch.autograd.grad(lp.sum(), x)[0]))
    (lp, g), (lp_few, g_few) = got
    assert float(lp[0]) == 0.0 and abs(float(lp[1]) + math.log(V)) < 1e-5
    bad = torch.isin(torch.arange(40, device=DEV), torch.tensor([3, 4, 5], device=DEV))
    assert torch.isnan(lp[3:6]).all() and torch.isnan(g[3:6]).all()
    for row in (7, 8, 2002):
        assert float(lp[row]) == 0.0 and not g[row].any()
    assert torch.isfinite(lp[6:]).all() and torch.isfinite(g[6:]).all()
    live = ~bad & (target[:40] >= 0) & (target[:40] < V)
    # both forms are within stat_error of the same value; rows 0 and 1 are exact or uniform; row 2's lowest entries add
    # exactly 0 (2^-inf), the others make an ordinary row of it (a target among the lowest: lp is -inf or near it in both)
    e = torch.zeros(40, 1, device=DEV, dtype=torch.float64)
    e[6:] = oracle.stat_error(torch.nan_to_num(z[6:40].double()), 0.7)
    e[:2] = 2.0 ** -20
    e[2] = oracle.stat_error(z[2:3, V // 2:].double(), 0.7)
    near = (lp[:40] - lp_few).abs() <= 2 * e[:, 0] + lp_few.abs() * 2.0 ** -23
    assert (near | (lp[:40] == lp_few))[live].all()
    tol = g_few.double().abs() * (2 * oracle.half_step(dtype) * 1.01 + 2 * e) + oracle.smallest(dtype) * 2
    assert ((g[:40].double() - g_few.double()).abs() <= tol + 2 * e / 0.7)[live].all()


@pytest.mark.parametrize("S", [6, 150])  # few rows, and enough for the policy loss's one-pass form
@pytest.mark.parametrize("which", ["logprobs", "policy", "preference"])
def test_second_derivatives_are_refused(which, S):
    """A gradient taken with create_graph is right as it is; whoever differentiates it is told, through whichever of its
    inputs, and nothing that lacks the gradient's own term comes back."""
    z, target, old, ref, adv = _case(4, S, 203, torch.float32)
    loss_of = {"logprobs": lambda x: preference.token_logprobs(x, target).mean(),
               "policy": lambda x: preference.policy_loss(x, target, old, adv, ref, kl_coef=0.1).loss,
               "preference": lambda x: preference.preference_loss(x, target).loss}[which]
    leaf = z.clone().requires_grad_()
    (want,) = torch.autograd.grad(loss_of(leaf), leaf)
    loss = loss_of(leaf)
    (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
    assert torch.equal(g.detach(), want)
    with pytest.raises(RuntimeError, match="differentiated once"):  # the loss and a penalty on its gradient
        (loss + g.square().sum()).backward()
    half = torch.full((), 0.5, device=DEV, requires_grad=True)
    for inputs in ([leaf], [half], [leaf, half]):  # by way of logits that are computed, and of the gradient that arrived
        loss = loss_of(leaf * 2.0) * half
        (g,) = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(g.square().sum(), inputs)
    # a penalty on a gradient that does not come through the losses
    w = torch.full((), 3.0, device=DEV, requires_grad=True)
    (gw,) = torch.autograd.grad(loss_of(leaf) + w ** 3, w, create_graph=True)
    gw.square().backward()
    assert float(w.grad) == 2 * 27.0 * 18.0


def _policy_forward_near(B, S, V, dtype):
    """The forward alone against the definition (test_policy_loss has the gradient's form, which may be another)."""
    z, target, old, ref, adv = _case(B, S, V, dtype, seed=B + S + V)
    with torch.no_grad():
        out = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1)
    loss, lp, mean_kl, clipped = oracle.policy64(z.double(), target, old, adv, ref, kl_coef=0.1)
    live = (target != -100).double()
    n = live.sum().clamp(min=1)
    e = oracle.stat_error(z.double())
    d = torch.where(live > 0, ref.double() - lp, torch.zeros_like(lp))
    # d/dlp of a token's term is at most r |A| + kl |expm1(d)|, of its KL |expm1(d)|; the second order in e behind it
    steep = (torch.exp(lp - old.double()) * adv.double().abs() + 0.1 * torch.expm1(d).abs() + e) * live / n
    assert abs(float(out.loss) - float(loss)) <= float(steep.sum()) * e * 1.01 + abs(float(loss)) * 2.0 ** -24
    assert ((out.logp.double() - lp).abs() <= e + lp.abs() * 2.0 ** -24).all()
    kl_tol = float(((torch.expm1(d).abs() + e) * live * e).sum() / n) * 1.01 + abs(float(mean_kl)) * 2.0 ** -24
    assert abs(float(out.kl) - float(mean_kl)) <= kl_tol
    assert abs(float(out.clip_fraction) - float(clipped)) <= 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,V", [(1, 3, 70001), (2, 20, 128251), (4, 10, 65543), (2, 127, 70001), (3, 85, 70001), (2, 1, 600001)])
def test_rows_in_pieces(B, S, V, dtype):
    """Under 256 rows of more than 65536 logits are cut into pieces: odd vocabularies (a remainder behind the last piece's whole
    chunks), 8 to 64 lanes a row in the kernels that join them, sequences over several of their workgroups."""
    test_token_logprobs(B, S, V, dtype, 0.7)
    test_policy_loss(B, S, V, dtype, 0.1, 0.28, "sequence", 0.25)
    _policy_forward_near(B, S, V, dtype)
    if B % 2 == 0:
        test_preference_loss(B, S, V, dtype, 0.1, True, False)


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_logits_in_pieces(dtype):
    test_extreme_logits(70001, dtype, 0.7)
    V = 70001  # nine pieces of 7784 logits
    z = torch.full((1, 5, V), float("-inf"), device=DEV, dtype=dtype)
    target = torch.full((1, 5), V - 1, device=DEV)
    z[0, 0, V - 1] = 3.0  # one logit, behind the last whole chunk
    z[0, 1, 7784 * 4], z[0, 1, V - 1] = 1.0, 1.0  # a piece of one logit between pieces of none
    z[0, 2, 5], z[0, 3, 60000] = float("nan"), float("inf")
    z.requires_grad_()
    lp = preference.token_logprobs(z, target)
    (grad,) = torch.autograd.grad(lp.sum(), z)
    lp = lp.detach()
    assert float(lp[0, 0]) == 0.0 and abs(float(lp[0, 1]) + math.log(2.0)) < 2.0 ** -20
    assert torch.isnan(lp[0, 2:]).all() and torch.isnan(grad[0, 2:]).any(-1).all()
    assert not grad[0, 0].any()
    # p = 1/2 with an error of stat_error's order in its exponent (reach 17 for V = 70001: under 2^-16), half a step of the type
    for j, want in ((7784 * 4, -0.5), (V - 1, 0.5)):
        assert abs(float(grad[0, 1, j]) - want) <= 0.5 * (oracle.half_step(dtype) + 2.0 ** -16)
    assert int(torch.count_nonzero(grad[0, 1])) == 2


@pytest.mark.parametrize("dtype", TYPES)
def test_long_rows_by_the_thousand(dtype):
    """More rows than their terms are added up one by one, each of 1024 threads."""
    _policy_forward_near(2, 2050, 60001, dtype)
    test_preference_loss(2, 2050, 60001, dtype, 0.1, True, False)


def test_rows_beyond_a_launch_of_wide_workgroups():
    """2^22 rows of a long vocabulary (expanded logits: no memory behind them): with 1024 threads a row the launch would take
    2^32, so these get 256.  All but a few positions are ignored, and those are as the definition says."""
    B, S, V = 2, 2 ** 21, 60001
    base = torch.randn(V, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    z = base.expand(B, S, V)
    target = torch.full((B, S), -100, device=DEV)
    at = torch.tensor([0, 1, S // 2, S - 1], device=DEV)
    target[:, at] = torch.tensor([[5, V - 1, 70, 0], [9, 9, V - 2, 1]], device=DEV)
    few = target[:, at]
    want, _ = oracle.logprobs64(base.double().expand(B, 4, V), few)
    e = oracle.stat_error(base.double()[None])
    lp = preference.token_logprobs(z, target)
    assert ((lp[:, at].double() - want).abs() <= e + want.abs() * 2.0 ** -24).all()
    lp[:, at] = 0.0
    assert not lp.any()
    zero, one = torch.zeros(B, S, device=DEV), torch.ones(B, device=DEV)
    out = preference.policy_loss(z, target, zero, one)
    r = want.exp()  # at most 1: unclipped, or clipped from below where the advantage is positive: -r A either way
    assert abs(float(out.loss) + float(r.mean())) <= float(r.mean()) * (e + 2.0 ** -24) * 1.01
    pair = preference.preference_loss(z, target, average=True)
    L = want.mean(1)
    assert ((pair.logp.double() - L).abs() <= e + L.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("S,grad", [(20, True), (20, False), (200, True), (5000, True), (5000, False)])
@pytest.mark.parametrize("step", [1e-5, -3e-4, 0.0077, 0.0079])
def test_small_kl(S, grad, step):
    """A reference next to the policy: exp(d) - 1 - d of a d of 1e-5 and more, in every form of the loss.  Uniform rows, whose
    log-probability -log V is exact to 64 bits: log2, its product with ln 2 and the oracle's logarithm are within 2^-52 of it each,
    d within their sum, the KL term within twice that of d (and the series within 2^-46); then one rounding to fp32."""
    V = 1003
    z = torch.zeros(1, S, V, device=DEV, requires_grad=grad)
    target = torch.arange(S, device=DEV).remainder(V)[None]
    lp = -math.log(V)
    ref = (lp + step * torch.linspace(0.9, 1.1, S, dtype=torch.float64)).float().to(DEV)[None]
    d = ref.double() - lp
    out = preference.policy_loss(z, target, torch.full_like(ref, lp), torch.zeros_like(ref), ref, kl_coef=0.5)
    # the same series to d^8, far below 2^-53 of it
    want = d * d * sum(d ** n / math.factorial(n + 2) for n in range(7))
    tol = 2.0 ** -24 * 1.01 + 2 * 3 * 2.0 ** -52 * abs(lp) / (0.9 * abs(step)) + 2.0 ** -46
    assert abs(float(out.kl) / float(want.mean()) - 1.0) <= tol
    assert abs(float(out.loss.detach()) / (0.5 * float(want.mean())) - 1.0) <= tol + 2.0 ** -24
    assert float(out.clip_fraction) == 0.0


@pytest.mark.parametrize("S", [9, 77, 700])
def test_coefficients_are_rounded_once(S):
    """Uniform rows of 1024 fp32 logits: a probability is 2^-10 exactly, so -2^10 times a gradient (not the target's) is the row's
    coefficient, slope x weight x arriving gradient / temperature, whose one rounding to fp32 is half a step."""
    B, V, T = 2, 1024, 0.7
    g = torch.Generator().manual_seed(S)
    z = torch.zeros(B, S, V, device=DEV, requires_grad=True)
    target = torch.zeros(B, S, dtype=torch.int64, device=DEV)
    target[1, S // 3:] = -100
    live = (target == 0).double()
    w, adv = torch.randn(B, S, generator=g).to(DEV), torch.randn(B, generator=g).to(DEV)
    lp = -10.0 * math.log(2.0)
    old = (lp + 0.1 * torch.rand(B, S, generator=g, dtype=torch.float64)).float().to(DEV)
    tokens = live.sum(1, keepdim=True)

    def near(loss, arriving, k):
        (grad,) = torch.autograd.grad(loss, z, arriving)
        k = k * live
        # (fp64: the slope's exponentials and products, a few 2^-53)
        off = (grad[..., 5].double() * -1024.0 - k).abs() - k.abs() * (2.0 ** -24 + 2.0 ** -46)
        assert (off <= 0).all(), float((off / k.abs()).nan_to_num(0.0).max())

    near(preference.token_logprobs(z, target, temperature=T), w, w.double() / T)
    r = torch.exp(lp - old.double())
    out = preference.policy_loss(z, target, old, adv, reduction="sequence", temperature=T, scale=0.3, clip=0.9)
    near(out.loss, None, -r * adv.double()[:, None] * 0.3 / T / tokens / B)
    out = preference.policy_loss(z, target, old, adv, reduction="sequence", temperature=T, scale=0.3, clip=0.9)
    arriving = torch.tensor(0.77, device=DEV)
    near(out.loss, arriving, -r * adv.double()[:, None] * 0.3 / T * arriving.double() / tokens / B)
    pair = preference.preference_loss(z, target, torch.tensor([0.3, -0.4], device=DEV), beta=0.37, average=True, scale=0.3)
    h = 0.37 * -(torch.tensor(0.3).double() + torch.tensor(0.4).double()).item()
    slope = 0.3 * 0.37 * (1.0 / (1.0 + math.exp(-h)) - 1.0)
    near(pair.loss, None, torch.tensor([[slope], [-slope]], device=DEV, dtype=torch.float64) / tokens)


@pytest.mark.parametrize("S", [12, 130])  # few rows, and enough for the policy loss's one-pass form
def test_captured_with_a_retained_and_scaled_backward(S):
    """One graph with a forward, a backward of a scaled loss that retains it, and another of it: every replay as the eager calls;
    and a graph of a backward alone, whose forward ran before on the same stream."""
    shape = (4, S, 2003)
    fixed = [t.clone() for t in _case(*shape, torch.bfloat16)]
    factor = torch.full((), 4.0, device=DEV)

    def both(z, target, old, ref, adv, factor):
        z = z.detach().requires_grad_()
        loss = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1).loss
        (a,) = torch.autograd.grad(loss, z, factor, retain_graph=True)
        (b,) = torch.autograd.grad(loss, z)
        return loss.detach(), a, b

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*fixed, factor)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*fixed, factor)
    for seed in range(1, 5):
        new = _case(*shape, torch.bfloat16, seed=seed)
        scale = torch.full((), 0.5 if seed % 2 else 1.0, device=DEV)
        want = both(*new, scale)
        for f, n in zip([*fixed, factor], [*new, scale]):
            f.copy_(n)
        out[1].zero_(), out[2].zero_()  # (the gradients are the caller's)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        del want, new
    # (a power of two scales the rounded gradient exactly)
    assert torch.equal(out[1], out[2])

    z, target, old, ref, adv = _case(*shape, torch.bfloat16)
    z.requires_grad_()
    (want,) = torch.autograd.grad(preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1).loss, z)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        loss = preference.policy_loss(z, target, old, adv, ref, kl_coef=0.1).loss
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        (got,) = torch.autograd.grad(loss, z, retain_graph=True)
    for _ in range(3):
        got.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    (again,) = torch.autograd.grad(loss, z)  # the eager backward of the same loss
    assert torch.equal(again, want)


def test_a_preference_step_under_fsdp():
    """The losses behind the FSDP engine: gradients against the same run with the losses in 64 bits, the clip over its shards,
    an optimizer step."""
    from distributed_training_amd.models.gpt2 import GPT2, GPT2Config
    from distributed_training_amd.ops.optim import FusedAdamW
    from distributed_training_amd.parallel.comm import RcclComm
    from distributed_training_amd.parallel.fsdp import FullyShardedDataParallel, lm_wrap_policy

    torch.manual_seed(0)
    dev = torch.device(DEV, 0)
    model = GPT2(GPT2Config(n_layer=2, n_head=2, n_embd=128, vocab_size=1000, block_size=64)).to(dev)
    w = FullyShardedDataParallel(model, comm=RcclComm(0, 1, dev), device=dev, wrap_policy=lm_wrap_policy(model),
                                 param_dtype=torch.bfloat16)
    opt = FusedAdamW(w.parameters(), lr=1e-3)
    idx = torch.randint(1000, (4, 64), device=DEV)
    target = torch.roll(idx, -1, 1)
    target[:, :8] = -100
    target[:, -1] = -100
    adv = torch.tensor([1.0, -0.5, 0.8, -1.2], device=DEV)
    with torch.no_grad():
        ref_tok = preference.token_logprobs(w(idx), target)
    for step in range(2):
        grads = []
        for exact in (True, False):
            w.zero_grad(set_to_none=True)
            logits = w(idx)
            if exact:
                z = logits.double()
                loss = (oracle.policy64(z, target, ref_tok + 0.1, adv, ref_tok, kl_coef=0.05)[0]
                        + oracle.pairs64(z, target, ref_tok.sum(1))[0]).float()
            else:
                loss = (preference.policy_loss(logits, target, ref_tok + 0.1, adv, ref_tok, kl_coef=0.05).loss
                        + preference.preference_loss(logits, target, ref_tok.sum(1)).loss)
            loss.backward()
            torch.cuda.synchronize()
            grads.append(w.shards.grad.double().clone())
        a, b = grads
        # bf16 logit gradients of two losses, rounded before their sum, and the 2 layers' roundings behind them, as under DDP
        assert a.norm() > 0 and (a - b).norm() <= 16 * 2.0 ** -9 * a.norm() + 1e-6
        want = float(b.norm())
        norm = w.clip_grad_norm_(0.1)
        assert want > 0.1 and abs(float(norm) - want) <= 2.0 ** -23 * want
        g = b * (0.1 / (want + 1e-6))
        assert ((w.shards.grad.double() - g).abs() <= g.abs() * (oracle.half_step(w.shards.grad.dtype) + 2.0 ** -22)).all()
        opt.step()
    assert all(torch.isfinite(p).all() for p in w.parameters())
