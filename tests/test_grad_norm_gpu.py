"""gfx950 kernels of the global gradient norm and clipping (csrc/grad_norm.hip) against 64-bit sums: any number of
tensors, sizes, types and addresses; extremes; the engines' own clip; captured graphs."""
import math

import pytest
import torch

from distributed_training_amd.ops import optim
from tests import preference_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def _params(sizes, dtypes, seed=0, scale=1.0, offset=0):
    """Parameters whose gradients are slices of one buffer a type, ``offset`` elements apart."""
    g = torch.Generator().manual_seed(seed)
    params = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        buf = torch.empty(n + offset, dtype=dt, device=DEV)
        buf.copy_(torch.randn(n + offset, generator=g) * scale)
        p = torch.nn.Parameter(torch.zeros((), device=DEV, dtype=dt).expand(n))
        p.grad = buf[offset:]
        params.append(p)
    return params


def _check(params, max_norm):
    before = [p.grad.double().clone() for p in params]
    norm = math.sqrt(sum(float(b.square().sum()) for b in before))
    got = optim.global_norm([p.grad for p in params])
    # fp64 sums: only the root's rounding to fp32 (and fp64 sums of the oracle, far below)
    assert got.dtype == torch.float32 and abs(float(got) - norm) <= 2.0 ** -24 * 1.01 * norm
    assert torch.equal(optim.clip_grad_norm_(params, max_norm), got)
    coef = min(1.0, max_norm / (norm + 1e-6))
    for p, b in zip(params, before):
        want = b * coef
        if coef == 1.0:
            assert torch.equal(p.grad.double(), b)
            continue
        # the coefficient in fp32, the product in fp32, one rounding to the type.  fp64 gradients see the two sums' own
        # rounding instead: a kernel's term passes at most 8192 / 256 x units of a workgroup + 6 + 4 + 2 + 6 + 16 fp64
        # additions, the oracle's at most 500 tensors + its pairwise sums: under 1024 of 2^-53 each, and the root halves
        # their sum (2^9 x 2^-53 x 2 sides = 2^-43)
        u = 2.0 ** -43 if p.dtype == torch.float64 else 2.0 ** -24
        tol = want.abs() * (oracle.half_step(p.dtype) + 3 * u) + oracle.smallest(p.dtype) * 1.01
        assert ((p.grad.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 255, 8191, 8192, 8193, 100003, 5 * 2 ** 20 + 1])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_one_tensor(n, dtype, offset):
    _check(_params([n], [dtype], seed=n, offset=offset), 0.3)


@pytest.mark.parametrize("count", [2, 159, 160, 161, 500])
def test_many_tensors_of_mixed_types(count):
    sizes = [(37 * i * i + 1) % 20011 for i in range(count)]
    sizes[1] = 0
    _check(_params(sizes, TYPES, seed=count, offset=1), 1.0)


@pytest.mark.parametrize("sizes", [[20 * 512, 512, 512, 1], [1] * 64, [0, 513, 0, 64 * 512 - 1024], [1] * 65, [32769],
                                   [7] * 161, [64] * 64, [1024 * 8192], [1024 * 8192 - 5, 9]])
def test_small_models(sizes):
    """Up to 64 units of 512 elements: one launch; up to 1024 of 8192 in at most 160 tensors: two.  The sizes around."""
    for dtypes in ([torch.float32], TYPES):
        for max_norm in (0.2, 1e6):
            _check(_params(sizes, dtypes, seed=len(sizes), offset=1), max_norm)
    q = torch.nn.Parameter(torch.empty(0, device=DEV))
    q.grad = torch.empty(0, device=DEV)
    assert float(optim.clip_grad_norm_([q], 1.0)) == 0.0


def test_within_the_bound_nothing_changes():
    _check(_params([1000, 3], [torch.bfloat16, torch.float32]), 1e6)
    params = _params([3000], [torch.float32])
    norm = float(optim.global_norm(params[0].grad))
    _check(params, norm * (1 + 2.0 ** -20) + 1e-6)
    _check(_params([3000], [torch.float32]), 0.0)  # a bound of 0 clears them


def test_layouts():
    """Transposed gradients are read as they lie; strided ones keep what is between their elements."""
    base = torch.randn(64, 48, device=DEV)
    p, q = (torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((48, 64), (64, 20)))
    p.grad = base.clone().t()
    wide = torch.randn(64, 50, device=DEV)
    keep = wide.clone()
    q.grad = wide[:, 7:27]
    before = torch.cat([p.grad.double().reshape(-1), q.grad.double().reshape(-1)])
    norm = float(before.square().sum().sqrt())
    got = optim.clip_grad_norm_([p, q, p], 0.5)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    want = before * (0.5 / (norm + 1e-6))
    after = torch.cat([p.grad.double().reshape(-1), q.grad.double().reshape(-1)])
    assert ((after - want).abs() <= want.abs() * 4 * 2.0 ** -24).all()
    assert torch.equal(wide[:, :7], keep[:, :7]) and torch.equal(wide[:, 27:], keep[:, 27:])


def test_what_is_listed_twice_is_clipped_once():
    p, q = _params([4000, 4000], [torch.float32])
    q.grad = p.grad
    before = p.grad.double().clone()
    norm = float(before.square().sum().sqrt())
    for params in ([p, q], [p, p, q]):
        p.grad.copy_(before)
        assert abs(float(optim.clip_grad_norm_(params, 0.5)) - norm) <= 2.0 ** -23 * norm
        assert ((p.grad.double() - before * (0.5 / (norm + 1e-6))).abs() <= before.abs() * 2.0 ** -22).all()
    optim.grad_clip_([p.grad, p.grad], optim.grad_sumsq([p.grad])[0], 0.25)
    want = before * (0.25 / norm)
    assert ((p.grad.double() - want).abs() <= want.abs() * 1e-5).all()


def test_gradients_that_share_a_part_are_refused():
    base = torch.ones(100, device=DEV)
    p, q = (torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (10, 100))
    for first in (base[:10], base[40:50], base[90:]):
        p.grad, q.grad = first, base
        for params in ([p, q], [q, p], [p, p, q]):
            with pytest.raises(ValueError, match="overlap"):
                optim.clip_grad_norm_(params, 0.5)
    assert torch.equal(base, torch.ones_like(base))
    r = torch.nn.Parameter(torch.zeros(90, device=DEV))
    p.grad, r.grad = base[:10], base[10:]  # (neighbours in memory are two gradients)
    assert abs(float(optim.clip_grad_norm_([r, p, r], 11.0)) - 10.0) < 1e-5
    square = torch.nn.Parameter(torch.zeros(10, 10, device=DEV))
    square.grad, q.grad = base.view(10, 10).t(), base.view(100)
    for flag in (False, True):  # one memory in two orders
        assert abs(float(optim.clip_grad_norm_([square, q], 11.0, error_if_nonfinite=flag)) - 10.0) < 1e-5


def test_extremes_and_nonfinite():
    assert abs(float(optim.global_norm(torch.full((10000,), 1e25, device=DEV))) / 1e27 - 1) < 1e-6
    assert abs(float(optim.global_norm(torch.full((10000,), 1e-30, device=DEV))) / 1e-28 - 1) < 1e-6
    for bad in (float("nan"), float("inf")):
        for dtype in TYPES:
            (p,) = _params([20000], [dtype])
            p.grad[19999] = bad
            q = torch.nn.Parameter(torch.zeros(20000, device=DEV, dtype=dtype))
            q.grad = p.grad.clone()
            with pytest.raises(RuntimeError, match="cannot be clipped"):
                optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
            assert torch.equal(p.grad.nan_to_num(5.0), q.grad.nan_to_num(5.0))
            optim.clip_grad_norm_(p, 1.0)
            torch.nn.utils.clip_grad_norm_(q, 1.0)
            torch.testing.assert_close(p.grad, q.grad, equal_nan=True, rtol=0, atol=0)


def test_more_than_2_to_the_31_elements():
    n = 2 ** 31 + 12345
    g = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g[-1], g[-8192], g[2 ** 31 - 1] = 3.0, 4.0, 12.0
    p = torch.nn.Parameter(torch.zeros((), device=DEV, dtype=torch.bfloat16).expand(n))
    p.grad = g
    assert float(optim.clip_grad_norm_(p, 6.5)) == 13.0
    assert [float(g[i]) for i in (-1, -8192, 2 ** 31 - 1, 5)] == [1.5, 2.0, 6.0, 0.0]


def test_same_bits_and_streams():
    params = _params([300007, 5, 70001], TYPES)
    want = optim.global_norm([p.grad for p in params])
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(optim.global_norm([p.grad for p in params]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_captured_and_replayed():
    params = _params([30001, 17, 9000], [torch.bfloat16, torch.float32])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.clip_grad_norm_(params, 1e9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(params, 1.0)
    for seed in range(1, 5):
        new = _params([30001, 17, 9000], [torch.bfloat16, torch.float32], seed=seed, scale=10.0 ** (seed - 3))
        for p, q in zip(params, new):
            p.grad.copy_(q.grad)
        want = optim.clip_grad_norm_(new, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(params, new))


@pytest.mark.parametrize("mixed", [False, True])
def test_the_engines_clip(mixed):
    """DDP's clip over its flat gradient (fp32, and bf16 under mixed precision) goes through the same kernels."""
    from distributed_training_amd.parallel.flat import build_flat_group, clip_flat_grad_norm_

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 7)).to(DEV)
    kw = dict(param_dtype=torch.bfloat16, grad_dtype=torch.bfloat16) if mixed else {}
    fg = build_flat_group(list(net.named_parameters()), torch.device(DEV, 0), **kw)
    fg.zero_grad()
    for p in net.parameters():
        p.grad.normal_()
    before = [p.grad.double().clone() for p in net.parameters()]
    want = math.sqrt(sum(float(b.square().sum()) for b in before))
    norm = clip_flat_grad_norm_(fg, 0.5)
    assert norm.shape == () and abs(float(norm) - want) <= 2.0 ** -23 * want
    for p, b in zip(net.parameters(), before):
        w = b * (0.5 / (want + 1e-6))
        assert ((p.grad.double() - w).abs() <= w.abs() * (oracle.half_step(p.grad.dtype) + 2.0 ** -22)).all()


def test_refusals_on_the_device():
    with pytest.raises(TypeError, match="gradient norm"):
        optim.global_norm([torch.ones(3, device=DEV, dtype=torch.int32)])
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_(_params([3], TYPES), -1.0)


def test_gradients_on_the_host_and_the_device():
    a, b = _params([100], [torch.float32])[0], torch.nn.Parameter(torch.zeros(50))
    b.grad = torch.full((50,), 2.0)
    want = math.sqrt(float(a.grad.double().square().sum()) + 200.0)
    before = a.grad.double()
    norm = optim.clip_grad_norm_([a, b], 1.0)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    assert torch.allclose(a.grad.double(), before / want, rtol=1e-6) and torch.allclose(b.grad, torch.full((50,), 2.0 / want), rtol=1e-6)


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_complex_gradients(dtype):
    """As their real and imaginary parts: dense, strided and conjugate ones beside real ones."""
    z = torch.randn(60, 70, dtype=dtype, generator=torch.Generator().manual_seed(0)).to(DEV)
    wide = z.clone()
    grads = [z[:, 20:50].contiguous(), wide[:, 1:3], z[:20].clone().conj(), z.real[0].float().contiguous()]
    before = [g.resolve_conj().clone() for g in grads]
    norm = math.sqrt(sum(float((b.abs().double() ** 2).sum()) for b in before))
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=DEV)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    for flag in (False, True):
        for g, b in zip(grads, before):
            g.copy_(b)
        got = optim.clip_grad_norm_(params + params[:1], 0.5, error_if_nonfinite=flag)
        # the oracle squares moduli that torch rounds to the parts' type (2 roundings of 2^-24 at most, halved by the root's mean)
        assert abs(float(got) - norm) <= 2.0 ** -22 * norm
        for p, b in zip(params, before):
            torch.testing.assert_close(p.grad.resolve_conj(), b * (0.5 / (norm + 1e-6)), rtol=2.0 ** -21, atol=0)
        assert torch.equal(wide[:, 3:], z[:, 3:]) and torch.equal(wide[:, :1], z[:, :1])


def test_a_coefficient_below_fp32():
    """Gradients near 1e37 clipped to a norm near 1 and below: the coefficient leaves fp32's normal numbers, the products do not.
    (fp32 coefficient and product, the sum of squares in 64 bits: 2^-24 each, and half a step of the type.)"""
    for dtype in (torch.float32, torch.bfloat16, torch.float64):
        for n in (100, 300007):
            base = (torch.rand(n, generator=torch.Generator().manual_seed(n)) + 0.5) * 1e37
            p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=DEV))
            before = base.to(dtype).to(DEV)
            norm = math.sqrt(float(before.double().square().sum()))
            for max_norm in (1.0, 1e-4):
                p.grad = before.clone()
                optim.clip_grad_norm_(p, max_norm)
                want = before.double() * (max_norm / (norm + 1e-6))
                step = 2.0 ** -40 if dtype == torch.float64 else oracle.half_step(dtype) * 1.01 + 3 * 2.0 ** -24
                assert ((p.grad.double() - want).abs() <= want * step).all(), (dtype, n, max_norm)
