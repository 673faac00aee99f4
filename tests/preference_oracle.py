"""64-bit forms of the preference-training losses, and how far a kernel's fp32 statistics and rounding may be from
them (used by test_preference_cpu.py and test_preference_gpu.py)."""
import math

import torch


def logprobs64(z, target, ignore_index=-100, temperature=1.0):
    """(log-probabilities, which positions count); ``z`` fp64."""
    V = z.shape[-1]
    live = (target != ignore_index) & (target >= 0) & (target < V)
    x = torch.where(live.unsqueeze(-1), z, torch.zeros_like(z)) / temperature
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    lp = lp.gather(-1, torch.where(live, target, torch.zeros_like(target)).unsqueeze(-1)).squeeze(-1)
    return torch.where(live, lp, torch.zeros_like(lp)), live


def policy64(z, target, old, adv, ref=None, clip=0.2, clip_high=None, kl_coef=0.0, reduction="token",
             ignore_index=-100, temperature=1.0, scale=1.0):
    """loss, log-probabilities, mean KL, clipped fraction -- term by term as the definition says."""
    lp, live = logprobs64(z, target, ignore_index, temperature)
    A = adv.double()
    A = (A.unsqueeze(-1) if A.dim() < target.dim() else A).expand(target.shape)
    hi, lo = 1.0 + (clip if clip_high is None else clip_high), 1.0 - clip
    zero = torch.zeros_like(lp)
    A, old = torch.where(live, A, zero), torch.where(live, old.double(), lp.detach())
    r = (lp - old).exp()
    up, down = (A > 0) & (r > hi), (A < 0) & (r < lo)
    each = -torch.where(up, hi * A, torch.where(down, lo * A, r * A))
    kl = zero
    if ref is not None:
        d = torch.where(live, ref.double(), lp.detach()) - lp
        kl = d.exp() - d - 1.0
        if kl_coef:
            each = each + kl_coef * kl
    n = max(1, int(live.sum()))
    if reduction == "token":
        loss = each.sum() / n
    else:
        loss = (each.sum(1) / live.sum(1).clamp(min=1)).sum() / target.shape[0]
    return loss * scale, lp, kl.detach().sum() / n, (up | down).sum() / n


def pairs64(z, target, ref=None, beta=0.1, label_smoothing=0.0, average=False, ignore_index=-100, scale=1.0):
    """loss, sequence log-probabilities, margins."""
    lp, live = logprobs64(z, target, ignore_index)
    L = lp.sum(1)
    if average:
        L = L / live.sum(1).clamp(min=1)
    gap = L if ref is None else L - ref.double()
    P = z.shape[0] // 2
    h = beta * (gap[:P] - gap[P:])
    sp = torch.nn.functional.softplus
    loss = ((1 - label_smoothing) * sp(-h, threshold=1000) + label_smoothing * sp(h, threshold=1000)).mean()
    return loss * scale, L, h


def stat_error(z, temperature=1.0):
    """Bound on the relative error of a row's sum of exponentials and probabilities, and so on the absolute error of its
    log-probability.  With u = 2^-24 and y = (z - M) c - log2 s the exponent of a term: the subtraction, c's own rounding,
    the multiplication and log2 s' rounding add at most 4 u |y| (plus u |log2 s|) to y, each times ln 2 < 1 in 2^y; the
    hardware exponential adds 2 u; a thread sums at most V / 256 + 32 terms in turn and the joins are under 32 more, u
    each.  Terms further than 30 nats below the maximum weigh under 1e-13 each and are left out of |y|'s range."""
    V = z.shape[-1]
    far = min(float((z.amax(-1) - z.amin(-1)).nan_to_num(0.0, 0.0, 0.0).max()) if z.numel() else 0.0, 30.0 * temperature)
    reach = far / temperature * 1.4427 + math.log2(V + 1)
    return 2.0 ** -24 * (5.0 * reach + 2.0 + V / 256 + 64.0)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the type's subnormal numbers."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2
