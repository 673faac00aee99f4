"""The workloads that the preference-training operators are timed on: token log-probabilities, the clipped
policy loss, the paired preference loss (each forward and backward) and global-norm gradient clipping.

``own`` false: the plain form in elementary torch operations.  ``own`` true: the framework's operators, called as
a training program calls them.  ``exact`` computes the same outputs in 64 bits.
"""
import math

import torch

own = False

VOCAB_GPT2, VOCAB_GPT2_PADDED, VOCAB_LLAMA = 50257, 50304, 128256
MOST = 4 * 1024 * VOCAB_LLAMA  # logits of the largest listed loss case; no drawn case has more
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # scoring one short sample with GPT-2's unpadded vocabulary: rows that begin at odd addresses, latency counts
        dict(name="logprobs_one_sample", op="logprobs", B=1, S=64, V=VOCAB_GPT2, dtype="bf16", temperature=0.7),
        # a GPT-2 batch (8 x 1024) scored with a gradient, e.g. for a reward-weighted likelihood
        dict(name="logprobs_gpt2", op="logprobs", B=8, S=1024, V=VOCAB_GPT2_PADDED, dtype="bf16", temperature=1.0),
        # Llama-3 logits kept in fp32, an odd number of tokens
        dict(name="logprobs_llama_fp32", op="logprobs", B=1, S=1999, V=VOCAB_LLAMA, dtype="fp32", temperature=1.0),
        # a toy policy, as in a unit test or a small control task: latency only
        dict(name="policy_toy", op="policy", B=4, S=16, V=1003, dtype="fp32", kl=0.05, high=0.2, reduction="token"),
        # a GPT-2 policy update: 8 samples of 1024 with their prompts masked, KL to a reference
        dict(name="policy_gpt2", op="policy", B=8, S=1024, V=VOCAB_GPT2_PADDED, dtype="bf16", kl=0.02, high=0.2,
             reduction="token"),
        # a group of Llama-3 samples, wider upper clip, no reference model, mean over sequences
        dict(name="policy_llama", op="policy", B=4, S=1024, V=VOCAB_LLAMA, dtype="bf16", kl=0.0, high=0.28,
             reduction="sequence"),
        # two pairs of short answers, fp16 logits, odd vocabulary and length
        dict(name="preference_short", op="preference", B=4, S=33, V=VOCAB_GPT2, dtype="fp16", smoothing=0.0,
             average=False, ref=True),
        # four GPT-2 pairs of full length
        dict(name="preference_gpt2", op="preference", B=8, S=1024, V=VOCAB_GPT2_PADDED, dtype="bf16", smoothing=0.1,
             average=False, ref=True),
        # two Llama-3 pairs, length-normalised and without a reference model
        dict(name="preference_llama", op="preference", B=4, S=1000, V=VOCAB_LLAMA, dtype="bf16", smoothing=0.0,
             average=True, ref=False),
        # the two-layer MLP's four gradients (20 -> 512 -> 1): latency only
        dict(name="clip_mlp", op="clip", model="mlp", layers=2, width=512, vocab=0, dtype="fp32"),
        # GPT-2 small's 148 gradients in bf16, the norms' in fp32
        dict(name="clip_gpt2", op="clip", model="gpt2", layers=12, width=768, vocab=VOCAB_GPT2_PADDED, dtype="bf16"),
        # the embedding and four blocks of Llama-3 8B: 1.4 G elements
        dict(name="clip_llama", op="clip", model="llama", layers=4, width=4096, vocab=VOCAB_LLAMA, dtype="bf16"),
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm of the range."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "clip"])
    if op == "clip":
        model = rng.choice(["mlp", "gpt2", "llama"])
        width = 8 * _between(rng, 4, 256)
        return dict(op=op, model=model, layers=rng.randint(1, 12), width=width,
                    vocab=_between(rng, 500, 60000), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    V = rng.choice([_between(rng, 500, VOCAB_LLAMA), _between(rng, 500, VOCAB_LLAMA), VOCAB_GPT2, VOCAB_LLAMA])
    B = 2 * rng.randint(1, 6)
    S = _between(rng, 32, max(33, min(2048, MOST // (B * V))))
    case = dict(op=op, B=B, S=S, V=V, dtype=rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"]))
    if op == "logprobs":
        case.update(temperature=rng.choice([1.0, 0.6, 1.3]))
    elif op == "policy":
        case.update(kl=rng.choice([0.0, 0.02, 0.1]), high=rng.choice([0.2, 0.28]),
                    reduction=rng.choice(["token", "sequence"]))
    else:
        average = rng.random() < 0.5
        # (summed log-probabilities of unequal lengths are compared against a reference model's only)
        case.update(smoothing=rng.choice([0.0, 0.1]), average=average, ref=not average or rng.random() < 0.5)
    return case


# ------------------------------------------------------------------ inputs
def _shapes(case):
    """(the model's parameter shapes, whether each is a norm's: those gradients are kept in fp32)."""
    C, n = case["width"], case["layers"]
    if case["model"] == "mlp":
        return [([C, 20], False), ([C], False)] + [([C, C], False), ([C], False)] * (n - 2) + [([1, C], False), ([1], False)]
    if case["model"] == "gpt2":
        block = [([C], True), ([C], True), ([3 * C, C], False), ([3 * C], False), ([C, C], False), ([C], False),
                 ([C], True), ([C], True), ([4 * C, C], False), ([4 * C], False), ([C, 4 * C], False), ([C], False)]
        return [([case["vocab"], C], False), ([1024, C], False)] + block * n + [([C], True), ([C], True)]
    block = [([C], True), ([C + C // 2, C], False), ([C, C], False), ([C], True), ([7 * C, C], False),
             ([C, 7 * C // 2], False)]
    return [([case["vocab"], C], False)] + block * n + [([C], True)]


def _clip_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, shapes = TYPES[case["dtype"]], _shapes(case)
    total = {False: sum(math.prod(s) for s, norm in shapes if not norm),
             True: sum(math.prod(s) for s, norm in shapes if norm)}
    flat = {}
    for norm, kind in ((False, dtype), (True, torch.float32)):
        # gradients of a step: mostly small, a heavier tail in the norms' scales
        flat[norm] = torch.empty(total[norm], device="cuda", dtype=kind).normal_(0.0, 3e-2 if norm else 1e-2, generator=gen)
    at, params = {False: 0, True: 0}, []
    for shape, norm in shapes:  # each gradient is its slice of the flat buffer, at whatever address that is
        count = math.prod(shape)
        g = flat[norm][at[norm]:at[norm] + count].view(shape)
        at[norm] += count
        p = torch.nn.Parameter(torch.zeros((), device="cuda", dtype=g.dtype).expand(shape), requires_grad=True)
        p.grad = g
        params.append(p)
    norm = math.sqrt(total[False] * 1e-2 ** 2 + total[True] * 3e-2 ** 2)
    # (clipping changes the gradients in place: the bound shrinks a little with each pass, so that every pass clips)
    return dict(params=params, grads=[flat[False]] + ([flat[True]] if total[True] else []), max_norm=0.37 * norm)


def _loss_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, S, V = case["B"], case["S"], case["V"]
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    target = torch.randint(V, (B, S), device="cuda", generator=gen)
    logits = torch.empty(B, S, V, device="cuda", dtype=TYPES[case["dtype"]]).normal_(0.0, 2.0, generator=gen)
    # a sampled token is mostly a likely one
    sampled = (math.log(V) + 1.0 + 1.5 * rand(B, S, 1)).to(logits.dtype)
    logits.scatter_(2, target.unsqueeze(2), sampled)
    x = logits.detach()
    temperature = case.get("temperature", 1.0)
    lp = torch.empty(B, S, device="cuda")
    for b in range(B):  # a row's statistics in fp32, one sequence at a time
        z = x[b].float() / temperature
        lp[b] = (z.gather(1, target[b].unsqueeze(1)) - torch.logsumexp(z, 1, keepdim=True)).squeeze(1)
    if case["op"] != "logprobs":
        # the prompt in front and the padding behind carry no loss; some sequences are all answer
        at = torch.arange(S, device="cuda")
        first = (torch.rand(B, 1, device="cuda", generator=gen) * 0.3 * S).long()
        last = S - (torch.rand(B, 1, device="cuda", generator=gen) * 0.2 * S).long()
        target = torch.where((at >= first) & (at < last), target, torch.full_like(target, -100))
    state = dict(logits=logits, target=target)
    if case["op"] == "logprobs":
        state["weight"] = rand(B, S) / (B * S)
    elif case["op"] == "policy":
        # log-ratios in steps of 1/64: none lies within rounding of the clip's borders (log 1.2, log 0.8, log 1.28),
        # where the gradient jumps and two right answers differ by a whole row
        state["old_logp"] = lp - torch.round(0.12 * 64 * rand(B, S)) / 64
        state["advantages"] = 0.4 + rand(B)
        if case["kl"]:
            state["ref_logp"] = lp + torch.round(0.25 * 64 * rand(B, S)) / 64
    elif case["ref"]:
        live = target != -100
        total = (lp * live).double().sum(1)
        shift = (0.3 if case["average"] else 0.3 * math.sqrt(S)) * rand(B).double()
        state["ref_logp"] = ((total / live.sum(1).clamp(min=1) if case["average"] else total) + shift).float()
    return state


def prepare(case, seed):
    state = _clip_inputs(case, seed) if case["op"] == "clip" else _loss_inputs(case, seed)
    if case["op"] != "clip":
        state["logits"].requires_grad_()
    state["case"] = case
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return {"logprobs": _logprobs, "policy": _policy, "preference": _preference, "clip": _clip}[state["case"]["op"]](state)


def _beta(case):
    return 2.0 if case["average"] else 0.1


def _row_terms(state, temperature=1.0):
    """Plain: (the tokens' log-probabilities in 64 bits, the softmax, which rows count, the targets to index with)."""
    live = state["target"] != -100
    at = torch.where(live, state["target"], 0).unsqueeze(2)
    x = state["logits"].detach().float()
    if temperature != 1.0:
        x = x / temperature
    top = x.amax(2, keepdim=True)
    chosen = (x.gather(2, at) - top).double()
    x = torch.exp(x - top)
    total = x.sum(2, keepdim=True)
    lp = (chosen - torch.log(total.double())).squeeze(2)
    return torch.where(live, lp, 0.0), x.div_(total), live, at


def _logits_gradient(softmax, at, coefficient, dtype):
    """Plain: coefficient (onehot - softmax), rounded once; the coefficients are 0 where a row does not count."""
    softmax.neg_()
    softmax.scatter_add_(2, at, torch.ones_like(at, dtype=softmax.dtype))
    return softmax.mul_(coefficient.float().unsqueeze(2)).to(dtype)


def _logprobs(state):
    logits, case = state["logits"], state["case"]
    if own:
        from distributed_training_amd.ops.preference import token_logprobs

        lp = token_logprobs(logits, state["target"], temperature=case["temperature"])
        (grad,) = torch.autograd.grad(lp, logits, state["weight"])
        return {"logp": lp.detach(), "grad": grad}
    lp, p, live, at = _row_terms(state, case["temperature"])
    return {"logp": lp.float(), "grad": _logits_gradient(p, at, state["weight"] / case["temperature"], logits.dtype)}


def _policy(state):
    logits, case = state["logits"], state["case"]
    if own:
        from distributed_training_amd.ops.preference import policy_loss

        out = policy_loss(logits, state["target"], state["old_logp"], state["advantages"], ref_logp=state.get("ref_logp"),
                          clip=0.2, clip_high=case["high"], kl_coef=case["kl"], reduction=case["reduction"])
        (grad,) = torch.autograd.grad(out.loss, logits)
        return {"loss": out.loss.detach(), "logp": out.logp, "kl": out.kl, "clip_fraction": out.clip_fraction, "grad": grad}
    lp, p, live, at = _row_terms(state)
    A = state["advantages"].double().unsqueeze(1)
    ratio = torch.exp(lp - state["old_logp"].double())
    clipped = live & (((A > 0) & (ratio > 1.0 + case["high"])) | ((A < 0) & (ratio < 0.8)))
    loss = -torch.minimum(ratio * A, ratio.clamp(0.8, 1.0 + case["high"]) * A)
    slope = torch.where(clipped, 0.0, -ratio * A)
    tokens = live.sum()
    if case["kl"]:
        d = state["ref_logp"].double() - lp
        k3 = torch.expm1(d) - d
        kl = torch.where(live, k3, 0.0).sum() / tokens
        loss, slope = loss + case["kl"] * k3, slope - case["kl"] * torch.expm1(d)
    else:
        kl = torch.zeros((), device=logits.device)
    if case["reduction"] == "token":
        weight = live / tokens.double()
    else:
        weight = live / live.sum(1, keepdim=True).clamp(min=1).double() / case["B"]
    return {"loss": torch.where(live, loss * weight, 0.0).sum().float(), "logp": lp.float(), "kl": kl.float(),
            "clip_fraction": (clipped.sum() / tokens).float(),
            "grad": _logits_gradient(p, at, torch.where(live, slope * weight, 0.0), logits.dtype)}


def _preference(state):
    logits, case = state["logits"], state["case"]
    if own:
        from distributed_training_amd.ops.preference import preference_loss

        out = preference_loss(logits, state["target"], ref_logp=state.get("ref_logp"), beta=_beta(case),
                              label_smoothing=case["smoothing"], average=case["average"])
        (grad,) = torch.autograd.grad(out.loss, logits)
        return {"loss": out.loss.detach(), "logp": out.logp, "margin": out.margin, "grad": grad}
    lp, p, live, at = _row_terms(state)
    P, share = case["B"] // 2, live.double()
    if case["average"]:
        share = share / live.sum(1, keepdim=True).clamp(min=1)
    total = (lp * share).sum(1)
    gap = total - state["ref_logp"].double() if "ref_logp" in state else total
    h = _beta(case) * (gap[:P] - gap[P:])
    e = case["smoothing"]
    loss = (1 - e) * torch.log1p(torch.exp(-h.abs())) + e * torch.log1p(torch.exp(-h.abs()))
    loss = (loss + (1 - e) * torch.clamp(-h, min=0) + e * torch.clamp(h, min=0)).mean()
    slope = _beta(case) / P * (1 / (1 + torch.exp(-h)) - (1 - e))
    slope = torch.cat([slope, -slope]).unsqueeze(1) * share
    return {"loss": loss.float(), "logp": total.float(), "margin": h.float(),
            "grad": _logits_gradient(p, at, slope, logits.dtype)}


def _clip(state):
    bound = state["max_norm"]
    state["max_norm"] = 0.999 * bound
    if own:
        from distributed_training_amd.ops.optim import clip_grad_norm_

        norm = clip_grad_norm_(state["params"], bound)
        return {"norm": norm, "grads": state["grads"]}
    # (every gradient is a slice of one of the flat buffers: a few passes over those, not over each of them)
    norm = torch.stack([g.float().square().sum() for g in state["grads"]]).double().sum().sqrt()
    factor = (bound / (norm + 1e-6)).clamp(max=1.0).float()
    for g in state["grads"]:
        g.copy_(g.float() * factor)
    return {"norm": norm.float(), "grads": state["grads"]}


# ------------------------------------------------------------------ floors and 64 bits
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "clip":
        bytes_ = sum(math.prod(s) * (4 if norm else size) for s, norm in _shapes(case))
        return {"bytes": 2 * bytes_, "flops": 3 * sum(math.prod(s) for s, _ in _shapes(case))}
    N, V = case["B"] * case["S"], case["V"]
    # logits read once and their gradient written once; a few numbers a token
    return {"bytes": 2 * N * V * size + 24 * N, "flops": 8 * N * V}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        grads = [g.double() for g in state["grads"]]
        norm = math.sqrt(sum((g * g).sum().item() for g in grads))
        factor = min(1.0, state["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g.mul_(factor) for g in grads]}
    z = state["logits"].detach().double().requires_grad_()
    target = state["target"]
    live = target != -100
    logp = torch.log_softmax(z / case.get("temperature", 1.0), -1)
    lp = logp.gather(-1, target.clamp(min=0).unsqueeze(-1)).squeeze(-1) * live
    del logp
    if case["op"] == "logprobs":
        (grad,) = torch.autograd.grad(lp, z, state["weight"].double())
        return {"logp": lp.detach(), "grad": grad}
    if case["op"] == "policy":
        A = state["advantages"].double()[:, None].expand_as(lp)
        logratio = (lp - state["old_logp"].double()) * live
        surrogate = torch.min(logratio.exp() * A, logratio.exp().clamp(1 - 0.2, 1 + case["high"]) * A)
        shift = (state["ref_logp"].double() - lp) * live if "ref_logp" in state else torch.zeros_like(lp)
        kl = torch.expm1(shift) - shift
        each = (kl * case["kl"] - surrogate) * live
        clipped = ((logratio.exp() * A) > surrogate) & live
        if case["reduction"] == "token":
            loss = each.sum() / live.sum()
        else:
            loss = (each.sum(1) / live.sum(1).clamp(min=1)).mean()
        (grad,) = torch.autograd.grad(loss, z)
        count = live.sum().double()
        return {"loss": loss.detach(), "logp": lp.detach(), "kl": (kl.detach() * live).sum() / count,
                "clip_fraction": clipped.sum() / count, "grad": grad}
    total = lp.sum(1) / (live.sum(1).clamp(min=1) if case["average"] else 1)
    gap = total - (state["ref_logp"].double() if "ref_logp" in state else 0.0)
    h = _beta(case) * (gap[: case["B"] // 2] - gap[case["B"] // 2:])
    e = case["smoothing"]
    loss = -((1 - e) * torch.nn.functional.logsigmoid(h) + e * torch.nn.functional.logsigmoid(-h)).mean()
    (grad,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "logp": total.detach(), "margin": h.detach(), "grad": grad}
