"""What is measured of the post-training operators: attention over packed sequences, token
log-probabilities through the output head, and the clipped policy loss through the output head.

``run`` computes an operator either in its plain form (elementary torch operations in fp32 or
fp64) or, where ``own`` is true, through the package's public entry points."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a handful of short prompts, a tiny model's heads: the call's own latency
        dict(name="attn_fwd_few", op="attention", train=False, dtype="fp16", tokens=77, seqs=5, hq=4, hk=2, d=64,
             tail=3, fused=True),
        # scoring a batch of prompts and answers (old / reference log-probabilities): forward only
        dict(name="attn_fwd_ragged", op="attention", train=False, dtype="bf16", tokens=4096, seqs=7, hq=32, hk=8, d=128,
             tail=0, fused=False),
        # many short sequences packed to an odd total, some of one token or none
        dict(name="attn_train_many", op="attention", train=True, dtype="fp16", tokens=5001, seqs=64, hq=4, hk=2, d=64,
             tail=7, fused=True),
        # a packed training batch
        dict(name="attn_train_ragged", op="attention", train=True, dtype="bf16", tokens=4096, seqs=9, hq=32, hk=8, d=128,
             tail=0, fused=False),
        # the benchmark's training sequence
        dict(name="attn_train_8k", op="attention", train=True, dtype="bf16", tokens=8192, seqs=1, hq=32, hk=8, d=128,
             tail=0, fused=False),
        # the longest single-GPU sequence of the benchmark, one rank's share of the heads
        dict(name="attn_train_16k", op="attention", train=True, dtype="bf16", tokens=16384, seqs=1, hq=8, hk=2, d=128,
             tail=0, fused=False),
        # scoring one short answer against the full vocabulary
        dict(name="logp_fwd_few", op="log_probs", train=False, dtype="bf16", rows=61, hidden=4096, vocab=151936),
        # scoring a batch of answers
        dict(name="logp_fwd_batch", op="log_probs", train=False, dtype="bf16", rows=4096, hidden=4096, vocab=151936),
        # log-probabilities with their gradient, a small head with an odd vocabulary
        dict(name="logp_train_small", op="log_probs", train=True, dtype="fp16", rows=1003, hidden=256, vocab=4099),
        # a micro-batch of a small policy
        dict(name="policy_small", op="policy", train=True, dtype="bf16", rows=517, hidden=1024, vocab=32000, seqs=6,
             per_sequence=True, kl=0.0),
        # a training step's loss, token mean, with the KL term
        dict(name="policy_tokens", op="policy", train=True, dtype="bf16", rows=2048, hidden=4096, vocab=151936, seqs=8,
             per_sequence=False, kl=0.05),
        # the same at a whole packed batch, averaged per sequence
        dict(name="policy_sequences", op="policy", train=True, dtype="bf16", rows=4096, hidden=4096, vocab=151936,
             seqs=13, per_sequence=True, kl=0.02),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "log_probs", "policy"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attention":
        d = rng.choice([64, 128, 128, 80])
        hk = rng.choice([1, 2, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 5])
        most = int(math.sqrt(32 * 8192 * 8192 / hq))
        tokens = _log_uniform(rng, 64, min(16384, most))
        return dict(op=op, train=rng.random() < 0.6, dtype=dtype, tokens=tokens, seqs=_log_uniform(rng, 1, 64), hq=hq,
                    hk=hk, d=d, tail=rng.choice([0, 0, 1, 13]), fused=rng.random() < 0.5)
    vocab = rng.choice([4096, 4099, 32000, 151936, _log_uniform(rng, 1000, 151936)])
    case = dict(op=op, dtype=dtype, rows=_log_uniform(rng, 64, 4096), hidden=8 * rng.randint(32, 512), vocab=vocab)
    if op == "log_probs":
        return dict(case, train=rng.random() < 0.5)
    return dict(case, train=True, seqs=rng.randint(1, 16), per_sequence=rng.random() < 0.5, kl=rng.choice([0.0, 0.05]))


def work(case):
    if case["op"] == "attention":
        lens = _lengths(case)
        pairs = sum(n * (n + 1) // 2 for n in lens)
        tokens = case["tokens"]
        flops = 4 * case["d"] * case["hq"] * pairs
        nbytes = 2 * tokens * case["d"] * (2 * case["hq"] + 2 * case["hk"])
        if case["train"]:
            flops += 10 * case["d"] * case["hq"] * pairs
            nbytes += 2 * tokens * case["d"] * (2 * case["hq"] + 2 * case["hk"])
        return {"bytes": nbytes, "flops": flops}
    n, h, v = case["rows"], case["hidden"], case["vocab"]
    flops = 2 * n * h * v * (3 if case["train"] else 1)
    nbytes = 2 * (n * h + v * h) * (2 if case["train"] else 1) + n * 12
    return {"bytes": nbytes, "flops": flops}


def _lengths(case):
    """Sequence lengths of an attention case, the same for every seed: a geometric-like spread with
    empty and one-token sequences among many, summing to tokens - tail."""
    total, b = case["tokens"] - case["tail"], case["seqs"]
    if b == 1:
        return [total]
    weights = [((37 * i + 11) % 29 + 1) ** 2 if i % 9 != 4 else 0 for i in range(b)]
    extra = [int(i % 9 == 7 and total >= b) for i in range(b)]
    share = total - sum(extra)
    lens = [share * w // sum(weights) * (1 - e) + e for w, e in zip(weights, extra)]
    lens[0] += total - sum(lens)
    return lens


# ----------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "attention":
        t, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        # q and k come out of a per-head RMS norm (unit root mean square) and RoPE; a learned norm
        # weight sharpens some heads
        qkv = torch.randn(t, hq + 2 * hk, d, generator=g, device="cuda")
        qkv[:, :hq + hk] /= qkv[:, :hq + hk].square().mean(-1, keepdim=True).sqrt()
        qkv[:, :hq] *= torch.rand(1, hq, 1, generator=g, device="cuda") * 2 + 0.5
        qkv = qkv.to(dtype)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        if not case["fused"]:  # three tensors of their own instead of views of one
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        state = dict(case=case, q=q, k=k, v=v, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        if case["train"]:
            state["dout"] = torch.randn(t, hq, d, generator=g, device="cuda").to(dtype)
            for name in "qkv":
                state[name] = state[name].detach().requires_grad_(True)
        return state
    n, h, v = case["rows"], case["hidden"], case["vocab"]
    # final-norm output against a 0.02-initialised head, rows of different sharpness
    hidden = torch.randn(n, h, generator=g, device="cuda")
    hidden *= (torch.rand(n, 1, generator=g, device="cuda") * 2.5 + 0.5) * (64.0 / math.sqrt(h))
    weight = torch.empty(v, h, dtype=dtype, device="cuda")
    weight.normal_(0.0, 0.02, generator=g)
    hidden = hidden.to(dtype)
    # tokens sampled from the policy itself (Gumbel argmax); every seventh position is prompt
    logits = hidden.float() @ weight.float().t()
    noise = torch.empty_like(logits).exponential_(generator=g).clamp_(min=1e-20).log_()
    target = (logits - noise).argmax(-1)
    del noise
    logp = logits.gather(-1, target[:, None])[:, 0].double() - torch.logsumexp(logits, -1).double()
    del logits
    target[::7] = -100
    state = dict(case=case, hidden=hidden, weight=weight, target=target)
    if case["train"]:
        hidden.requires_grad_(True)
        weight.requires_grad_(True)
    if case["op"] == "log_probs":
        state["dlogp"] = torch.randn(n, generator=g, device="cuda")
        return state
    # the policy that sampled is a few updates old; ratios are kept off the two clip borders, where a
    # rounding of either side would pick the other branch
    delta = 0.15 * torch.randn(n, generator=g, device="cuda").double()
    for border in (math.log(0.8), math.log(1.28)):
        near = (delta - border).abs() < 2e-3
        delta = torch.where(near, delta + 5e-3, delta)
    state["old"] = (logp - delta).float()
    # the policy has moved well away from its reference; a reward that rises above its lagging baseline
    # gives mostly positive advantages, one value per sequence
    state["ref"] = (logp + 0.5 * torch.randn(n, generator=g, device="cuda")).float()
    cu = torch.linspace(0, n, case["seqs"] + 1, device="cuda").round().to(torch.int32)
    state["cu"] = cu
    adv = 1.0 + 0.6 * torch.randn(case["seqs"], generator=g, device="cuda")
    state["adv"] = torch.repeat_interleave(adv, (cu[1:] - cu[:-1]).long()).contiguous()
    return state


# -------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _attention(state, case)
    if case["op"] == "log_probs":
        return _log_probs(state, case)
    return _policy(state, case)


def _attention(s, case):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"]
    if own:
        from bastile_b200.ops.packed_attention import pack_sequences, packed_attention

        seqs = pack_sequences(cu, case["tokens"])
        if not case["train"]:
            with torch.no_grad():
                return {"out": packed_attention(q, k, v, seqs)}
        out = packed_attention(q, k, v, seqs)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        t, hq, d = q.shape
        hk = k.shape[1]
        scale = d ** -0.5
        pos = torch.arange(t, device=q.device)
        seq = torch.searchsorted(cu[1:].long(), pos, right=True)
        mask = (seq[:, None] == seq[None, :]) & (pos[None, :] <= pos[:, None]) & (pos[:, None] < cu[-1])
        # [hk, group, t, d] against [hk, 1, t, d]
        qf = q.float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3)
        kf = k.float().permute(1, 0, 2)[:, None]
        vf = v.float().permute(1, 0, 2)[:, None]
        p = (qf @ kf.transpose(-1, -2)).mul_(scale).masked_fill_(~mask, float("-inf"))
        top = p.amax(-1, keepdim=True)
        p.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total == 0, torch.ones_like(total), total))
        of = p @ vf
        out = of.permute(2, 0, 1, 3).reshape(t, hq, d).to(q.dtype)
        if not case["train"]:
            return {"out": out}
        do = s["dout"].float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3)
        dv = (p.transpose(-1, -2) @ do).sum(1)
        ds = do @ vf.transpose(-1, -2)
        ds.sub_((do * of).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        del p
        dq = ds @ kf
        dk = (ds.transpose(-1, -2) @ qf).sum(1)
        return {"out": out, "dq": dq.permute(2, 0, 1, 3).reshape(t, hq, d).to(q.dtype),
                "dk": dk.transpose(0, 1).to(q.dtype), "dv": dv.transpose(0, 1).to(q.dtype)}


def _plain_logits(s):
    """fp32 logits, log-sum-exp and log-probabilities (0 at ignored positions)."""
    hf, wf = s["hidden"].float(), s["weight"].float()
    logits = hf @ wf.t()
    top = logits.amax(-1, keepdim=True)
    lse = (logits - top).exp().sum(-1, keepdim=True, dtype=torch.float64).log() + top
    live = s["target"] >= 0
    col = torch.where(live, s["target"], torch.zeros_like(s["target"]))[:, None]
    logp = torch.where(live, (logits.gather(-1, col).double() - lse)[:, 0], 0.0)
    return hf, wf, logits, lse, live, col, logp


def _plain_grads(s, hf, wf, logits, lse, live, col, coef):
    """Gradients of hidden and weight where d(loss)/d(logp) = coef."""
    coef = torch.where(live, coef, torch.zeros_like(coef)).float()[:, None]
    dlogits = logits.sub_(lse.float()).exp_().mul_(-coef)
    dlogits.scatter_add_(1, col, coef)
    return (dlogits @ wf).to(s["hidden"].dtype), (dlogits.t() @ hf).to(s["weight"].dtype)


def _log_probs(s, case):
    if own:
        from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs

        if not case["train"]:
            with torch.no_grad():
                return {"logp": fused_linear_log_probs(s["hidden"], s["weight"], s["target"])}
        logp = fused_linear_log_probs(s["hidden"], s["weight"], s["target"])
        dh, dw = torch.autograd.grad(logp, (s["hidden"], s["weight"]), s["dlogp"])
        return {"logp": logp.detach(), "dhidden": dh, "dweight": dw}
    with torch.no_grad():
        hf, wf, logits, lse, live, col, logp = _plain_logits(s)
        if not case["train"]:
            return {"logp": logp.float()}
        dh, dw = _plain_grads(s, hf, wf, logits, lse, live, col, s["dlogp"])
        return {"logp": logp.float(), "dhidden": dh, "dweight": dw}


def _policy(s, case):
    if own:
        from bastile_b200.ops.fused_linear_policy_loss import fused_linear_policy_loss

        got = fused_linear_policy_loss(s["hidden"], s["weight"], s["target"], s["old"], s["adv"],
                                       ref_log_probs=s["ref"] if case["kl"] else None, clip_low=0.2, clip_high=0.28,
                                       kl_coef=case["kl"], cu_seqlens=s["cu"] if case["per_sequence"] else None)
        dh, dw = torch.autograd.grad(got.loss, (s["hidden"], s["weight"]))
        return {"loss": got.loss.detach(), "logp": got.log_probs, "kl": got.kl, "dhidden": dh, "dweight": dw}
    with torch.no_grad():
        hf, wf, logits, lse, live, col, logp = _plain_logits(s)
        w = live.double()
        if case["per_sequence"]:
            seq = torch.searchsorted(s["cu"][1:].long(), torch.arange(len(live), device=live.device), right=True)
            count = torch.zeros(case["seqs"], dtype=torch.float64, device=live.device).index_add_(0, seq, w)
            w = w / count.clamp(min=1.0)[seq] / (count > 0).sum()
        else:
            w = w / w.sum()
        adv = s["adv"].double()
        ratio = (logp - s["old"].double()).exp()
        held = ratio.clamp(0.8, 1.28)
        coef = torch.where(ratio * adv <= held * adv, -adv * ratio, torch.zeros_like(adv))
        terms = -torch.minimum(ratio * adv, held * adv)
        kl = torch.zeros_like(terms)
        if case["kl"]:
            gap = s["ref"].double() - logp
            kl = gap.exp() - gap - 1
            terms = terms + case["kl"] * kl
            coef = coef + case["kl"] * (1 - gap.exp())
        zero = torch.zeros_like(terms)
        loss = (torch.where(live, terms, zero) * w).sum()
        mean_kl = (torch.where(live, kl, zero) * w).sum()
        dh, dw = _plain_grads(s, hf, wf, logits, lse, live, col, coef * w)
        return {"loss": loss.float(), "logp": logp.float(), "kl": mean_kl.float(), "dhidden": dh, "dweight": dw}


# --------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if case["op"] == "attention":
            q, k, v = (s[n].detach().to(f64) for n in "qkv")
            group = q.shape[1] // k.shape[1]
            out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
            ends = s["cu"].tolist()
            for a, b in zip(ends[:-1], ends[1:]):
                if b == a:
                    continue
                upper = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu_(1)
                for head in range(q.shape[1]):
                    kv = head // group
                    z = torch.einsum("id,jd->ij", q[a:b, head], k[a:b, kv]) / math.sqrt(case["d"])
                    prob = torch.softmax(z.masked_fill_(upper, -math.inf), dim=1)
                    out[a:b, head] = prob @ v[a:b, kv]
                    if case["train"]:
                        do = s["dout"][a:b, head].to(f64)
                        dv[a:b, kv] += prob.t() @ do
                        dprob = do @ v[a:b, kv].t()
                        dz = prob * (dprob - (prob * dprob).sum(1, keepdim=True)) / math.sqrt(case["d"])
                        dq[a:b, head] = dz @ k[a:b, kv]
                        dk[a:b, kv] += dz.t() @ q[a:b, head]
            return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"out": out}
        x, w = s["hidden"].detach().to(f64), s["weight"].detach().to(f64)
        z = torch.log_softmax(x @ w.t(), dim=1)
        use = s["target"] != -100
        rows = use.nonzero()[:, 0]
        token = s["target"][rows]
        logp = torch.zeros(len(use), dtype=f64, device=x.device)
        logp[rows] = z[rows, token]
        if not case["train"]:
            return {"logp": logp}
        got = {"logp": logp}
        slope = torch.zeros_like(logp)
        if case["op"] == "log_probs":
            slope[rows] = s["dlogp"][rows].to(f64)
        else:
            share = torch.zeros_like(logp)
            if case["per_sequence"]:
                ends = s["cu"].tolist()
                spans = [use[a:b] for a, b in zip(ends[:-1], ends[1:])]
                filled = sum(bool(span.any()) for span in spans)
                for (a, b), span in zip(zip(ends[:-1], ends[1:]), spans):
                    share[a:b] = span.to(f64) / max(1, int(span.sum())) / filled
            else:
                share = use.to(f64) / int(use.sum())
            a = s["adv"].to(f64)
            r = torch.exp(logp - s["old"].to(f64))
            over = ((a > 0) & (r > 1.28)) | ((a < 0) & (r < 0.8))
            bound = torch.where(a > 0, torch.full_like(r, 1.28), torch.full_like(r, 0.8))
            value = -a * torch.where(over, bound, r)
            slope = torch.where(over, torch.zeros_like(r), -a * r)
            kl = torch.zeros_like(r)
            if case["kl"]:
                gap = s["ref"].to(f64) - logp
                kl = torch.expm1(gap) - gap
                value = value + case["kl"] * kl
                slope = slope - case["kl"] * torch.expm1(gap)
            got["loss"] = torch.dot(value, share)
            got["kl"] = torch.dot(kl, share)
            slope = slope * share
        z.exp_().mul_(-slope[:, None])
        z[rows, token] += slope[rows]
        got["dhidden"], got["dweight"] = z @ w, z.t() @ x
        return got
