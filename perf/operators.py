"""Cases that measure the post-training objectives: token log-probabilities through the LM head, the clipped policy
loss, the preference loss and distillation from a teacher's top logits.

Each case runs either a plain statement of the formula in elementary torch operations (fp32) or, with ``own`` set,
the framework's operator; ``exact`` states the definition once more in 64 bits.
"""
import math

import torch

own = False

V_QWEN = 151936  # vocabulary of the framework's Qwen3 configurations


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token scored against a 1024-wide head: the latency of reading the head once
        dict(name="score_one_token", op="score", T=1, H=1024, V=V_QWEN, tau=1.0, ignored=0.0),
        # a ragged batch of completions, odd vocabulary, sampling temperature below one
        dict(name="score_ragged_odd_vocab", op="score", T=1237, H=2048, V=32003, tau=0.7, ignored=0.25),
        # the reference policy's pass over one training batch (4 x 2048 tokens)
        dict(name="score_batch", op="score", T=8192, H=1024, V=V_QWEN, tau=1.0, ignored=0.2),
        # the policy's own pass over that batch, with the gradients of hidden states and head
        dict(name="train_batch", op="train", T=8192, H=1024, V=V_QWEN, tau=1.0, ignored=0.2),
        # a short micro-batch on a wide head: few rows, long reductions over the vocabulary
        dict(name="train_few_rows_wide", op="train", T=333, H=4096, V=V_QWEN, tau=1.0, ignored=0.1),
        # policy loss of one small rollout group, token mean, with a KL term
        dict(name="policy_small", op="policy", B=8, S=509, reduction="token", ref=True, adv="sequence"),
        # policy loss of a whole rollout batch, sequence mean, advantages per token
        dict(name="policy_large", op="policy", B=512, S=4096, reduction="sequence", ref=True, adv="token"),
        # preference loss of a few pairs
        dict(name="preference_small", op="preference", P=4, S=300, ref=True, average=False, smoothing=0.0),
        # preference loss of a large batch of long pairs, smoothed labels
        dict(name="preference_large", op="preference", P=256, S=4096, ref=True, average=False, smoothing=0.1),
        # distillation of a handful of positions from eight teacher logits
        dict(name="distill_few_rows", op="distill", T=17, V=V_QWEN, K=8, tau=1.0, dtype="bf16"),
        # distillation of a training batch from 64 teacher logits, softened
        dict(name="distill_batch", op="distill", T=8192, V=V_QWEN, K=64, tau=2.0, dtype="bf16"),
        # fp32 logits of an odd vocabulary: rows that start at any 4-byte address
        dict(name="distill_fp32_odd", op="distill", T=1021, V=32003, K=20, tau=1.5, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "train", "policy", "preference", "distill"])
    if op in ("score", "train"):
        H = rng.choice([256, 640, 1024, 1536, 2048, 2560, 4096])
        V = rng.choice([V_QWEN, 32003, 50257, 128256, _log_int(rng, 1000, 150000)])
        T = _log_int(rng, 1, min(8192, 8192 * 1024 * V_QWEN // (H * V)))
        return dict(op=op, T=T, H=H, V=V, tau=rng.choice([1.0, 1.0, 0.7, 1.3]), ignored=rng.choice([0.0, 0.1, 0.5]))
    if op == "policy":
        S = _log_int(rng, 1, 8192)
        B = _log_int(rng, 1, min(2048, 512 * 4096 // S))
        return dict(op=op, B=B, S=S, reduction=rng.choice(["token", "sequence"]), ref=rng.choice([True, False]),
                    adv=rng.choice(["token", "sequence"]))
    if op == "preference":
        S = _log_int(rng, 1, 8192)
        P = _log_int(rng, 1, min(1024, 256 * 4096 // S))
        return dict(op=op, P=P, S=S, ref=rng.choice([True, True, False]), average=rng.choice([False, True]),
                    smoothing=rng.choice([0.0, 0.1]))
    dtype = rng.choice(["bf16", "fp32"])
    V = rng.choice([V_QWEN, 32003, 50257, 128256, _log_int(rng, 1000, 150000)])
    T = _log_int(rng, 1, min(8192, 8192 * V_QWEN // (V * (2 if dtype == "fp32" else 1))))
    return dict(op=op, T=T, V=V, K=_log_int(rng, 1, 128), tau=rng.choice([1.0, 2.0, 1.5]), dtype=dtype)


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    op = case["op"]
    if op in ("score", "train"):
        # unit-RMS hidden states (the final norm's output) and a head that gives logits of standard deviation 2.5;
        # most tokens are pulled towards their id, so that log-probabilities run from about -15 to 0
        T, H, V = case["T"], case["H"], case["V"]
        w = (randn(V, H) * (2.5 / math.sqrt(H))).to(torch.bfloat16)
        ids = torch.randint(0, V, (T,), device=dev, generator=gen)
        h = (randn(T, H) + (10.0 * rand(T, 1)) * (w[ids].float() / 2.5)).to(torch.bfloat16)
        ids = ids.masked_fill(rand(T) < case["ignored"], -100)  # prompt and padding positions
        inp = dict(h=h, w=w, ids=ids)
        if op == "train":
            inp["g"] = randn(T) / T  # what a loss sends back: advantages or pair weights over the token count
        return inp
    if op in ("policy", "preference"):
        B, S = (case["B"], case["S"]) if op == "policy" else (2 * case["P"], case["S"])
        logp = 1.2 * rand(B, S).clamp_min(1e-6).log()  # minus an exponential of mean 1.2
        # a prompt in front, padding behind; a row in ten has no token that counts
        pos = torch.arange(S, device=dev)[None, :]
        start = (rand(B, 1) * S * 0.3).long()
        stop = start + 1 + (rand(B, 1) * S).long()
        mask = (pos >= start) & (pos < stop) & (rand(B, 1) >= 0.1)
        if op == "policy":
            d = 0.15 * randn(B, S)  # log ratio to the policy that sampled
            # the gradient jumps where the ratio meets a clip edge: stay 1e-3 clear of both
            for edge in (math.log(0.8), math.log(1.28)):
                d = torch.where((d - edge).abs() < 1e-3, torch.full_like(d, edge + 2e-3), d)
            adv = randn(B, S) if case["adv"] == "token" else randn(B, 1)
            return dict(logp=logp, old=logp - d, adv=adv, mask=mask,
                        ref=logp + 0.3 * randn(B, S) if case["ref"] else None)
        return dict(logp=logp, mask=mask, ref=logp + 0.05 * randn(B, S) if case["ref"] else None)
    # student logits around a teacher that ranks some tokens high; the last entries of some rows are absent
    T, V, K = case["T"], case["V"], case["K"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = randn(T, V) * 2.5
    top = (6.0 + 5.0 * rand(T, K)).sort(dim=1, descending=True).values
    # K different ids a row: a random start and equal steps through the vocabulary
    start = torch.randint(0, V, (T, 1), device=dev, generator=gen)
    ids = (start + torch.arange(K, device=dev)[None, :] * max(1, V // (K + 1))) % V
    logits.scatter_add_(1, ids, 0.9 * top)
    have = 1 + (rand(T, 1) * 1.5 * K).long()
    ids = ids.masked_fill(torch.arange(K, device=dev)[None, :] >= have, -1)
    return dict(logits=logits.to(dt), top=top, ids=ids, mask=rand(T) >= 0.1)


CLIP_LOW, CLIP_HIGH, KL_COEF, BETA = 0.2, 0.28, 0.05, 0.1


def prepare(case, seed):
    inp = _inputs(case, seed)
    if own:
        for name in {"train": ("h", "w"), "policy": ("logp",), "preference": ("logp",),
                     "distill": ("logits",)}.get(case["op"], ()):
            inp[name].requires_grad_(True)
    return dict(case=case, **inp)


# ------------------------------------------------------------------ one pass
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from parallel_b200.ops import objectives as O

    c = s["case"]
    op = c["op"]
    if op == "score":
        with torch.no_grad():
            return [O.lm_head_log_probs(s["h"], s["w"], s["ids"], temperature=c["tau"])]
    if op == "train":
        logp = O.lm_head_log_probs(s["h"], s["w"], s["ids"], temperature=c["tau"])
        return [logp.detach(), *torch.autograd.grad(logp, (s["h"], s["w"]), s["g"])]
    if op == "policy":
        out = O.policy_loss(s["logp"], s["old"], s["adv"], mask=s["mask"], ref_logp=s["ref"], clip_low=CLIP_LOW,
                            clip_high=CLIP_HIGH, kl_coef=KL_COEF, reduction=c["reduction"])
        return [out.loss.detach(), out.clip_fraction, out.kl, *torch.autograd.grad(out.loss, s["logp"])]
    if op == "preference":
        out = O.preference_loss(s["logp"], ref_logp=s["ref"], mask=s["mask"], beta=BETA,
                                label_smoothing=c["smoothing"], average=c["average"])
        return [out.loss.detach(), out.rewards, *torch.autograd.grad(out.loss, s["logp"])]
    loss = O.distillation_loss(s["logits"], s["top"], s["ids"], mask=s["mask"], temperature=c["tau"])
    return [loss.detach(), *torch.autograd.grad(loss, s["logits"])]


@torch.no_grad()
def _plain(s):
    c = s["case"]
    op = c["op"]
    if op in ("score", "train"):
        h, w, ids = s["h"].float(), s["w"].float(), s["ids"]
        valid = ids >= 0
        at = ids.clamp_min(0)[:, None]
        x = h @ w.t()
        # logp = -log(1 + sum over the other tokens of exp(l_v - l_id)): it keeps its digits where id is nearly
        # certain, given that l_id, which all of it hangs on, is summed on its own
        x -= (h * w[at[:, 0]]).sum(1, keepdim=True)
        x /= c["tau"]
        e = x.exp().scatter_(1, at, 0.0)
        logp = -torch.log1p(e.sum(1))
        logp = torch.where(valid, logp, torch.zeros_like(logp))
        if op == "score":
            return [logp]
        coef = torch.where(valid, s["g"] / c["tau"], torch.zeros_like(logp))[:, None]
        dl = e.mul_(-coef * logp[:, None].exp())
        dl.scatter_(1, at, -coef * torch.expm1(logp)[:, None])
        return [logp, (dl @ w).to(s["h"].dtype), (dl.t() @ h).to(s["w"].dtype)]
    if op == "policy":
        m = s["mask"]
        zero = torch.zeros_like(s["logp"])
        ratio = (s["logp"] - s["old"]).exp()
        u = ratio * s["adv"]
        cl = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * s["adv"]
        per = -torch.minimum(u, cl)
        grad = torch.where(u <= cl, -u, zero)
        kl = zero
        if s["ref"] is not None:
            r = s["ref"] - s["logp"]
            kl = r.exp() - r - 1
            per = per + KL_COEF * kl
            grad = grad + KL_COEF * (1 - r.exp())
        n = m.sum().clamp_min(1)
        if c["reduction"] == "token":
            wt = (1.0 / n).expand(m.shape)
        else:
            rows = m.sum(1, keepdim=True)
            wt = 1.0 / (rows.clamp_min(1) * (rows > 0).sum().clamp_min(1))
        loss = (torch.where(m, per, zero) * wt).sum()
        return [loss, ((u > cl) & m).sum() / n, torch.where(m, kl, zero).sum() / n, torch.where(m, grad, zero) * wt]
    if op == "preference":
        m = s["mask"]
        zero = torch.zeros_like(s["logp"])
        diff = s["logp"] if s["ref"] is None else s["logp"] - s["ref"]
        n = m.sum(1).clamp_min(1).float() if c["average"] else torch.ones(m.shape[0], device=m.device)
        rewards = BETA * torch.where(m, diff, zero).sum(1) / n
        P, e = c["P"], c["smoothing"]
        delta = rewards[:P] - rewards[P:]
        # -log sigmoid(x) = log(1 + exp(-|x|)) + max(-x, 0)
        soft = (1 + (-delta.abs()).exp()).log()
        loss = ((1 - e) * (soft + (-delta).clamp_min(0)) + e * (soft + delta.clamp_min(0))).mean()
        sig = 1 / (1 + (-delta).exp())
        dd = (e * sig - (1 - e) * (1 - sig)) / P
        row = BETA * torch.cat([dd, -dd]) / n
        return [loss, rewards, torch.where(m, row[:, None].expand(m.shape), zero)]
    tau = c["tau"]
    have = s["ids"] >= 0
    at = s["ids"].clamp_min(0)
    counts = s["mask"] & have.any(1)
    n = counts.sum().clamp_min(1)
    t = (s["top"].float() / tau).masked_fill(~have, -math.inf)
    t = t - t.amax(1, keepdim=True).clamp_min(-1e30)
    e = t.exp()
    q = e / e.sum(1, keepdim=True).clamp_min(1e-30)
    logq = torch.where(have, t - e.sum(1, keepdim=True).clamp_min(1e-30).log(), torch.zeros_like(t))
    x = s["logits"].float() / tau
    m = x.amax(1, keepdim=True)
    lse = (x - m).exp().sum(1, keepdim=True).log() + m
    per = tau * tau * (q * (logq - torch.where(have, x.gather(1, at) - lse, torch.zeros_like(q)))).sum(1)
    loss = torch.where(counts, per, torch.zeros_like(per)).sum() / n
    grad = x.sub_(lse).exp_()
    grad.scatter_add_(1, at, -q)
    grad = grad.mul_(torch.where(counts, tau / n, torch.zeros_like(per))[:, None])
    return [loss, grad.to(s["logits"].dtype)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op in ("score", "train"):
        T, H, V = case["T"], case["H"], case["V"]
        if op == "score":
            return {"bytes": 2 * T * H + 2 * V * H + 8 * T + 4 * T, "flops": 2 * T * V * H}
        return {"bytes": 2 * (2 * T * H + 2 * V * H) + 8 * T + 4 * T + 4 * T, "flops": 6 * T * V * H}
    if op == "policy":
        n = case["B"] * case["S"]
        adv = n if case["adv"] == "token" else case["B"]
        return {"bytes": 4 * n + 4 * n + 4 * adv + n + (4 * n if case["ref"] else 0) + 4 * n,
                "flops": (20 if case["ref"] else 12) * n}
    if op == "preference":
        n = 2 * case["P"] * case["S"]
        return {"bytes": 4 * n + n + (4 * n if case["ref"] else 0) + 4 * n, "flops": 3 * n}
    T, V, K = case["T"], case["V"], case["K"]
    es = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": 2 * es * T * V + 12 * T * K + T, "flops": 6 * T * V}


# ------------------------------------------------------------------ the definitions in 64 bits
@torch.no_grad()
def exact(case, seed):
    inp = _inputs(case, seed)
    op = case["op"]
    if op in ("score", "train"):
        return _exact_head(case, inp)
    if op == "policy":
        return _exact_policy(case, inp)
    if op == "preference":
        return _exact_preference(case, inp)
    return _exact_distill(case, inp)


def _exact_head(case, inp):
    h, ids, tau = inp["h"].double(), inp["ids"], case["tau"]
    w = inp["w"].double()
    logp = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    train = case["op"] == "train"
    dh, dw = torch.zeros_like(h), torch.zeros_like(w) if train else None
    for r in range(0, h.shape[0], 1024):
        rows = torch.arange(r, min(r + 1024, h.shape[0]), device=h.device)
        rows = rows[ids[rows] >= 0]
        if not rows.numel():
            continue
        z = torch.log_softmax(torch.mm(h[rows], w.T) / tau, dim=1)
        pick = torch.arange(rows.numel(), device=h.device)
        logp[rows] = z[pick, ids[rows]]
        if train:
            g = inp["g"][rows].double() / tau
            dz = z.exp_().neg_()
            dz[pick, ids[rows]] += 1.0
            dz *= g[:, None]
            dh[rows] = torch.mm(dz, w)
            dw.addmm_(dz.T, h[rows])
    return [logp, dh, dw] if train else [logp]


def _exact_policy(case, inp):
    m = inp["mask"]
    lp, old, adv = inp["logp"].double(), inp["old"].double(), inp["adv"].double().expand_as(inp["logp"])
    ratio = torch.exp(lp - old)
    low, high = 1 - CLIP_LOW, 1 + CLIP_HIGH
    # the clipped branch counts where the ratio has gone past an edge in the direction the advantage rewards
    past = ((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))
    edge = torch.where(adv > 0, torch.full_like(lp, high), torch.full_like(lp, low))
    per = -torch.where(past, edge * adv, ratio * adv)
    grad = torch.where(past, torch.zeros_like(lp), -ratio * adv)
    kl = torch.zeros_like(lp)
    if inp["ref"] is not None:
        x = inp["ref"].double() - lp
        kl = torch.expm1(x) - x
        per = per + KL_COEF * kl
        grad = grad - KL_COEF * torch.expm1(x)
    n = max(1, int(m.sum()))
    if case["reduction"] == "token":
        weight = m.double() / n
    else:
        counts = m.sum(1)
        live = max(1, int((counts > 0).sum()))
        weight = m.double() / counts.clamp(min=1)[:, None].double() / live
    return [(per * weight).sum(), (past & m).double().sum() / n, (kl * m).sum() / n, grad * weight]


def _exact_preference(case, inp):
    m = inp["mask"].double()
    diff = inp["logp"].double() - (0.0 if inp["ref"] is None else inp["ref"].double())
    scale = BETA * (1.0 / m.sum(1).clamp(min=1) if case["average"] else torch.ones_like(m[:, 0]))
    rewards = scale * (diff * m).sum(1)
    P, e = case["P"], case["smoothing"]
    gap = rewards[:P] - rewards[P:]
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - e) * ls(gap) + e * ls(-gap)).mean()
    d = (e * torch.sigmoid(gap) - (1 - e) * torch.sigmoid(-gap)) / P
    return [loss, rewards, m * (scale * torch.cat([d, -d]))[:, None]]


def _exact_distill(case, inp):
    tau, ids = case["tau"], inp["ids"]
    counts = inp["mask"] & (ids >= 0).any(1)
    n = max(1, int(counts.sum()))
    T, V = inp["logits"].shape
    total = torch.zeros((), dtype=torch.float64, device=ids.device)
    grad = torch.zeros(T, V, dtype=torch.float64, device=ids.device)
    for r in range(0, T, 1024):
        rows = torch.arange(r, min(r + 1024, T), device=ids.device)
        rows = rows[counts[rows]]
        if not rows.numel():
            continue
        logp = torch.log_softmax(inp["logits"][rows].double() / tau, dim=1)
        have = ids[rows] >= 0
        top = torch.where(have, inp["top"][rows].double() / tau, torch.full_like(inp["top"][rows], -math.inf).double())
        logq = torch.log_softmax(top, dim=1)
        q = logq.exp()
        at = torch.where(have, ids[rows], torch.zeros_like(ids[rows]))
        part = torch.where(have, q * (logq - logp.gather(1, at)), torch.zeros_like(q))
        total += tau * tau * part.sum()
        g = logp.exp_()
        g.scatter_add_(1, at, -torch.where(have, q, torch.zeros_like(q)))
        grad[rows] = g * (tau / n)
    return [total / n, grad]
