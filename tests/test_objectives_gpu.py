"""Post-training objectives on the GPU against the formulas in 64 bits.

Tolerances, fixed from the arithmetic:

* a logit of the tensor core is truncated once per 16-deep step, to 24 bits:
  its error is at most H / 16 steps x 2^-23 x the largest partial sum, taken
  as the row's largest |logit| plus the spread of a partial sum;
* bf16 rounds by at most 2^-8 of a value: three roundings lie between the
  formula and a gradient (exponential, logit gradient, output), 3 x 2^-8 of
  the norm at most;
* fp32 sums of n terms in trees of depth <= 40: 40 x 2^-24 of the sum of
  magnitudes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

GRAD_TOL = 3 * 2.0 ** -8


def _synced():
    from parallel_b200.ops._ext import check_device_errors

    torch.cuda.synchronize()
    check_device_errors()


def _err(a, b):
    """Norm of the difference over the norm of b (absolute where b is all zero)."""
    b = b.double()
    n = b.norm().item()
    return (a.double() - b).norm().item() / (n if n else 1.0)


# ----------------------------------------------------------------- log-probabilities through the LM head
def _head_inputs(T, H, V, ignored=0.3, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, H, device="cuda", generator=g) * (2.5 / math.sqrt(H))).bfloat16()
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    pull = 10 * torch.rand(T, 1, device="cuda", generator=g)
    h = (torch.randn(T, H, device="cuda", generator=g) + pull * w[ids].float() / 2.5).bfloat16()
    ids = ids.masked_fill(torch.rand(T, device="cuda", generator=g) < ignored, -100)
    return h, w, ids, torch.randn(T, device="cuda", generator=g)


def _head_reference(h, w, ids, g, tau):
    hd, wd = h.detach().double(), w.detach().double()
    rows = (ids >= 0).nonzero()[:, 0]
    logits = hd[rows] @ wd.T / tau
    at = torch.arange(rows.numel(), device="cuda")
    others = (logits - logits[at, ids[rows]][:, None]).exp()
    others[at, ids[rows]] = 0
    # 1 - p and log p of a nearly certain token vanish in 64 bits too if they are taken as differences
    log_p = -torch.log1p(others.sum(1))
    logp = torch.zeros(ids.shape[0], dtype=torch.float64, device="cuda")
    logp[rows] = log_p
    dl = -others * log_p.exp()[:, None]
    dl[at, ids[rows]] = -torch.expm1(log_p)
    dl *= (g[rows].double() / tau)[:, None]
    dh = torch.zeros_like(hd)
    dh[rows] = dl @ wd
    return logp, dh, dl.T @ hd[rows], (logits.abs().max().item() if rows.numel() else 0.0)


@pytest.mark.parametrize("T,H,V", [(1, 64, 8), (130, 256, 5001), (1000, 128, 20011)])
def test_lm_head_log_probs_scored_and_trained_are_the_same_bits(T, H, V):
    """A policy's ratio to itself is exactly 1: scoring a batch and training on it give one and the same number."""
    from parallel_b200.ops import objectives as O

    h, w, ids, _ = _head_inputs(T, H, V, seed=V)
    with torch.no_grad():
        scored = O.lm_head_log_probs(h, w, ids)
    trained = O.lm_head_log_probs(h.requires_grad_(True), w, ids)
    _synced()
    assert torch.equal(scored, trained.detach())


@pytest.mark.parametrize("H,V", [(64, 32003), (192, 5001), (64, 151936)])
def test_lm_head_log_probs_do_not_depend_on_the_batch(H, V):
    """A rollout scored in one batch and trained on in others, split by `max_block_bytes` or not: the same bits, so the
    first update's ratios are exactly 1."""
    from parallel_b200.ops import objectives as O

    T = 4096
    h, w, ids, _ = _head_inputs(T, H, V, ignored=0.2, seed=91)
    with torch.no_grad():
        scored = O.lm_head_log_probs(h, w, ids)
        parts = [O.lm_head_log_probs(h[a:b], w, ids[a:b]) for a, b in ((0, 1), (1, 9), (9, 300), (300, 1500), (1500, T))]
    hg = h.clone().requires_grad_(True)
    whole = O.lm_head_log_probs(hg, w, ids)
    micro = torch.cat([O.lm_head_log_probs(hg[a:a + 1024], w, ids[a:a + 1024]) for a in range(0, T, 1024)])
    split = O.lm_head_log_probs(hg, w, ids, max_block_bytes=2 * V * 512)
    _synced()
    for other in (torch.cat(parts), whole.detach(), micro.detach(), split.detach()):
        assert torch.equal(scored, other)


@pytest.mark.parametrize("T,H,V,tau", [(1, 64, 8, 1.0), (1, 1024, 32003, 1.0), (5, 72, 1, 1.0), (2, 8, 2, 0.5),
                                       (33, 128, 257, 1.3), (255, 200, 1000, 1.0), (256, 64, 4096, 2.0),
                                       (257, 512, 5001, 0.7), (1000, 1024, 32003, 1.0), (130, 4096, 20011, 1.0)])
def test_lm_head_log_probs(T, H, V, tau):
    from parallel_b200.ops import objectives as O

    h, w, ids, g = _head_inputs(T, H, V, seed=T + V)
    h.requires_grad_(True)
    w.requires_grad_(True)
    logp = O.lm_head_log_probs(h, w, ids, temperature=tau)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    with torch.no_grad():
        scored = O.lm_head_log_probs(h, w, ids, temperature=tau)
    _synced()
    ref, rdh, rdw, top = _head_reference(h, w, ids, g, tau)
    assert logp.dtype == torch.float32 and logp.shape == ids.shape and dh.dtype == dw.dtype == torch.bfloat16
    tol = (H / 16 + 8) * 2.0 ** -23 * (top + 4)
    assert (logp.double() - ref).abs().max().item() <= tol
    assert (scored.double() - ref).abs().max().item() <= tol
    assert torch.equal(logp[ids < 0], torch.zeros_like(logp[ids < 0]))
    assert torch.equal(dh[ids < 0], torch.zeros_like(dh[ids < 0]))
    assert _err(dh, rdh) <= GRAD_TOL and _err(dw, rdw) <= GRAD_TOL


def test_lm_head_log_probs_nearly_certain_tokens_keep_their_digits():
    """logp down to 1e-6: the sum runs over the other tokens and is not a difference of two large numbers."""
    from parallel_b200.ops import objectives as O

    h, w, ids, g = _head_inputs(64, 512, 1000, ignored=0.0, seed=3)
    h = (h.float() + 9.0 * w[ids].float()).bfloat16()
    logp = O.lm_head_log_probs(h, w, ids)
    _synced()
    ref = _head_reference(h, w, ids, g, 1.0)[0]
    assert ref.max().item() > -1e-5
    # a relative error of 2^-23 per step in a logit of about 30 moves exp(l_v - l_id) by this much
    assert ((logp.double() - ref) / ref).abs().max().item() <= (512 / 16 + 8) * 2.0 ** -23 * 40


@pytest.mark.parametrize("at", [0, 4095])
@pytest.mark.parametrize("sign", [1, -1])
def test_lm_head_log_probs_of_hidden_states_with_one_large_component(at, sign):
    """The whole of a logit in one component, the first or the last: the sum has its full size in every step or in
    none.  Either way a step loses less than a unit in the 24th bit, and what is given back is a quarter of that."""
    from parallel_b200.ops import objectives as O

    T, H, V = 64, 4096, 5001
    g = torch.Generator(device="cuda").manual_seed(95)
    h = (0.01 * torch.randn(T, H, device="cuda", generator=g))
    w = (torch.randn(V, H, device="cuda", generator=g) / math.sqrt(H))
    h[:, at], w[:, at] = 40.0, sign * (0.75 + 0.05 * torch.rand(V, device="cuda", generator=g))
    h, w = h.bfloat16(), w.bfloat16()
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    logp = O.lm_head_log_probs(h, w, ids)
    _synced()
    ref, _, _, top = _head_reference(h, w, ids, torch.ones(T, device="cuda"), 1.0)
    assert (logp.double() - ref).abs().max().item() <= (H / 16 + 8) * 2.0 ** -23 * top


@pytest.mark.parametrize("ignored", [0.0, 0.5, 1.0])
def test_lm_head_log_probs_row_blocks_and_garbage_in_ignored_rows(ignored):
    """Rows beyond the block are scored twice and the head's gradient adds up over blocks; ignored rows may hold
    anything without reaching a gradient."""
    from parallel_b200.ops import objectives as O

    T, H, V = 1000, 256, 5001
    h, w, ids, g = _head_inputs(T, H, V, ignored=ignored, seed=5)
    h[ids < 0] = float("nan")
    g[ids < 0] = float("inf")
    h.requires_grad_(True)
    w.requires_grad_(True)
    out = []
    for block_bytes in (6 << 30, 2 * V * 256, 0):
        logp = O.lm_head_log_probs(h, w, ids, max_block_bytes=block_bytes)
        out.append((logp.detach(), *torch.autograd.grad(logp, (h, w), g)))
    _synced()
    ref, rdh, rdw, top = _head_reference(h, w, ids, g, 1.0)
    for logp, dh, dw in out:
        assert (logp.double() - ref).abs().max().item() <= (H / 16 + 8) * 2.0 ** -23 * (top + 4)
        assert _err(dh, rdh) <= GRAD_TOL and _err(dw, rdw) <= GRAD_TOL


def test_lm_head_log_probs_layouts_streams_and_partial_gradients():
    from parallel_b200.ops import objectives as O

    T, H, V = 300, 128, 1003
    h, w, ids, g = _head_inputs(T, H, V, seed=7)
    ref, rdh, rdw, top = _head_reference(h, w, ids, g, 1.0)
    tol = (H / 16 + 8) * 2.0 ** -23 * (top + 4)
    wide = torch.zeros(T, H + 3, device="cuda", dtype=torch.bfloat16)  # rows at odd addresses
    wide[:, 1:H + 1] = h
    wt = w.t().contiguous().t()  # column-major head
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a = O.lm_head_log_probs(wide[:, 1:H + 1], wt, ids)
        one = O.lm_head_log_probs(wide[3:4, 1:H + 1], w, ids[3:4])
        shaped = O.lm_head_log_probs(h.view(3, 100, H), w, ids.view(3, 100))
        hg = h.clone().requires_grad_(True)
        dh = torch.autograd.grad(O.lm_head_log_probs(hg, w, ids), hg, g)[0]
        wg = w.clone().requires_grad_(True)
        dw = torch.autograd.grad(O.lm_head_log_probs(h, wg, ids), wg, g)[0]
    torch.cuda.current_stream().wait_stream(stream)
    _synced()
    assert (a.double() - ref).abs().max().item() <= tol and (one.double() - ref[3:4]).abs().max().item() <= tol
    assert shaped.shape == (3, 100) and (shaped.reshape(-1).double() - ref).abs().max().item() <= tol
    assert _err(dh, rdh) <= GRAD_TOL and _err(dw, rdw) <= GRAD_TOL


def test_lm_head_log_probs_against_differences():
    """Central differences of the summed log-probabilities along a direction whose steps bf16 holds exactly."""
    from parallel_b200.ops import objectives as O

    T, H, V = 40, 64, 301
    g = torch.Generator(device="cuda").manual_seed(11)
    h = torch.randint(-96, 97, (T, H), device="cuda", generator=g).float().div_(64)
    d = torch.randint(-1, 2, (T, H), device="cuda", generator=g).float().div_(64)
    w = (torch.randn(V, H, device="cuda", generator=g) * 0.4).bfloat16()
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    assert torch.equal((h + d).bfloat16().float(), h + d)
    hb = h.bfloat16().requires_grad_(True)
    dh = torch.autograd.grad(O.lm_head_log_probs(hb, w, ids).sum(), hb)[0]
    with torch.no_grad():
        up = O.lm_head_log_probs((h + d).bfloat16(), w, ids).double()
        down = O.lm_head_log_probs((h - d).bfloat16(), w, ids).double()
    _synced()
    per_row = (dh.double() * d.double()).sum(1)
    # third-order term of a log-softmax along d: at most (max |d . w| - mean)^3; bf16 gradient; two fp32 log-probs
    step = (d @ w.float().t()).abs().max(1).values.double() * 2
    tol = step ** 3 + GRAD_TOL * (dh.double() * d.double()).abs().sum(1) + 1e-5
    assert (((up - down) / 2 - per_row).abs() <= tol).all()


def test_lm_head_log_probs_special_values_and_refusals():
    from parallel_b200.ops import objectives as O

    h, w, ids, g = _head_inputs(40, 64, 300, ignored=0.0, seed=13)
    ref = _head_reference(h, w, ids, g, 1.0)[0]
    h[3] = float("nan")
    h[4] = float("inf")
    ids[5] = 300  # outside the vocabulary
    logp = O.lm_head_log_probs(h, w, ids)
    _synced()
    assert torch.isnan(logp[3:6]).all()
    rest = [i for i in range(40) if i not in (3, 4, 5)]
    assert (logp[rest].double() - ref[rest]).abs().max().item() <= 1e-4
    empty = O.lm_head_log_probs(h[:0].requires_grad_(True), w, ids[:0])
    assert empty.shape == (0,)
    empty.sum().backward()
    ok = ids.clamp_max(299)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ok, temperature=0.0)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w[:, :32], ok)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ok[:39])
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ok.int())
    with pytest.raises(TypeError):
        O.lm_head_log_probs(h.float(), w, ok)
    with pytest.raises(RuntimeError):  # 12 columns: rows that TMA cannot read
        O.lm_head_log_probs(h[:, :12].contiguous(), w[:, :12].contiguous(), ok)
    hg = h[:2].clone().requires_grad_(True)
    out = O.lm_head_log_probs(hg, w, ok[:2]).sum()
    out.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="one backward"):
        out.backward()
    _synced()


# ----------------------------------------------------------------- policy loss
LOW, HIGH, KL = 0.2, 0.28, 0.05
F32 = 2.0 ** -24


def _token_inputs(B, S, seed, masked=True):
    """Log-probabilities with garbage outside the mask: a prompt, a padded tail and whole empty rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    logp = -randn(B, S).abs() * 1.5
    d = 0.2 * randn(B, S)
    for edge in (math.log(1 - LOW), math.log(1 + HIGH)):  # a ratio on the clip's edge is decided by rounding
        d = torch.where((d - edge).abs() < 1e-3, torch.full_like(d, edge + 2e-3), d)
    old, ref, adv = logp - d, logp + 0.3 * randn(B, S), randn(B, S)
    mask = None
    if masked:
        pos = torch.arange(S, device="cuda")[None]
        start = (torch.rand(B, 1, device="cuda", generator=g) * S * 0.4).long()
        mask = (pos >= start) & (pos < start + 1 + (torch.rand(B, 1, device="cuda", generator=g) * S).long())
        mask &= torch.rand(B, 1, device="cuda", generator=g) >= 0.2
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda")
        out = junk[torch.randint(0, 4, (B, S), device="cuda", generator=g)]
        logp, old, ref, adv = (torch.where(mask, t, out) for t in (logp, old, ref, adv))
    return logp, old, ref, adv, mask


def _policy_reference(logp, old, ref, adv, mask, per_sequence):
    m = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask

    def clean(t):
        return torch.where(m, t, torch.zeros_like(t)).double()

    lp, o, a = clean(logp), clean(old), clean(adv.expand_as(logp))
    r = (lp - o).exp()
    past = ((a > 0) & (r > 1 + HIGH)) | ((a < 0) & (r < 1 - LOW))
    edge = torch.where(a > 0, torch.full_like(a, 1 + HIGH), torch.full_like(a, 1 - LOW))
    per = -torch.where(past, edge * a, r * a)
    grad, scale, kl = torch.where(past, 0.0, -r * a), (r * a).abs(), torch.zeros_like(lp)
    if ref is not None:
        x = clean(ref) - lp
        kl = torch.expm1(x) - x
        per, grad, scale = per + KL * kl, grad - KL * torch.expm1(x), scale + KL * torch.expm1(x).abs()
    n, rows = max(1, int(m.sum())), m.sum(1)
    w = m.double() / n
    if per_sequence:
        w = m.double() / rows.clamp(min=1)[:, None] / max(1, int((rows > 0).sum()))
    return ((per * w).sum(), (past & m).sum().double() / n, (kl * m).sum() / n, grad * w, scale * w,
            ((per.abs() + 1) * w).sum())


@pytest.mark.parametrize("B,S", [(1, 1), (3, 1), (1, 33), (8, 509), (5, 1000), (64, 300), (600, 7), (40, 5003)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss(B, S, reduction):
    from parallel_b200.ops import objectives as O

    for masked, with_ref, per_row_adv in ((True, True, False), (False, False, True), (True, False, True)):
        logp, old, ref, adv, mask = _token_inputs(B, S, seed=B + S, masked=masked)
        if per_row_adv:
            adv = torch.randn(B, device="cuda")
        logp.requires_grad_(True)
        args = dict(mask=mask, ref_logp=ref if with_ref else None, clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                    reduction=reduction)
        out = O.policy_loss(logp, old, adv, **args)
        (grad,) = torch.autograd.grad(3.0 * out.loss, logp)
        with torch.no_grad():
            scored = O.policy_loss(logp, old, adv, **args)
        _synced()
        wide = adv[:, None] if per_row_adv else adv
        loss, clip, kl, rgrad, scale, size = _policy_reference(logp.detach(), old, ref if with_ref else None, wide,
                                                               mask, reduction == "sequence")
        # exp of a log ratio of a few units: an argument off by 2^-24 of |logp| <= 8, and 2 ulp of exp itself
        tol = 40 * F32
        assert abs(out.loss.item() - loss.item()) <= tol * size.item()
        assert abs(out.clip_fraction.item() - clip.item()) <= 2 * F32
        assert abs(out.kl.item() - kl.item()) <= tol * (kl.item() + 1)
        assert ((grad.double() - 3 * rgrad).abs() <= 3 * tol * scale).all()
        if mask is not None:
            assert torch.equal(grad[~mask], torch.zeros_like(grad[~mask]))
        assert all(torch.equal(a.detach(), b) for a, b in zip(out, scored))


def test_policy_loss_strided_inputs_streams_and_same_bits():
    from parallel_b200.ops import objectives as O

    B, S = 70, 777
    logp, old, ref, adv, mask = _token_inputs(B, S, seed=1)
    want = O.policy_loss(logp, old, adv, mask=mask, ref_logp=ref, clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                         reduction="sequence")

    def shifted(t):
        wide = torch.zeros(B, S + 5, device="cuda", dtype=t.dtype)
        wide[:, 2:S + 2] = t
        return wide[:, 2:S + 2]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        lp = shifted(logp).requires_grad_(True)
        got = O.policy_loss(lp, shifted(old), adv.t().contiguous().t(), mask=shifted(mask),
                            ref_logp=ref.t().contiguous().t(), clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                            reduction="sequence")
        g1 = torch.autograd.grad(got.loss, lp)[0]
    torch.cuda.current_stream().wait_stream(stream)
    g2 = torch.autograd.grad(
        O.policy_loss(lp, old, adv, mask=mask, ref_logp=ref, clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                      reduction="sequence").loss, lp)[0]
    _synced()
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, want)) and torch.equal(g1, g2)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_without_a_kl_term_takes_any_reference(reduction):
    """kl_coef 0: the reference is reported on and nothing else, where the estimate is infinite too."""
    from parallel_b200.ops import objectives as O

    lp = -torch.rand(3, 7, device="cuda")
    ref = lp.clone()
    ref[1, 2], ref[2, 3] = -float("inf"), 3e38
    adv = torch.randn(3, 7, device="cuda")
    outs = []
    for r in (None, ref):
        x = lp.clone().requires_grad_(True)
        out = O.policy_loss(x, lp - 0.1, adv, ref_logp=r, reduction=reduction)
        outs.append((out.loss.detach(), out.clip_fraction, torch.autograd.grad(out.loss, x)[0]))
    _synced()
    assert out.kl.item() == float("inf")
    assert torch.isfinite(outs[0][0]) and all(torch.equal(a, b) for a, b in zip(*outs))


def test_policy_loss_without_tokens_and_refusals():
    from parallel_b200.ops import objectives as O

    lp = torch.full((3, 5), float("nan"), device="cuda", requires_grad=True)
    none = torch.zeros(3, 5, device="cuda", dtype=torch.bool)
    for reduction in ("token", "sequence"):
        out = O.policy_loss(lp, lp, lp, mask=none, ref_logp=lp, kl_coef=1.0, reduction=reduction)
        (g,) = torch.autograd.grad(out.loss, lp)
        assert out.loss.item() == 0 and out.kl.item() == 0 and torch.equal(g, torch.zeros_like(g))
    empty = torch.zeros(4, 0, device="cuda")
    assert O.policy_loss(empty, empty, torch.zeros(4, device="cuda")).loss.item() == 0
    x = torch.zeros(3, 5, device="cuda")
    for bad in (dict(logp=x[0]), dict(logp=x.bfloat16()), dict(mask=none.int()), dict(mask=none[:2]),
                dict(reduction="mean"), dict(clip_low=1.5), dict(clip_high=-0.1), dict(advantages=x[:, :2]),
                dict(old_logp=x[:2])):
        with pytest.raises(ValueError):
            O.policy_loss(**{**dict(logp=x, old_logp=x, advantages=x), **bad})
    for bad in (dict(advantages=x.double()), dict(ref_logp=x.half())):
        with pytest.raises(TypeError):
            O.policy_loss(**{**dict(logp=x, old_logp=x, advantages=x), **bad})
    with pytest.raises(RuntimeError):
        O.policy_loss(x, x.cpu(), x)
    _synced()


# ----------------------------------------------------------------- preference loss
def _preference_reference(logp, ref, mask, beta, e, average):
    m = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask
    zero = torch.zeros_like(logp)
    diff = torch.where(m, logp, zero).double() - (0 if ref is None else torch.where(m, ref, zero).double())
    w = beta / (m.sum(1).clamp(min=1).double() if average else 1.0)
    rewards = w * diff.sum(1)
    P = logp.shape[0] // 2
    gap = rewards[:P] - rewards[P:]
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - e) * ls(gap) + e * ls(-gap)).mean()
    d = (e * torch.sigmoid(gap) - (1 - e) * torch.sigmoid(-gap)) / P
    grad = m * (w * torch.cat([d, -d]))[:, None]
    return loss, rewards, grad, (w * diff.abs().sum(1))


@pytest.mark.parametrize("P,S", [(1, 1), (1, 300), (4, 300), (3, 2000), (100, 65), (700, 3), (20, 5003)])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss(P, S, average):
    from parallel_b200.ops import objectives as O

    for masked, with_ref, e in ((True, True, 0.0), (False, True, 0.1), (True, False, 0.1)):
        logp, ref, _, _, mask = _token_inputs(2 * P, S, seed=P + S, masked=masked)
        logp.requires_grad_(True)
        args = dict(ref_logp=ref if with_ref else None, mask=mask, beta=0.1, label_smoothing=e, average=average)
        out = O.preference_loss(logp, **args)
        (grad,) = torch.autograd.grad(-2.0 * out.loss, logp)
        with torch.no_grad():
            scored = O.preference_loss(logp, **args)
        _synced()
        loss, rewards, rgrad, size = _preference_reference(logp.detach(), ref if with_ref else None, mask, 0.1, e,
                                                           average)
        # a lane adds up to 32 differences, a warp's tree 5 levels, the rest in 64 bits
        tol = 40 * F32 * size + 2 * F32
        assert ((out.rewards.double() - rewards).abs() <= tol).all()
        gap_tol = (tol[:P] + tol[P:]).max().item()
        assert abs(out.loss.item() - loss.item()) <= gap_tol + 8 * F32 * (1 + loss.item())
        # the gradient of a row moves with the gap by at most a quarter of it, relative to the smaller sigmoid at most once
        assert ((grad.double() + 2 * rgrad).abs() <= 2 * (gap_tol + 16 * F32) * rgrad.abs() + 1e-30).all()
        assert torch.equal(out.loss.detach(), scored.loss) and torch.equal(out.rewards, scored.rewards)


def test_preference_loss_extreme_gaps_empty_rows_and_refusals():
    from parallel_b200.ops import objectives as O

    # gaps of +-2000 with beta 1: the loss is 0 on one side and the gap on the other, nothing overflows
    lp = torch.zeros(4, 10, device="cuda")
    lp[0], lp[3] = -200.0, -200.0
    lp.requires_grad_(True)
    out = O.preference_loss(lp, beta=1.0)
    (g,) = torch.autograd.grad(out.loss, lp)
    _synced()
    assert out.rewards.tolist() == [-2000.0, 0.0, 0.0, -2000.0] and out.loss.item() == 1000.0
    assert g[:, 0].tolist() == [-0.5, 0.0, 0.5, 0.0]
    mask = torch.zeros(4, 10, device="cuda", dtype=torch.bool)
    nan = torch.full((4, 10), float("nan"), device="cuda", requires_grad=True)
    for average in (False, True):
        out = O.preference_loss(nan, ref_logp=nan, mask=mask, average=average)
        (g,) = torch.autograd.grad(out.loss, nan)
        assert abs(out.loss.item() - math.log(2)) < 1e-6 and torch.equal(g, torch.zeros_like(g))
    x = torch.zeros(4, 5, device="cuda")
    for bad in (dict(logp=x[:3]), dict(logp=x[:0]), dict(label_smoothing=1.5), dict(beta=float("nan")),
                dict(mask=x), dict(ref_logp=x[:2])):
        with pytest.raises(ValueError):
            O.preference_loss(**{**dict(logp=x), **bad})
    with pytest.raises(TypeError):
        O.preference_loss(x, ref_logp=x.double())
    _synced()


def test_preference_loss_of_impossible_tokens():
    """A rejected token of probability zero: an infinite gap, and a loss of 0 with unsmoothed labels.  A chosen one:
    an infinite loss with the gradient of a certain error."""
    from parallel_b200.ops import objectives as O

    inf = float("inf")
    for side, smoothing, want, grads in ((2, 0.0, 0.0, (0.0, 0.0)), (0, 0.0, inf, (-0.5, 0.5)), (2, 0.25, inf, (0.125, -0.125)),
                                         (0, 0.25, inf, (-0.375, 0.375)), (0, 1.0, 0.0, (0.0, 0.0)), (2, 1.0, inf, (0.5, -0.5))):
        lp = torch.zeros(4, 6, device="cuda")
        lp[side, 3] = -inf  # pair 0; pair 1 has a gap of 0
        lp.requires_grad_(True)
        out = O.preference_loss(lp, beta=1.0, label_smoothing=smoothing)
        (grad,) = torch.autograd.grad(out.loss, lp)
        _synced()
        assert out.loss.item() == want if want else abs(out.loss.item() - math.log(2) / 2) < 1e-6
        assert grad[0].tolist() == [grads[0]] * 6 and grad[2].tolist() == [grads[1]] * 6
        assert torch.isfinite(grad).all()


def test_policy_and_preference_gradients_against_differences():
    """Central differences on the kernels' own losses, summed over a batch small enough for fp32 to resolve them."""
    from parallel_b200.ops import objectives as O

    B, S = 4, 6
    logp, old, ref, adv, mask = _token_inputs(B, S, seed=9, masked=False)
    fns = {"policy": lambda t: O.policy_loss(t, old, adv, ref_logp=ref, clip_low=LOW, clip_high=HIGH, kl_coef=KL).loss,
           "preference": lambda t: O.preference_loss(t, ref_logp=ref, beta=0.5, label_smoothing=0.1).loss}
    # within +-eps of the edges the policy loss has a corner: those positions are left out
    r = (logp - old).exp()
    eps = 2.0 ** -7
    away = ((r.log() - math.log(1 - LOW)).abs() > 2 * eps) & ((r.log() - math.log(1 + HIGH)).abs() > 2 * eps)
    for fn in fns.values():
        x = logp.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(fn(x), x)
        for b in range(B):
            for s in range(S):
                if not away[b, s]:
                    continue
                d = torch.zeros_like(logp)
                d[b, s] = eps
                with torch.no_grad():
                    fd = (fn(logp + d).double() - fn(logp - d).double()).item() / (2 * eps)
                # loss of order 1 in fp32 over 2 eps, and eps^2 / 6 times a third derivative of order 1
                assert abs(fd - grad[b, s].item()) <= 8 * F32 / (2 * eps) * 8 + eps ** 2


@pytest.mark.parametrize("B,S", [(2, 1), (8, 2), (4, 185), (30, 2000), (300, 333)])
def test_policy_and_preference_losses_are_rounded_once(B, S):
    """Losses, KL and rewards are sums that cancel, worked out in 64 bits and rounded to fp32 at the end."""
    from parallel_b200.ops import objectives as O

    for seed in range(4):
        for masked in (False, True):
            logp, old, ref, adv, mask = _token_inputs(B, S, seed=200 + seed, masked=masked)
            for reduction in ("token", "sequence"):
                out = O.policy_loss(logp, old, adv, mask=mask, ref_logp=ref, clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                                    reduction=reduction)
                loss, _, kl, _, _, size = _policy_reference(logp, old, ref, adv, mask, reduction == "sequence")
                assert abs(out.loss.item() - loss.item()) <= F32 * abs(loss.item()) + 1e-13 * size.item()
                assert abs(out.kl.item() - kl.item()) <= F32 * kl.item() + 1e-13 * (1 + kl.item())
            out = O.preference_loss(logp, ref_logp=ref, mask=mask, beta=0.1, label_smoothing=0.1)
            loss, rewards, _, size = _preference_reference(logp, ref, mask, 0.1, 0.1, False)
            assert ((out.rewards.double() - rewards).abs() <= F32 * rewards.abs() + 1e-13 * size).all()
            assert abs(out.loss.item() - loss.item()) <= F32 * loss.item() + 1e-13 * (1 + size.max().item())
    _synced()


# ----------------------------------------------------------------- distillation
def _teacher_inputs(T, V, K, dtype, seed):
    """Logits with junk in rows outside the mask and teacher entries with absent ids (junk values) among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(T, V, device="cuda", generator=g) * 2.5
    top = 4 + 5 * torch.rand(T, K, device="cuda", generator=g)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)  # some twice
    logits.scatter_add_(1, ids, 0.8 * top)
    absent = torch.rand(T, K, device="cuda", generator=g) < 0.2
    ids, top = ids.masked_fill(absent, -1), top.masked_fill(absent, float("nan"))
    mask = torch.rand(T, device="cuda", generator=g) >= 0.2
    logits[~mask] = float("inf")
    if T > 3:
        ids[1] = -1  # a row without any entry
        ids[2], top[2] = 0, 1.0  # one id for all,
        top[2, : K // 2] = -float("inf")  # some of probability zero
    return logits.to(dtype), top, ids, mask


def _distill_reference(logits, top, ids, mask, tau):
    have = (ids >= 0) & (top != -float("inf"))
    rows = (mask & have.any(1)).nonzero()[:, 0]
    n = max(1, rows.numel())
    h, at = have[rows], ids[rows].clamp_min(0).long()
    lp = torch.log_softmax(logits[rows].double() / tau, 1)
    lq = torch.log_softmax((top[rows].double() / tau).masked_fill(~h, -float("inf")), 1)
    q = torch.where(h, lq.exp(), 0.0)
    loss = tau ** 2 * torch.where(h, q * (lq - lp.gather(1, at)), 0.0).sum() / n
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda")
    g = lp.exp()
    g.scatter_add_(1, at, -q)
    grad[rows] = g * (tau / n)
    return loss, grad


@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (4, 3, 2), (5, 7, 9), (3, 64, 5), (33, 1000, 20), (130, 4099, 33),
                                   (17, 32003, 64), (9, 151936, 128), (2, 262144, 7), (3, 50257, 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_loss(T, V, K, dtype):
    from parallel_b200.ops import objectives as O

    logits, top, ids, mask = _teacher_inputs(T, V, K, dtype, seed=T + V + K)
    for tau, t, i in ((1.0, top, ids), (2.0, top.bfloat16(), ids.int())):
        x = logits.clone().requires_grad_(True)
        loss = O.distillation_loss(x, t, i, mask=mask, temperature=tau)
        (grad,) = torch.autograd.grad(0.5 * loss, x)
        with torch.no_grad():
            scored = O.distillation_loss(x, t, i, mask=mask, temperature=tau)
        _synced()
        ref, rgrad = _distill_reference(logits, t, i, mask, tau)
        # a softmax over V terms: exponents of up to 40 units off by 2^-24 of themselves, trees of depth <= 40
        tol = 100 * F32
        assert abs(loss.item() - ref.item()) <= tol * tau ** 2 * (abs(ref.item()) + 40)
        assert torch.equal(loss.detach(), scored)
        assert grad.dtype == dtype and grad.shape == x.shape
        # scaling by the incoming 0.5 is exact; bf16 rounds once
        rounding = 2.0 ** -8 if dtype == torch.bfloat16 else tol
        n = max(1, int((mask & (i >= 0).any(1)).sum()))
        assert ((grad.double() - 0.5 * rgrad).abs() <= rounding * (0.5 * rgrad).abs() + tol * tau / n).all()
        assert torch.equal(grad[~mask], torch.zeros_like(grad[~mask]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_loss_row_strides_and_alignments(dtype):
    """Rows that start at every 2- or 4-byte offset, padded rows, column slices, another stream, the same bits."""
    from parallel_b200.ops import objectives as O

    T, V, K = 21, 1003, 6
    logits, top, ids, mask = _teacher_inputs(T, V, K, dtype, seed=2)
    ref, rgrad = _distill_reference(logits, top, ids, mask, 1.0)
    first = None
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for shift in range(0, 9):
            for pad in (0, 1, 5):
                wide = torch.zeros(T, V + shift + pad, device="cuda", dtype=dtype)
                wide[:, shift:shift + V] = logits
                x = wide[:, shift:shift + V].requires_grad_(True)
                loss = O.distillation_loss(x, top, ids, mask=mask)
                (grad,) = torch.autograd.grad(loss, x)
                rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 100 * F32
                assert abs(loss.item() - ref.item()) <= 100 * F32 * (ref.item() + 40)
                assert ((grad.double() - rgrad).abs() <= rounding * rgrad.abs() + 100 * F32).all()
                again = O.distillation_loss(x, top, ids, mask=mask)
                assert torch.equal(again, loss)
                if shift == 0 and pad == 0:
                    first = loss.detach()
        turned = O.distillation_loss(logits.t().contiguous().t(), top.t().contiguous().t(), ids.t().contiguous().t(),
                                     mask=torch.stack([mask, ~mask], 1)[:, 0])
    torch.cuda.current_stream().wait_stream(stream)
    _synced()
    assert torch.equal(turned, first)


@pytest.mark.parametrize("T,V", [(3, 262144), (17, 151936), (74, 65536), (148, 32768)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_of_few_rows_on_a_busy_gpu(T, V, dtype):
    """Rows shared by a cluster of CTAs while another stream's kernels take and free the SMs, so that clusters start
    at all times: the bits of a quiet GPU, every time."""
    from parallel_b200.ops import objectives as O

    logits, top, ids, mask = _teacher_inputs(T, V, 5, dtype, seed=T)
    x = logits.requires_grad_(True)
    first = O.distillation_loss(x, top, ids, mask=mask)
    want = (first.detach(), torch.autograd.grad(first, x)[0])
    other, busy = torch.cuda.Stream(), torch.randn(1 << 22, device="cuda")
    other.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(20):
        with torch.cuda.stream(other):
            for k in range(4):
                busy = busy[: (1 << 22) - 4096 * ((i + k) % 7)].sin().repeat(2)[: 1 << 22]
        loss = O.distillation_loss(x, top, ids, mask=mask)
        got.append((loss.detach(), torch.autograd.grad(loss, x)[0]))
    torch.cuda.current_stream().wait_stream(other)
    _synced()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


@pytest.mark.parametrize("weight", [1 / 3, -0.3, 1e-3, 0.0])
@pytest.mark.parametrize("T,V", [(300, 5003), (17, 40000), (5, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_gradient_times_a_weight_is_rounded_once(T, V, dtype, weight):
    """What the loss is multiplied with enters the gradient before it is rounded to the logits' type."""
    from parallel_b200.ops import objectives as O

    logits, top, ids, mask = _teacher_inputs(T, V, 6, dtype, seed=T)
    x = logits.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(weight * O.distillation_loss(x, top, ids, mask=mask, temperature=2.0), x)
    _synced()
    want = _distill_reference(logits, top, ids, mask, 2.0)[1] * torch.tensor(weight, dtype=torch.float32).item()
    # the softmax in fp32, as without a weight: exponents of up to 40 units off by 2^-24 of themselves
    assert _err(grad, want) <= 1.05 * _err(want.to(dtype), want) + 100 * F32
    assert torch.equal(grad[~mask], torch.zeros_like(grad[~mask]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_of_saved_logits_that_come_back_elsewhere(dtype):
    """Saved-tensor hooks (offloading, checkpointing) may return the logits in another layout than they had."""
    from parallel_b200.ops import objectives as O

    T, V = 21, 1003
    logits, top, ids, mask = _teacher_inputs(T, V, 6, dtype, seed=3)
    wide = torch.zeros(T, V + 4, device="cuda", dtype=dtype)
    wide[:, 1:V + 1] = logits
    x = wide[:, 1:V + 1].requires_grad_(True)
    grads = []
    for hooks in (False, True):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu() if hooks else t,
                                                      lambda t: t.cuda().contiguous() if hooks else t):
            loss = O.distillation_loss(x, top, ids, mask=mask)
        grads.append([torch.autograd.grad(loss / 3, x)[0]])
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu() if hooks else t,
                                                      lambda t: t.cuda().contiguous() if hooks else t):
            loss = O.distillation_loss(x, top, ids, mask=mask)
        grads[-1].append(torch.autograd.grad(loss, x)[0])
    _synced()
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_distillation_loss_against_differences():
    from parallel_b200.ops import objectives as O

    T, V, K = 3, 13, 4
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(T, V, device="cuda", generator=g)
    top = torch.randn(T, K, device="cuda", generator=g)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)
    leaf = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(O.distillation_loss(leaf, top, ids, temperature=1.5), leaf)
    eps = 2.0 ** -6
    for t in range(T):
        for v in range(V):
            d = torch.zeros_like(x)
            d[t, v] = eps
            up = O.distillation_loss(x + d, top, ids, temperature=1.5).item()
            down = O.distillation_loss(x - d, top, ids, temperature=1.5).item()
            # fp32 losses of order 1 over 2 eps; eps^2 / 6 times a third derivative below 1
            assert abs((up - down) / (2 * eps) - grad[t, v].item()) <= 16 * F32 / (2 * eps) + eps ** 2 / 6


def test_distillation_loss_special_rows_and_refusals():
    from parallel_b200.ops import objectives as O

    x = torch.zeros(4, 10, device="cuda", requires_grad=True)
    top, ids = torch.zeros(4, 3, device="cuda"), torch.tensor([[1, 2, 3]] * 4, device="cuda")
    none = torch.zeros(4, device="cuda", dtype=torch.bool)
    loss = O.distillation_loss(x, top, ids, mask=none)
    (grad,) = torch.autograd.grad(loss, x)
    assert loss.item() == 0 and torch.equal(grad, torch.zeros_like(grad))
    assert O.distillation_loss(x[:0], top[:0], ids[:0]).item() == 0
    # a teacher token that the student forbids: an infinite loss with a finite gradient
    y = torch.zeros(4, 10, device="cuda")
    y[0, 2] = -float("inf")
    y.requires_grad_(True)
    loss = O.distillation_loss(y, top, ids)
    (grad,) = torch.autograd.grad(loss, y)
    assert loss.item() == float("inf") and torch.isfinite(grad).all()
    # an id outside the vocabulary, a NaN among the teacher's values, a NaN among the logits
    assert math.isnan(O.distillation_loss(x, top, ids + 8).item())
    assert math.isnan(O.distillation_loss(x, top.masked_fill(ids == 2, float("nan")), ids).item())
    z = torch.zeros(4, 10, device="cuda").index_fill(1, torch.tensor([5], device="cuda"), float("nan"))
    assert math.isnan(O.distillation_loss(z, top, ids).item())
    _synced()
    for bad in (dict(temperature=0.0), dict(top_logits=top[:3]), dict(top_ids=ids[:, :2]), dict(mask=none.int()),
                dict(mask=none[:2]), dict(top_logits=top[:, :0], top_ids=ids[:, :0])):
        with pytest.raises(ValueError):
            O.distillation_loss(**{**dict(logits=x, top_logits=top, top_ids=ids), **bad})
    for bad in (dict(top_ids=ids.float()), dict(top_logits=top.half()), dict(top_logits=ids)):
        with pytest.raises(TypeError):
            O.distillation_loss(**{**dict(logits=x, top_logits=top, top_ids=ids), **bad})
    big = torch.zeros(4, 1025, device="cuda")
    for bad in (dict(logits=x.half()), dict(top_logits=top.cpu()), dict(top_logits=big, top_ids=big.long())):
        with pytest.raises(RuntimeError):
            O.distillation_loss(**{**dict(logits=x, top_logits=top, top_ids=ids), **bad})
    wide = O.distillation_loss(torch.zeros(1, 262145, device="cuda"), top[:1], ids[:1])  # uniform over all, over 3
    assert abs(wide.item() - (math.log(262145) - math.log(3))) < 1e-4
    loss = O.distillation_loss(x, top, ids)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="one backward"):
        loss.backward()
    _synced()


@pytest.mark.parametrize("T,V,blocks", [(700, 5003, 1), (700, 5003, 3), (261, 50257, 2), (3, 40000, 1)])
def test_lm_head_distillation(T, V, blocks):
    """Blocks of rows, the last of them with few rows of a large vocabulary; rows outside the mask hold NaN."""
    from parallel_b200.ops import objectives as O

    H, K, tau = 192, 12, 2.0
    h, w, _, _ = _head_inputs(T, H, V, ignored=0.0, seed=21)
    g = torch.Generator(device="cuda").manual_seed(22)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=g)
    top = 6 * torch.rand(T, K, device="cuda", generator=g)
    mask = torch.rand(T, device="cuda", generator=g) >= 0.3
    mask[-1] = True
    clean = h.clone()
    h[~mask] = float("nan")
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = O.lm_head_distillation(h, w, top, ids, mask=mask, temperature=tau,
                                  max_block_bytes=(6 << 30) if blocks == 1 else 2 * V * 256)
    dh, dw = torch.autograd.grad(2 * loss, (h, w))
    with torch.no_grad():
        scored = O.lm_head_distillation(h, w, top, ids, mask=mask, temperature=tau)
    _synced()
    logits = clean.double() @ w.detach().double().t()
    ref, dl = _distill_reference(logits, top, ids, mask, tau)
    # bf16 logits: each off by up to 2^-8 of itself, which moves log p by as much
    tol = 2.0 ** -8 * logits.abs().max().item() * tau
    assert abs(loss.item() - ref.item()) <= tol and abs(scored.item() - ref.item()) <= tol
    # the softmax of rounded logits is off by up to 2^-8 x 10 (logits that carry probability) of its entries
    assert _err(dh, 2 * dl @ w.detach().double()) <= 10 * 2.0 ** -8
    assert _err(dw, 2 * dl.t() @ clean.double()) <= 10 * 2.0 ** -8
    assert torch.equal(dh[~mask], torch.zeros_like(dh[~mask]))


@pytest.mark.parametrize("weight", [1.0, 1 / 3, -0.3, 1e-3])
@pytest.mark.parametrize("blocks", [1, 3])
def test_lm_head_distillation_gradients_times_a_weight_are_rounded_once(blocks, weight):
    """Logits that bf16 holds exactly, so that the logits' gradient is known to its rounding (one in 10^4 entries may
    fall to the other side): its products with the head and the hidden states, times the weight, are rounded once."""
    from parallel_b200.ops import objectives as O

    T, H, V, K, tau = 700, 64, 1003, 6, 2.0
    gen = torch.Generator(device="cuda").manual_seed(81)
    h = torch.zeros(T, H, device="cuda")
    h.scatter_(1, torch.rand(T, H, device="cuda", generator=gen).topk(8, 1).indices, 1.0)
    h *= torch.randint(0, 2, (T, H), device="cuda", generator=gen) * 2 - 1
    w = torch.randint(-8, 9, (V, H), device="cuda", generator=gen) / 4  # logits: quarters up to 16
    logits = h.double() @ w.double().t()
    assert torch.equal(logits.bfloat16().double(), logits)
    ids = torch.randint(0, V, (T, K), device="cuda", generator=gen)
    top = 6 * torch.rand(T, K, device="cuda", generator=gen)
    mask = torch.rand(T, device="cuda", generator=gen) >= 0.3
    hg, wg = h.bfloat16().requires_grad_(True), w.bfloat16().requires_grad_(True)
    loss = O.lm_head_distillation(hg, wg, top, ids, mask=mask, temperature=tau,
                                  max_block_bytes=(6 << 30) if blocks == 1 else 2 * V * 256)
    dh, dw = torch.autograd.grad(weight * loss, (hg, wg))
    _synced()
    ref, dl = _distill_reference(logits, top, ids, mask, tau)
    assert abs(loss.item() - ref.item()) <= 100 * F32 * tau ** 2 * (ref.item() + 40)
    dl = dl.bfloat16().double() * torch.tensor(weight, dtype=torch.float32).item()
    for got, want in ((dh, dl @ w.double()), (dw, dl.t() @ h.double())):
        assert _err(got, want) <= 1.05 * _err(want.bfloat16(), want)
    assert torch.equal(dh[~mask], torch.zeros_like(dh[~mask]))


# ----------------------------------------------------------------- values at the ends of the types
@pytest.mark.parametrize("V", [40, 1003, 40000])
@pytest.mark.parametrize("tau", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_of_logits_masked_with_the_lowest_value(V, tau, dtype):
    """Masks of the type's lowest value: columns in front and behind, all but one, all; and the same for a teacher."""
    from parallel_b200.ops import objectives as O

    K, low = 5, torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = torch.randn(6, V, device="cuda", generator=g).to(dtype)
    logits[0, 10:] = low
    logits[1, : V - 10] = low
    logits[2, V // 2 + 1:] = low
    logits[2, : V // 2] = low
    logits[3] = low  # nothing left: uniform
    top = 3 * torch.rand(6, K, device="cuda", generator=g)
    ids = torch.randint(0, 10, (6, K), device="cuda", generator=g)
    ids[1] += V - 10
    ids[2] = V // 2
    top[4] = torch.finfo(torch.float32).min  # one value for all entries
    top[5, 1:] = torch.finfo(torch.float32).min
    x = logits.clone().requires_grad_(True)
    loss = O.distillation_loss(x, top, ids, temperature=tau)
    (grad,) = torch.autograd.grad(loss, x)
    _synced()
    ref, rgrad = _distill_reference(logits, top, ids, torch.ones(6, dtype=torch.bool, device="cuda"), tau)
    tol = 100 * F32
    assert abs(loss.item() - ref.item()) <= tol * tau ** 2 * (abs(ref.item()) + 40)
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else tol
    assert ((grad.double() - rgrad).abs() <= rounding * rgrad.abs() + tol * tau / 6).all()


@pytest.mark.parametrize("V", [333, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_of_large_logits(V, dtype):
    """|logit| / temperature up to 1e8: what counts are differences to the maximum, and these are exact."""
    from parallel_b200.ops import objectives as O

    T, K = 24, 4
    g = torch.Generator(device="cuda").manual_seed(V)
    # rows of 2^0, 2^1, ... times a mantissa: in bf16 neighbours at the top are 2^-7 of the logit apart
    size = 2.0 ** torch.arange(T, device="cuda")[:, None]
    logits = (size * (1 + torch.rand(T, V, device="cuda", generator=g))).to(dtype)
    logits[::2] = -logits[::2]
    ids = logits.float().topk(K, dim=1).indices
    top = torch.rand(T, K, device="cuda", generator=g)
    for tau in (1.0, 0.125):
        x = logits.clone().requires_grad_(True)
        loss = O.distillation_loss(x, top, ids, temperature=tau)
        (grad,) = torch.autograd.grad(loss, x)
        _synced()
        ref, rgrad = _distill_reference(logits, top, ids, torch.ones(T, dtype=torch.bool, device="cuda"), tau)
        # differences of up to 40 units matter in the exponentials; in the loss all do, off by 2^-22 of themselves.
        # bf16: one multiply-add up to exponents of 1024 (base 2), its addend rounded to 2^-15
        tol = 100 * F32 + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)
        assert abs(loss.item() - ref.item()) <= tol * tau ** 2 * (abs(ref.item()) / tau ** 2 + 40)
        rounding = 2.0 ** -8 + tol if dtype == torch.bfloat16 else tol
        assert ((grad.double() - rgrad).abs() <= rounding * rgrad.abs() + tol * tau / T).all()

@pytest.mark.parametrize("power", [0, 4, 8, 10, 11])
@pytest.mark.parametrize("V", [40, 1003])
def test_lm_head_log_probs_gradient_of_large_logits(power, V):
    """Logits of 2^(2 power) and a small whole number: exact in 24 bits, so their gradient hangs on the
    differences alone.  The target has a probability of about exp(-90): its logit is not part of the others' sum."""
    from parallel_b200.ops import objectives as O

    T, H = 20, 64
    g = torch.Generator(device="cuda").manual_seed(power)
    big = 2.0 ** power
    h = torch.zeros(T, H, device="cuda")
    w = torch.zeros(V, H, device="cuda")
    h[:, 0] = big * (1 + torch.arange(T, device="cuda") / 32)  # 6 bits of mantissa
    w[:, 0] = big
    h[:, 1:9] = torch.randint(-2, 3, (T, 8), device="cuda", generator=g).float()
    w[:, 1:9] = torch.randint(-1, 2, (V, 8), device="cuda", generator=g).float()
    ids = torch.arange(T, device="cuda")
    w[ids, 9 + ids] = -64.0  # column 9 + t lowers the target of row t, and it alone
    h[ids, 9 + ids] = 1.5
    h, w = h.bfloat16().requires_grad_(True), w.bfloat16().requires_grad_(True)
    logp = O.lm_head_log_probs(h, w, ids)
    dh, dw = torch.autograd.grad(logp.sum(), (h, w))
    _synced()
    ref, rdh, rdw, top = _head_reference(h, w, ids, torch.ones(T, device="cuda"), 1.0)
    # logp: the truncation given back to the others, at most 1 / 2^24 per 16-deep step, and fp32
    assert (logp.double() - ref).abs().max().item() <= (H / 16 + 8) * 2.0 ** -23 * (top + 4)
    # column 9 + t of dh: -64 x (gradient of the target's logit = 1); column 9 + t of dw sums 1.5 x that of row t
    assert _err(dh[:, 1:], rdh[:, 1:]) <= GRAD_TOL
    assert _err(dw[:, 9:9 + T], rdw[:, 9:9 + T]) <= GRAD_TOL and _err(dw[:, 1:9], rdw[:, 1:9]) <= GRAD_TOL
    # every vocabulary entry on its own: what row t alone sends it, over the hidden state's columns 9 and up
    want = -torch.softmax(h.detach().double() @ w.detach().double().t(), 1)
    want[ids, ids] += 1
    got = dw[:, 9:9 + T].t().double() / 1.5
    assert ((got - want).abs() <= GRAD_TOL * want.abs() + 1e-12).all()


def test_lm_head_log_probs_one_logit_above_all():
    """Logits of 2^14 to 2^31, far apart: the whole probability stands at the largest one."""
    from parallel_b200.ops import objectives as O

    T, H, V = 64, 64, 1003
    g = torch.Generator(device="cuda").manual_seed(0)
    h, w = torch.zeros(T, H, device="cuda"), torch.zeros(V, H, device="cuda")
    h[:, 0] = 2.0 ** (torch.arange(T, device="cuda") % 16) * (1 + torch.rand(T, device="cuda", generator=g))
    w[:, 0] = 2.0 ** 14 * (1 + torch.rand(V, device="cuda", generator=g))
    best = 700
    w[best, 0] = 2.0 ** 15 * 1.5
    ids = torch.randint(0, best, (T,), device="cuda", generator=g)
    h, w = h.bfloat16().requires_grad_(True), w.bfloat16()
    logp = O.lm_head_log_probs(h, w, ids)
    (dh,) = torch.autograd.grad(logp.sum(), h)
    _synced()
    want = w[ids].double() - w[best].double()  # the gradient: the target's row of the head less the best one's
    size = h.detach()[:, 0].double() * w[best, 0].double()
    assert ((logp.double() - want[:, 0] * h.detach()[:, 0].double()).abs() <= (H / 16 + 8) * 2.0 ** -23 * size).all()
    assert _err(dh, want) <= GRAD_TOL


@pytest.mark.parametrize("T,H,V,blocks", [(1, 1024, 32003, 1), (8, 4096, 32003, 1), (130, 1536, 5001, 1),
                                          (700, 64, 1003, 3)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_lm_head_log_probs_gradients_are_rounded_once_at_the_target(T, H, V, blocks, seed):
    """The target's part of both gradients is fp32 until the result is rounded; the others' coefficients are rounded
    to bf16, each on its own: the norms of what these add, sum of squares, at 2^-9 rms and three times that."""
    from parallel_b200.ops import objectives as O

    h, w, ids, g = _head_inputs(T, H, V, ignored=0.0, seed=100 + seed)
    h.requires_grad_(True)
    w.requires_grad_(True)
    logp = O.lm_head_log_probs(h, w, ids, max_block_bytes=(6 << 30) if blocks == 1 else 2 * V * 256)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    _synced()
    _, rdh, rdw, _ = _head_reference(h, w, ids, g, 1.0)
    p = torch.softmax(h.detach().double() @ w.detach().double().t(), 1)
    p[torch.arange(T, device="cuda"), ids] = 0
    p2 = (p * g.double()[:, None]) ** 2
    others_h = (p2 @ (w.detach().double() ** 2).sum(1)).sum().sqrt().item()
    others_w = (p2.sum(1) @ (h.detach().double() ** 2).sum(1)).sqrt().item()
    for got, want, others in ((dh, rdh, others_h), (dw, rdw, others_w)):
        once = _err(want.bfloat16(), want)
        assert _err(got, want) <= 1.05 * once + 3 * 2.0 ** -9 * others / want.norm().item()


@pytest.mark.parametrize("blocks", [1, 3])
def test_lm_head_log_probs_of_tokens_that_repeat(blocks):
    """One id for all rows, few ids, and ids in runs: the head's gradient adds them up, in the same bits every time."""
    from parallel_b200.ops import objectives as O

    T, H, V = 3000, 136, 1003
    h, w, _, g = _head_inputs(T, H, V, ignored=0.0, seed=61)
    gen = torch.Generator(device="cuda").manual_seed(62)
    for ids in (torch.full((T,), 7, device="cuda"), torch.randint(0, 3, (T,), device="cuda", generator=gen),
                torch.arange(T, device="cuda") // 40):
        ids = ids.masked_fill(torch.rand(T, device="cuda", generator=gen) < 0.1, -1)
        out = []
        for _ in range(2):
            hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            logp = O.lm_head_log_probs(hg, wg, ids, max_block_bytes=(6 << 30) if blocks == 1 else 2 * V * 1024)
            out.append(torch.autograd.grad(logp, (hg, wg), g))
        _synced()
        _, rdh, rdw, _ = _head_reference(h, w, ids, g, 1.0)
        assert _err(out[0][0], rdh) <= GRAD_TOL and _err(out[0][1], rdw) <= GRAD_TOL
        assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("T,H", [(16384, 64), (9000, 2056)])
def test_lm_head_gradient_of_one_token_in_many_rows_is_rounded_once(T, H):
    """All rows have one token and weights of both signs.  The product has nothing to add to that token's row of the
    head's gradient, so the row is a sum in fp32 (off by about sqrt(T) 2^-24 of itself) and one rounding."""
    from parallel_b200.ops import objectives as O

    V = 300
    h, w, _, g = _head_inputs(T, H, V, ignored=0.0, seed=71)
    ids = torch.full((T,), 7, device="cuda")
    wg = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(O.lm_head_log_probs(h, wg, ids), wg, g)
    _synced()
    want = _head_reference(h, w, ids, g, 1.0)[2][7]
    assert _err(dw[7], want) <= 1.05 * _err(want.bfloat16(), want)


def test_rows_that_share_memory_and_an_empty_vocabulary():
    """Broadcast and overlapping hidden states and heads are read as what they stand for; no vocabulary is refused."""
    from parallel_b200.ops import objectives as O

    h, w, ids, g = _head_inputs(33, 64, 300, ignored=0.1, seed=51)
    flat = torch.randn(33 * 8 + 64, device="cuda").bfloat16()
    for a, b in ((h[:1].expand(33, 64), w), (flat.as_strided((33, 64), (8, 1)), w), (h, w[:1].expand(300, 64))):
        ref, rdh, rdw, top = _head_reference(a, b, ids, g, 1.0)
        with torch.no_grad():
            scored = O.lm_head_log_probs(a, b, ids)
        ag, bg = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        logp = O.lm_head_log_probs(ag, bg, ids)
        dh, dw = torch.autograd.grad(logp, (ag, bg), g)
        _synced()
        assert (scored.double() - ref).abs().max().item() <= (64 / 16 + 8) * 2.0 ** -23 * (top + 4)
        assert torch.equal(scored, logp.detach())
        assert _err(dh, rdh) <= GRAD_TOL or rdh.abs().max().item() < 1e-12
        assert _err(dw, rdw) <= GRAD_TOL
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h.requires_grad_(True), w[:0], ids.clamp_max(-1))


# ----------------------------------------------------------------- offsets past 32 bits
def test_more_than_2_to_the_31_logits():
    """15,000 rows of a 151,936 vocabulary: 2.28e9 exponentials, logits and gradients, checked where offsets are
    largest and in a head-gradient column that every row reaches."""
    from parallel_b200.ops import objectives as O

    T, H, V = 15000, 64, 151936
    h, w, ids, g = _head_inputs(T, H, V, ignored=0.0, seed=41)
    h.requires_grad_(True)
    w.requires_grad_(True)
    logp = O.lm_head_log_probs(h, w, ids, max_block_bytes=8 << 30)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    _synced()
    rows = torch.cat([torch.arange(4), torch.arange(T - 300, T)]).cuda()
    ref, rdh, _, top = _head_reference(h.detach()[rows], w.detach(), ids[rows], g[rows], 1.0)
    assert (logp[rows].double() - ref).abs().max().item() <= (H / 16 + 8) * 2.0 ** -23 * (top + 4)
    assert _err(dh[rows], rdh) <= GRAD_TOL
    # the head's gradient at the last token and at one that is some row's target
    for v in (V - 1, int(ids[T - 1])):
        p = (h.detach().double() @ w.detach()[v].double()
             - (h.detach().double() * w.detach()[ids].double()).sum(1) + logp.double()).exp()
        want = (g.double() * ((ids == v).double() - p))[:, None].mul(h.detach().double()).sum(0)
        size = (g.double() * ((ids == v).double() + p))[:, None].mul(h.detach().double()).norm()
        assert (dw[v].double() - want).norm().item() <= GRAD_TOL * (want.norm().item() + size.item())
    del logp, dh, dw, h, w
    torch.cuda.empty_cache()

    gen = torch.Generator(device="cuda").manual_seed(42)
    x = torch.randn(T, V, device="cuda", generator=gen, dtype=torch.bfloat16)
    tid = torch.randint(0, V, (T, 4), device="cuda", generator=gen)
    teacher = 4 * torch.rand(T, 4, device="cuda", generator=gen)
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    mask[rows] = True
    x.requires_grad_(True)
    loss = O.distillation_loss(x, teacher, tid, mask=mask)
    (grad,) = torch.autograd.grad(loss, x)
    _synced()
    ref, rgrad = _distill_reference(x.detach()[rows], teacher[rows], tid[rows], mask[rows], 1.0)
    assert abs(loss.item() - ref.item()) <= 100 * F32 * (ref.item() + 40)
    assert ((grad[rows].double() - rgrad).abs() <= 2.0 ** -8 * rgrad.abs() + 100 * F32 / rows.numel()).all()
    assert not grad[4:T - 300].any()


# ----------------------------------------------------------------- together, as they are used
@pytest.mark.parametrize("name", ["small-qwen3", "small-qwen3-moe"])
def test_model_objectives_match_its_logits(name):
    from parallel_b200.models.config import resolve_config
    from parallel_b200.models.qwen3 import build_model
    from parallel_b200.ops import objectives as O

    m = build_model(resolve_config(name), device="cuda", dtype=torch.bfloat16, seed=0)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randint(0, 2048, (2, 136), device="cuda", generator=g)
    targets = torch.randint(0, 2048, (2, 136), device="cuda", generator=g)
    targets[0, :40] = -100
    with torch.no_grad():
        h = m(input_ids=x, targets=targets).hidden_states
        logits = h.double() @ m.lm_head.weight.double().t()
        out = m(input_ids=x, targets=targets, temperature=0.8)
        _synced()
        want = torch.log_softmax(logits / 0.8, -1).gather(-1, targets.clamp_min(0)[..., None])[..., 0]
        assert out.logits is None and out.loss is None
        # the hidden states of two passes may differ in the routing's atomics order; logits of order 1 here
        assert (out.log_probs.double() - want.masked_fill(targets < 0, 0)).abs().max().item() < 2e-2
        top = logits.float().topk(8, dim=-1)
    out = m(input_ids=x, teacher=(top.values, top.indices, targets >= 0), temperature=2.0)
    ref = O.distillation_loss(logits.float(), top.values, top.indices, mask=targets >= 0, temperature=2.0)
    aux = 0.0 if out.aux_loss is None else m.config.router_aux_loss_coef * out.aux_loss.item()
    assert abs(out.loss.item() - aux - ref.item()) < 2e-2
    out.loss.backward()
    assert torch.isfinite(m.lm_head.weight.grad).all()
    _synced()


@pytest.mark.parametrize("objective", ["policy", "preference", "distill"])
def test_post_training_example(objective):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "post_training.py")
    spec = importlib.util.spec_from_file_location("post_training", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    history = mod.main([objective, "--steps", "6", "--device", "cuda"])
    _synced()
    assert all(math.isfinite(v) for row in history for v in row.values())
    assert history[-1]["loss"] < history[0]["loss"]
    if objective == "policy":
        assert history[0]["kl"] == 0 and history[0]["clipped"] == 0


def test_objectives_replay_in_a_cuda_graph():
    """One captured step - log-probabilities, policy loss, gradients, distillation - replayed on other inputs, other
    masks included (the count of rows with a token lives on the device)."""
    from parallel_b200.ops import objectives as O

    T, H, V, K = 300, 128, 1003, 5
    sets = []
    for seed in (31, 32, 33):
        h, w, ids, _ = _head_inputs(T, H, V, ignored=0.2 * (seed - 30), seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        sets.append((h, w, ids, torch.randn(3, 100, device="cuda", generator=g),
                     torch.randint(0, V, (T, K), device="cuda", generator=g),
                     4 * torch.rand(T, K, device="cuda", generator=g)))
    static = [t.clone() for t in sets[0]]
    static[0].requires_grad_(True)
    static[1].requires_grad_(True)

    def step():
        h, w, ids, adv, tid, top = static
        logp = O.lm_head_log_probs(h.view(3, 100, H), w, ids.view(3, 100))
        out = O.policy_loss(logp, logp.detach() + 0.1, adv, mask=(ids >= 0).view(3, 100))
        kd = O.lm_head_distillation(h, w, top, tid, mask=ids >= 0)
        return (logp.detach(), out.loss.detach(), kd.detach(), *torch.autograd.grad(out.loss + kd, (h, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for inputs in sets[1:] + sets[:1]:
        with torch.no_grad():
            for dst, src in zip(static, inputs):
                dst.copy_(src)
        graph.replay()
        got = [t.clone() for t in outs]
        _synced()
        want = step()
        _synced()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_only_the_first_argument_gets_a_gradient():
    """Old and reference log-probabilities, advantages and teachers that carry a graph of their own get none."""
    from parallel_b200.ops import objectives as O

    B, S = 4, 40
    leaf = torch.randn(B, S, device="cuda", requires_grad=True)
    other = torch.randn(B, S, device="cuda", requires_grad=True)
    for fn in (lambda lp: O.policy_loss(lp, other, other, ref_logp=other, kl_coef=0.1).loss,
               lambda lp: O.policy_loss(lp, other, other[:, :1], ref_logp=other, reduction="sequence").loss,
               lambda lp: O.preference_loss(lp, ref_logp=other).loss,
               lambda lp: O.distillation_loss(lp, other[:, :3], torch.arange(3, device="cuda").expand(B, 3))):
        leaf.grad = other.grad = None
        fn(leaf).backward()
        assert leaf.grad is not None and other.grad is None
        assert not fn(leaf.detach()).requires_grad
    _synced()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad):
    """The kernels have no tangents: a dual tensor is refused, with or without a gradient, instead of losing its."""
    import torch.autograd.forward_ad as fwd

    from parallel_b200.ops import objectives as O

    def leaf(*shape):
        return torch.randn(*shape, device="cuda").requires_grad_(grad)

    h, w, lp, x = leaf(4, 64).bfloat16(), leaf(30, 64).bfloat16(), leaf(4, 5), leaf(4, 30)
    ids, top, tid = torch.arange(4, device="cuda"), torch.rand(4, 3, device="cuda"), torch.arange(12, device="cuda").view(4, 3)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for call in (lambda: O.lm_head_log_probs(dual(h), w, ids), lambda: O.lm_head_log_probs(h, dual(w), ids),
                     lambda: O.policy_loss(dual(lp), lp, lp), lambda: O.preference_loss(dual(lp)),
                     lambda: O.distillation_loss(dual(x), top, tid), lambda: O.lm_head_distillation(dual(h), w, top, tid),
                     lambda: O.lm_head_distillation(h, dual(w), top, tid)):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        # what takes no gradient takes no tangent either
        O.policy_loss(lp, dual(lp), dual(lp), ref_logp=dual(lp))
    _synced()
