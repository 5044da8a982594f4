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
