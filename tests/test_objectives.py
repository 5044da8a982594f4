"""Post-training objectives on CPU: the plain formulas and the refusals."""
import os
import re

import pytest
import torch

from parallel_b200.ops import objectives as O

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc")


def _device_functions():
    """(file, name, body without comments) of every kernel and device function in csrc."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, name)) as f:
            src = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__(?:global|device)__ (?:__forceinline__ )?[\w:]+\s+(?:__launch_bounds__\([^)]*\)\s*)?(\w+)\s*\("
                             r"[^;{]*\)\s*\{", src):
            depth, end = 1, m.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(src[end], 0)
                end += 1
            yield name, m.group(1), src[m.end():end]


def test_peers_of_a_cluster_have_started_before_their_shared_memory_is_addressed():
    """A CTA may write a peer's shared memory only once the peer has started, which a cluster barrier tells: its wait
    stands before the first such access in every function that makes one, but for the helpers that are the access."""
    seen = 0
    for file, kernel, body in _device_functions():
        if re.fullmatch(r"st_cluster_\w+|mapa_shared", kernel):
            continue
        remote = re.search(r"\b(st_cluster_\w+|mapa_shared)\(", body)
        if remote is None:
            continue
        seen += 1
        barrier = re.search(r"\b(cluster_sync|cluster_wait)\(\)", body)
        assert barrier is not None and barrier.start() < remote.start(), f"{file}: {kernel}"
    assert seen >= 3



def test_log_probs_plain_matches_log_softmax_and_ignores_rows():
    torch.manual_seed(0)
    h, w = torch.randn(3, 5, 16), torch.randn(11, 16)
    ids = torch.randint(0, 11, (3, 5))
    ids[1] = -100
    h[1] = float("nan")
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    logp = O.lm_head_log_probs(hg, wg, ids, temperature=0.7)
    ref = torch.log_softmax((h[[0, 2]] @ w.t()) / 0.7, -1).gather(-1, ids[[0, 2]][..., None])[..., 0]
    assert torch.allclose(logp[[0, 2]], ref, atol=1e-5) and torch.equal(logp[1], torch.zeros(5))
    logp.sum().backward()
    assert torch.isfinite(wg.grad).all() and torch.equal(hg.grad[1], torch.zeros(5, 16))


def test_log_probs_refusals():
    h, w, ids = torch.randn(4, 8), torch.randn(9, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ids, temperature=-1.0)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w[:, :4], ids)
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ids[:3])
    with pytest.raises(ValueError):
        O.lm_head_log_probs(h, w, ids.int())
    with pytest.raises(IndexError):
        O.lm_head_log_probs(h, w, ids + 9)
    assert O.lm_head_log_probs(h[:0], w, ids[:0]).shape == (0,)


def test_log_probs_refuse_an_empty_head_and_a_temperature_without_end():
    h, w, ids = torch.randn(4, 8), torch.randn(9, 8), torch.full((4,), -100)
    for bad in (dict(w=w[:0]), dict(h=h[:, :0], w=w[:, :0]), dict(temperature=float("inf")),
                dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            O.lm_head_log_probs(**{**dict(h=h, w=w, ids=ids), **bad})
    top, tid = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    with pytest.raises(ValueError):
        O.lm_head_distillation(h, w[:0], top, tid)
    with pytest.raises(ValueError):
        O.distillation_loss(h, top, tid, temperature=float("inf"))


def _differences(fn, x):
    """Autograd against central differences in 64 bits along a random direction."""
    x = x.detach().double().requires_grad_(True)
    (grad,) = torch.autograd.grad(fn(x), x)
    d = torch.randn_like(x)
    with torch.no_grad():
        fd = (fn(x + 1e-6 * d) - fn(x - 1e-6 * d)) / 2e-6
    assert abs((fd - (grad * d).sum()).item()) < 1e-6


def test_policy_loss_formula_and_gradient():
    torch.manual_seed(1)
    B, S = 5, 9
    logp = -torch.rand(B, S).double() * 3
    old, ref, adv = logp - 0.3 * torch.randn(B, S), logp + 0.2 * torch.randn(B, S), torch.randn(B).double()
    mask = torch.rand(B, S) < 0.7
    mask[2] = False
    for t in (old, ref):
        t[~mask] = float("nan")
    for reduction in ("token", "sequence"):
        def fn(x):
            return O.policy_loss(x, old, adv, mask=mask, ref_logp=ref, clip_low=0.1, clip_high=0.3, kl_coef=0.2,
                                 reduction=reduction).loss
        r = (logp - old).exp()
        a = adv[:, None]
        k = (ref - logp).exp() - (ref - logp) - 1
        per = torch.where(mask, -torch.minimum(r * a, r.clamp(0.9, 1.3) * a) + 0.2 * k, torch.zeros_like(r))
        rows = mask.sum(1)
        ref_loss = per.sum() / mask.sum() if reduction == "token" else \
            (per.sum(1) / rows.clamp_min(1)).sum() / (rows > 0).sum()
        assert torch.allclose(fn(logp), ref_loss)
        _differences(fn, logp)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_without_a_kl_term_takes_any_reference(reduction):
    """kl_coef 0: the reference is reported on and nothing else, where the estimate is infinite too."""
    lp = -torch.rand(3, 7)
    ref = lp.clone()
    ref[1, 2], ref[2, 3] = -float("inf"), 3e38
    adv = torch.randn(3, 7)
    outs = []
    for r in (None, ref):
        x = lp.clone().requires_grad_(True)
        out = O.policy_loss(x, lp - 0.1, adv, ref_logp=r, reduction=reduction)
        outs.append((out.loss.detach(), out.clip_fraction, torch.autograd.grad(out.loss, x)[0]))
    assert out.kl.item() == float("inf")
    assert torch.isfinite(outs[0][0]) and all(torch.equal(a, b) for a, b in zip(*outs))


def test_policy_loss_of_ratios_past_the_range_of_fp32():
    """A clipped ratio sends no gradient however large it is, and an advantage of 0 no loss."""
    for gap, adv, want in ((200.0, 1.0, -1.28), (1000.0, 1.0, -1.28), (200.0, 0.0, 0.0), (-200.0, -1.0, 0.8)):
        lp = torch.tensor([[gap, -0.5]], requires_grad=True)
        old = torch.tensor([[0.0, -0.5]])
        out = O.policy_loss(lp, old, torch.tensor([[adv, 2.0]]), clip_low=0.2, clip_high=0.28)
        (grad,) = torch.autograd.grad(out.loss, lp)
        assert abs(out.loss.item() - (want - 2.0) / 2) < 1e-6 and out.clip_fraction.item() == (0.5 if adv else 0.0)
        assert grad.tolist() == [[0.0, -1.0]]


def test_preference_loss_formula_and_gradient():
    torch.manual_seed(2)
    P, S = 3, 8
    logp = -torch.rand(2 * P, S).double()
    ref = logp + torch.randn(2 * P, S)
    mask = torch.rand(2 * P, S) < 0.6
    mask[4] = False
    ref[~mask] = float("inf")
    for average in (False, True):
        def fn(x):
            return O.preference_loss(x, ref_logp=ref, mask=mask, beta=0.7, label_smoothing=0.2, average=average).loss
        r = torch.where(mask, logp - ref, torch.zeros_like(logp)).sum(1)
        r = 0.7 * (r / mask.sum(1).clamp_min(1) if average else r)
        gap = r[:P] - r[P:]
        want = -(0.8 * torch.sigmoid(gap).log() + 0.2 * torch.sigmoid(-gap).log()).mean()
        assert torch.allclose(fn(logp), want)
        _differences(fn, logp)


def test_preference_loss_of_impossible_tokens():
    """A rejected token of probability zero: an infinite gap, and a loss of 0 with unsmoothed labels.  A chosen one:
    an infinite loss with the gradient of a certain error."""
    inf = float("inf")
    for side, smoothing, want, grads in ((2, 0.0, 0.0, (0.0, 0.0)), (0, 0.0, inf, (-0.5, 0.5)), (2, 0.25, inf, (0.125, -0.125)),
                                         (0, 0.25, inf, (-0.375, 0.375)), (0, 1.0, 0.0, (0.0, 0.0)), (2, 1.0, inf, (0.5, -0.5))):
        lp = torch.zeros(4, 6)
        lp[side, 3] = -inf  # pair 0; pair 1 has a gap of 0
        lp.requires_grad_(True)
        out = O.preference_loss(lp, beta=1.0, label_smoothing=smoothing)
        (grad,) = torch.autograd.grad(out.loss, lp)
        assert out.loss.item() == want if want else abs(out.loss.item() - 0.5 * 0.6931471805599453) < 1e-6
        assert grad[0].tolist() == [grads[0]] * 6 and grad[2].tolist() == [grads[1]] * 6
        assert torch.isfinite(grad).all()


def test_policy_and_preference_refusals():
    x = torch.zeros(4, 5)
    with pytest.raises(ValueError):
        O.policy_loss(x, x, x, reduction="sum")
    with pytest.raises(ValueError):
        O.policy_loss(x[0], x[0], x[0])
    with pytest.raises(ValueError):
        O.policy_loss(x, x, x[:, :3])
    with pytest.raises(TypeError):
        O.policy_loss(x, x.double(), x)
    with pytest.raises(ValueError):
        O.preference_loss(x[:3])
    with pytest.raises(ValueError):
        O.preference_loss(x, mask=x)


def test_distillation_of_values_at_the_end_of_their_range():
    """Masks of the type's lowest value, in the student's logits and in the teacher's, at a temperature below 1."""
    low = torch.finfo(torch.float32).min
    x, top = torch.randn(3, 6), torch.rand(3, 2)
    x[0, 3:], x[1], top[2] = low, low, low
    ids = torch.tensor([[0, 2]] * 3)
    x.requires_grad_(True)
    loss = O.distillation_loss(x, top, ids, temperature=0.5)
    (grad,) = torch.autograd.grad(loss, x)
    lp = torch.log_softmax(x.detach().double() / 0.5, 1).gather(1, ids)
    lq = torch.log_softmax(top.double() / 0.5, 1)
    want = 0.25 * (lq.exp() * (lq - lp)).sum(1).mean()
    assert abs(loss.item() - want.item()) < 1e-6 and torch.isfinite(grad).all()
    assert grad[0, 3:].abs().max() == 0 and grad[1].sum().abs() < 1e-6


def test_distillation_loss_formula_and_gradient():
    torch.manual_seed(3)
    T, V, K, tau = 6, 11, 4, 1.7
    logits, top = torch.randn(T, V).double(), torch.randn(T, K).double()
    ids = torch.randint(0, V, (T, K))
    ids[0], top[0] = torch.tensor([2, 2, 5, -1]), torch.tensor([1.0, 0.5, 2.0, float("nan")])
    ids[1] = -100
    mask = torch.tensor([True, True, False, True, True, True])
    logits[2] = float("nan")

    def fn(x):
        return O.distillation_loss(torch.where(mask[:, None], x, logits), top, ids, mask=mask, temperature=tau)

    want = 0.0
    for t in (0, 3, 4, 5):
        k = [i for i in range(K) if ids[t, i] >= 0]
        q = torch.softmax(top[t, k] / tau, 0)
        p = torch.softmax(logits[t] / tau, 0)
        want += tau ** 2 * sum(q[j] * (q[j].log() - p[ids[t, i]].log()) for j, i in enumerate(k)) / 4
    x = torch.where(torch.isnan(logits), torch.zeros_like(logits), logits)
    assert torch.allclose(fn(x), want)
    _differences(fn, x)


def test_lm_head_distillation_plain_and_refusals():
    torch.manual_seed(4)
    h, w = torch.randn(2, 3, 8, requires_grad=True), torch.randn(9, 8, requires_grad=True)
    top, ids = torch.randn(2, 3, 2), torch.randint(0, 9, (2, 3, 2))
    a = O.lm_head_distillation(h, w, top, ids, temperature=1.3)
    b = O.distillation_loss(h @ w.t(), top, ids.int(), temperature=1.3)
    assert torch.allclose(a, b)
    a.backward()
    assert torch.isfinite(h.grad).all() and torch.isfinite(w.grad).all()
    x = (h @ w.t()).detach()
    assert O.distillation_loss(x, top, ids, mask=torch.zeros(2, 3, dtype=torch.bool)).item() == 0
    with pytest.raises(IndexError):
        O.distillation_loss(x, top, ids + 9)
    with pytest.raises(ValueError):
        O.distillation_loss(x, top[:1], ids[:1])
    with pytest.raises(ValueError):
        O.distillation_loss(x, top, ids, temperature=0)
    with pytest.raises(TypeError):
        O.distillation_loss(x, top, ids.float())
    with pytest.raises(ValueError):
        O.lm_head_distillation(h, w[:, :4], top, ids)


@pytest.mark.parametrize("objective", ["policy", "preference", "distill"])
def test_post_training_example_on_cpu(objective):
    """The example's loop through the engine: the loss falls, and the first step's statistics are those of a policy
    that still is its own reference."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "post_training.py")
    spec = importlib.util.spec_from_file_location("post_training", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    history = mod.main([objective, "--steps", "4", "--device", "cpu"])
    assert history[-1]["loss"] < history[0]["loss"]
    if objective == "policy":
        assert history[0]["kl"] == 0 and history[0]["clipped"] == 0
    if objective == "preference":
        assert abs(history[0]["loss"] - 0.6931) < 1e-3 and history[-1]["reward_gap"] > 0


def test_model_objectives_match_its_logits_and_refuse_mixtures():
    from parallel_b200.models.config import resolve_config
    from parallel_b200.models.qwen3 import build_model

    m = build_model(resolve_config("tiny-qwen3"), dtype=torch.float32, seed=0)
    x = torch.randint(0, 1024, (2, 9), generator=torch.Generator().manual_seed(0))
    targets = torch.randint(0, 1024, (2, 9), generator=torch.Generator().manual_seed(1))
    targets[0, :3] = -100
    logits = m(input_ids=x).logits
    out = m(input_ids=x, targets=targets, temperature=0.8)
    want = torch.log_softmax(logits / 0.8, -1).gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    assert out.logits is None and out.loss is None
    assert torch.allclose(out.log_probs, want.masked_fill(targets < 0, 0.0), atol=1e-5)
    top = logits.detach().topk(4, dim=-1)
    out = m(input_ids=x, teacher=(top.values, top.indices, targets >= 0), temperature=2.0)
    ref = O.distillation_loss(logits, top.values, top.indices, mask=targets >= 0, temperature=2.0)
    assert torch.allclose(out.loss, ref, atol=1e-6) and out.logits is None
    with pytest.raises(ValueError):
        m(input_ids=x, labels=x, targets=targets)
    with pytest.raises(ValueError):
        m(input_ids=x, targets=targets, teacher=(top.values, top.indices, None))


def _fsdp_preference_worker(rank, world, out):
    """Each rank holds one pair (two sequences) of the batch; four preference steps under FSDP."""
    from dist_utils import cpu_cfg
    from parallel_b200.models.config import resolve_config
    from parallel_b200.models.qwen3 import build_model
    from parallel_b200.parallel.engine import ParallelEngine
    from parallel_b200.state import ParallelConfig

    cfg = cpu_cfg(**{"parallel.dp_shard": world, "engine.activation_checkpoint": "true"})
    pc = ParallelConfig(cfg)
    pc.set_device_mesh("cpu")
    m = build_model(resolve_config("tiny-qwen3"), dtype=torch.float32, seed=0)
    eng = ParallelEngine(m, None, pc, cfg, torch.device("cpu"))
    tok = torch.randint(0, 1024, (2 * world, 33), generator=torch.Generator().manual_seed(5))
    mine = tok[[rank, world + rank]]  # the chosen and the rejected sequence of this rank's pair
    x, y = mine[:, :-1], mine[:, 1:]
    with torch.no_grad():
        ref = eng.log_probs(x, y).log_probs
    losses = []
    for _ in range(4):
        loss = O.preference_loss(eng.log_probs(x, y).log_probs, ref_logp=ref).loss
        eng.backward(loss)
        eng.step()
        losses.append(eng.reduce_loss(loss.detach().clone()).item())
    if rank == 0:
        torch.save({"losses": losses}, out)


def test_preference_training_under_fsdp_equals_one_process(tmp_path):
    from dist_utils import run_ranks

    out = str(tmp_path / "out.pt")
    run_ranks(_fsdp_preference_worker, 2, out)
    sharded = torch.load(out, weights_only=False)

    from parallel_b200.models.config import resolve_config
    from parallel_b200.models.qwen3 import build_model
    from parallel_b200.parallel.optim import FusedAdamW

    m = build_model(resolve_config("tiny-qwen3"), dtype=torch.float32, seed=0)
    opt = FusedAdamW(list(m.parameters()), lr=1e-3, betas=(0.9, 0.999), weight_decay=0.01)
    tok = torch.randint(0, 1024, (4, 33), generator=torch.Generator().manual_seed(5))
    x, y = tok[:, :-1], tok[:, 1:]
    with torch.no_grad():
        ref = m(input_ids=x, targets=y).log_probs
    for want in sharded["losses"]:
        loss = O.preference_loss(m(input_ids=x, targets=y).log_probs, ref_logp=ref).loss
        loss.backward()
        torch.nn.utils.clip_grad_norm_(list(m.parameters()), 1.0)
        opt.step()
        opt.zero_grad(set_to_none=True)
        assert abs(loss.item() - want) < 1e-5
