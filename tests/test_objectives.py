"""Post-training objectives on CPU: the plain formulas and the refusals."""
import pytest
import torch

from parallel_b200.ops import objectives as O




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
