"""Differentiable post-training objectives: what a trained language model is tuned with after pre-training.

* ``lm_head_log_probs``  log-probabilities of given tokens through the LM head,
  for scoring (no gradient: the logits are never stored) and for training;
* ``policy_loss``        clipped policy-gradient loss with a KL term over token
  log-probabilities;
* ``preference_loss``    loss on paired sequences (log-ratio of the chosen and
  the rejected one against a reference);
* ``distillation_loss``  distillation of given logits from a teacher's top
  logits, and ``lm_head_distillation``, the same through the LM head.

As in ``functional``, CUDA tensors run the sm_100a kernels and CPU tensors run
the plain PyTorch statement of the same formula.  The kernels have first-order
gradients; forward-mode derivatives are refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from ._ext import ext


def _rows_bf16(t: torch.Tensor, what: str) -> torch.Tensor:
    """``t`` as bf16 rows that TMA can read: unit inner stride, 16-byte row
    stride and base, no row inside another (a copy if it has another layout)."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be bfloat16 on CUDA, got {t.dtype}")
    if t.stride(-1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _check_temperature(temperature) -> None:
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"temperature has to be positive and finite, got {temperature}")


def _check_head(h: torch.Tensor, w: torch.Tensor) -> None:
    if w.dim() != 2 or h.dim() < 1 or h.shape[-1] != w.shape[1]:
        raise ValueError(f"h {tuple(h.shape)} and w {tuple(w.shape)} must share their last dimension")
    if w.numel() == 0:
        raise ValueError(f"w {tuple(w.shape)} has no entry")


# ----------------------------------------------------------------- log-probabilities through the LM head
def lm_head_log_probs(h: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, temperature: float = 1.0,
                      max_block_bytes: int = 6 << 30) -> torch.Tensor:
    """fp32 ``log_softmax(h @ w.T / temperature)[..., ids]``, shaped as ``ids``.

    h [..., H] hidden states, w [V, H] the LM head, ids int64 with one entry
    per row of h.  A negative id (``IGNORE_INDEX``) marks a row without a
    token: its log-probability is 0 and it sends back no gradient.  An id >= V
    gives NaN (an ``IndexError`` on CPU).  The gradient goes to h and w; one
    backward pass per forward.  ``max_block_bytes`` bounds the [rows, V] block
    held between forward and backward; rows beyond it are computed twice.  On
    CUDA a row's log-probability has the same bits in whatever batch it comes."""
    _check_temperature(temperature)
    _check_head(h, w)
    if ids.dtype != torch.int64 or ids.numel() * h.shape[-1] != h.numel():
        raise ValueError(f"ids must be int64 with one entry per row of h, got {ids.dtype} {tuple(ids.shape)} for "
                         f"{tuple(h.shape)}")
    h2, flat = h.reshape(-1, h.shape[-1]), ids.reshape(-1).contiguous()
    if not h2.is_cuda:
        return _log_probs_plain(h2, w, flat, temperature).view(ids.shape)
    if flat.numel() == 0:
        return (h2.float().sum(-1) + w[:0].float().sum()).view(ids.shape)
    h2, w = _rows_bf16(h2, "h"), _rows_bf16(w, "w")
    return ext().lm_head_log_probs(h2, w, flat, 1.0 / float(temperature), int(max_block_bytes)).view(ids.shape)


def _log_probs_plain(h, w, ids, temperature):
    if ids.numel() and int(ids.max()) >= w.shape[0]:
        raise IndexError(f"token id {int(ids.max())} is outside the vocabulary of {w.shape[0]}")
    rows = (ids >= 0).nonzero()[:, 0]
    logp = torch.log_softmax(F.linear(h[rows], w).float() / temperature, dim=-1)
    picked = logp.gather(1, ids[rows][:, None])[:, 0]
    return torch.zeros(ids.shape, dtype=torch.float32, device=h.device).index_put((rows,), picked)


# ----------------------------------------------------------------- losses over token log-probabilities
class PolicyLoss(NamedTuple):
    loss: torch.Tensor           # scalar, differentiable in logp
    clip_fraction: torch.Tensor  # share of the tokens whose ratio was clipped
    kl: torch.Tensor             # mean over the tokens of the KL estimate (0 without a reference)


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor     # scalar, differentiable in logp
    rewards: torch.Tensor  # [2P] beta x log ratio of each sequence (chosen rows, then rejected rows)


def _tokens(t: torch.Tensor | None, like: torch.Tensor, what: str) -> torch.Tensor | None:
    """[B, S] of logp's type, rows of unit inner stride."""
    if t is None:
        return None
    if t.dtype != like.dtype:
        raise TypeError(f"{what} must be {like.dtype}, got {t.dtype}")
    if t.shape != like.shape:
        raise ValueError(f"{what} {tuple(t.shape)} must have logp's shape {tuple(like.shape)}")
    return t if t.stride(-1) == 1 else t.contiguous()


def _check_logp(logp: torch.Tensor, mask: torch.Tensor | None) -> None:
    if logp.dim() != 2 or (logp.is_cuda and logp.dtype != torch.float32) or not logp.is_floating_point():
        raise ValueError(f"logp must be fp32 [sequences, tokens], got {logp.dtype} {tuple(logp.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != logp.shape):
        raise ValueError(f"mask must be bool {tuple(logp.shape)}, got {mask.dtype} {tuple(mask.shape)}")


def _unit_inner(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def policy_loss(logp: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                mask: torch.Tensor | None = None, ref_logp: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, reduction: str = "token") -> PolicyLoss:
    """Clipped policy loss of token log-probabilities, logp fp32 [B, S], in 64 bits and rounded once.

    With r = exp(logp - old_logp) and advantage A, a token's loss is
    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef k`` with
    ``k = exp(ref_logp - logp) - (ref_logp - logp) - 1``.  advantages: [B, S],
    or [B] / [B, 1] for one value per sequence.  mask (bool [B, S]) selects the
    tokens that count; the others may hold anything.  ``reduction``: "token" is
    the mean over all tokens that count, "sequence" the mean over sequences
    (those with a token that counts) of their token means; without any token
    the loss is 0.  The gradient goes to logp alone; where the ratio stands
    exactly on the edge of the clip range it is that of the unclipped side."""
    _check_logp(logp, mask)
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction has to be 'token' or 'sequence', got {reduction!r}")
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError(f"clip range: 0 <= clip_low <= 1 and clip_high >= 0, got {clip_low} and {clip_high}")
    B, S = logp.shape
    adv = advantages if advantages.dim() != 1 else advantages[:, None]
    if adv.dtype != logp.dtype:
        raise TypeError(f"advantages must be {logp.dtype}, got {adv.dtype}")
    if tuple(adv.shape) not in ((B, S), (B, 1)):
        raise ValueError(f"advantages {tuple(advantages.shape)}: [{B}, {S}], [{B}, 1] or [{B}] expected")
    old, ref = _tokens(old_logp, logp, "old_logp"), _tokens(ref_logp, logp, "ref_logp")
    low, high, per_sequence = 1.0 - clip_low, 1.0 + clip_high, reduction == "sequence"
    if not logp.is_cuda:
        return _policy_plain(logp, old.detach(), adv.detach().expand(B, S), mask,
                             None if ref is None else ref.detach(), low, high, kl_coef, per_sequence)
    return PolicyLoss(*ext().policy_loss(_unit_inner(logp), old, adv, _unit_inner(mask), ref, low, high,
                                         float(kl_coef), per_sequence))


def _policy_plain(logp, old, adv, mask, ref, low, high, kl_coef, per_sequence):
    m = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask
    at = m.nonzero(as_tuple=True)  # the tokens that count; the others never enter
    x, a = logp[at].double(), adv[at].double()
    gap = x - old[at]
    with torch.no_grad():
        ratio = torch.exp(gap)
        c = ratio.clamp(low, high) * a
        clipped = ratio * a > c
    # the ratio of a clipped token stays out of the graph: it may be infinite
    per = -torch.where(clipped, c, torch.exp(gap.masked_fill(clipped, 0.0)) * a)
    kl = torch.zeros_like(x)
    if ref is not None:
        d = ref[at] - x
        kl = torch.expm1(d) - d
        if kl_coef:  # without the term the estimate may be infinite
            per = per + kl_coef * kl
    n = max(1, x.numel())
    if per_sequence:
        rows = m.sum(1)
        weight = (1.0 / rows.clamp_min(1).to(x.dtype) / max(1, int((rows > 0).sum())))[at[0]]
    else:
        weight = 1.0 / n
    out = (per * weight).sum(), clipped.double().sum() / n, kl.detach().sum() / n
    return PolicyLoss(*(t.to(logp.dtype) for t in out))


def preference_loss(logp: torch.Tensor, ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                    beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False) -> PreferenceLoss:
    """Loss on pairs of sequences from token log-probabilities, logp fp32 [2P, S].

    Row p is the chosen sequence of pair p and row P + p the rejected one.  A
    sequence's reward is ``beta`` times the sum (``average``: the mean) over
    its tokens in ``mask`` of logp - ref_logp (ref_logp None: logp alone), the
    gap d of a pair is the difference of its rewards, and the loss the mean
    over pairs of ``-(1 - label_smoothing) log sigmoid(d) - label_smoothing
    log sigmoid(-d)``.  Positions outside the mask may hold anything; a row
    without a token has reward 0.  The gradient goes to logp alone."""
    _check_logp(logp, mask)
    if logp.shape[0] < 2 or logp.shape[0] % 2:
        raise ValueError(f"logp holds P chosen rows and P rejected rows, got {logp.shape[0]} rows")
    if not 0.0 <= label_smoothing <= 1.0 or not math.isfinite(beta):
        raise ValueError(f"0 <= label_smoothing <= 1 and a finite beta, got {label_smoothing} and {beta}")
    ref = _tokens(ref_logp, logp, "ref_logp")
    if not logp.is_cuda:
        return _preference_plain(logp, None if ref is None else ref.detach(), mask, beta, label_smoothing, average)
    return PreferenceLoss(*ext().preference_loss(_unit_inner(logp), ref, _unit_inner(mask), float(beta),
                                                 float(label_smoothing), bool(average)))


def _preference_plain(logp, ref, mask, beta, smoothing, average):
    m = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask
    at = m.nonzero(as_tuple=True)
    diff = logp[at] - (0.0 if ref is None else ref[at])
    sums = torch.zeros(logp.shape[0], dtype=logp.dtype, device=logp.device).index_add(0, at[0], diff)
    rewards = beta * (sums / m.sum(1).clamp_min(1).to(logp.dtype) if average else sums)
    P = logp.shape[0] // 2
    gap = rewards[:P] - rewards[P:]
    # a side that does not count enters neither: its loss may be infinite
    sides = [share * F.logsigmoid(side) for share, side in ((1.0 - smoothing, gap), (smoothing, -gap)) if share]
    return PreferenceLoss(-sum(sides).mean(), rewards.detach())


# ----------------------------------------------------------------- distillation from a teacher's top logits
def _check_teacher(rows, top_logits, top_ids, mask, temperature):
    """Teacher entries as [T, K] and the mask as [T] for `rows` (the leading shape of the student's rows)."""
    _check_temperature(temperature)
    if top_logits.shape[:-1] != rows or top_ids.shape != top_logits.shape or top_logits.dim() < 1:
        raise ValueError(f"teacher logits {tuple(top_logits.shape)} and ids {tuple(top_ids.shape)}: "
                         f"[{', '.join(str(r) for r in rows)}, K] expected")
    if top_logits.shape[-1] < 1:
        raise ValueError("at least one teacher entry per row")
    if top_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"teacher ids must be int64 or int32, got {top_ids.dtype}")
    if not top_logits.is_floating_point() or (top_logits.is_cuda and top_logits.dtype not in (torch.bfloat16,
                                                                                              torch.float32)):
        raise TypeError(f"teacher logits must be bf16 or fp32, got {top_logits.dtype}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != rows):
        raise ValueError(f"mask must be bool {tuple(rows)}, got {mask.dtype} {tuple(mask.shape)}")
    K = top_logits.shape[-1]
    top, ids = top_logits.detach(), top_ids
    if top.dim() != 2:
        top, ids = top.reshape(-1, K), ids.reshape(-1, K)
    top, ids = _unit_inner(top), _unit_inner(ids)
    return top, ids, mask if mask is None or mask.dim() == 1 else mask.reshape(-1)


def distillation_loss(logits: torch.Tensor, top_logits: torch.Tensor, top_ids: torch.Tensor,
                      mask: torch.Tensor | None = None, temperature: float = 1.0) -> torch.Tensor:
    """Mean over rows of the KL divergence from a teacher's top tokens to the student, a scalar in fp32.

    logits [..., V] (bf16 or fp32) are the student's; top_logits [..., K]
    (bf16 or fp32) and top_ids [..., K] (int64 or int32) the teacher's highest
    logits and their tokens, an id < 0 marking an absent entry (K at most 1024
    on CUDA).  With q = softmax(top_logits / temperature) over the entries
    present and p = softmax(logits / temperature) over the vocabulary, a row's
    loss is ``temperature^2 sum_k q_k (log q_k - log p[id_k])``; an id that comes
    twice counts twice.  Rows outside mask (bool [...]) and rows without an
    entry do not count, and may hold anything; without any row the loss is 0.
    An id >= V makes the loss NaN (an ``IndexError`` on CPU).  The gradient
    goes to logits alone; one backward pass per forward, until which the logits
    stay as they are."""
    top, ids, m = _check_teacher(logits.shape[:-1], top_logits, top_ids, mask, temperature)
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    tau = float(temperature)
    if not x.is_cuda:
        return _distillation_plain(x, top, ids, m, tau)
    return ext().distillation_loss(_unit_inner(x), top, ids, m, tau)


def lm_head_distillation(h: torch.Tensor, w: torch.Tensor, top_logits: torch.Tensor, top_ids: torch.Tensor,
                         mask: torch.Tensor | None = None, temperature: float = 1.0,
                         max_block_bytes: int = 6 << 30) -> torch.Tensor:
    """``distillation_loss(h @ w.T, ...)`` for hidden states h [..., H] and the LM head w [V, H], with bf16 logits.  At
    most ``max_block_bytes`` of them are held at a time, the first block's until the backward pass; logits of rows
    beyond it are computed twice.  The gradient goes to h and w; one backward pass per forward."""
    _check_head(h, w)
    top, ids, m = _check_teacher(h.shape[:-1], top_logits, top_ids, mask, temperature)
    h2, tau = h.reshape(-1, h.shape[-1]), float(temperature)
    if not h2.is_cuda:
        return _distillation_plain(F.linear(h2, w), top, ids, m, tau)
    if h2.shape[0] == 0:
        return h2.float().sum() + w[:0].float().sum()
    h2, w = _rows_bf16(h2, "h"), _rows_bf16(w, "w")
    return ext().lm_head_distillation(h2, w, top, ids, m, tau, int(max_block_bytes))


def _distillation_plain(x, top, ids, mask, tau):
    if ids.numel() and int(ids.max()) >= x.shape[1]:
        raise IndexError(f"teacher id {int(ids.max())} is outside the vocabulary of {x.shape[1]}")
    dt = torch.promote_types(x.dtype, torch.float32)
    have = (ids >= 0) & (top != -math.inf)
    counts = have.any(1) if mask is None else have.any(1) & mask
    rows = counts.nonzero()[:, 0]
    have, ids = have[rows], ids[rows].clamp_min(0).long()
    # differences to the maximum before the temperature: values at the end of their type's range stay finite
    t, x = top[rows].to(dt).masked_fill(~have, -math.inf), x[rows].to(dt)
    log_q = torch.log_softmax((t - t.amax(1, keepdim=True)) / tau, dim=1)
    log_p = torch.log_softmax((x - x.detach().amax(1, keepdim=True)) / tau, dim=1).gather(1, ids)
    zero = torch.zeros((), dtype=dt, device=x.device)
    terms = torch.where(have, log_q.exp() * (torch.where(have, log_q, zero) - torch.where(have, log_p, zero)), zero)
    return tau * tau * terms.sum() / max(1, rows.numel())
