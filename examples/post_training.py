"""Post-training objectives on the training engine, on synthetic data.

    python examples/post_training.py policy|preference|distill [--steps N] [--device cuda|cpu] [--layers L]

* ``policy``      clipped policy optimisation: completions of a fixed batch are
  scored under the policy that "sampled" them and under the frozen reference,
  a toy reward (the share of even tokens) gives group-normalised advantages,
  and every step takes a clipped update with a KL term;
* ``preference``  preference tuning on pairs against the frozen reference;
* ``distill``     a student learns from another model's top 16 logits.

Prompts are masked out by targets of -100.  On CPU (fp32) the same calls run
their plain PyTorch form.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from parallel_b200.config import from_dotlist, load_cfg, merge  # noqa: E402
from parallel_b200.models.config import resolve_config  # noqa: E402
from parallel_b200.models.qwen3 import build_model  # noqa: E402
from parallel_b200.ops.objectives import policy_loss, preference_loss  # noqa: E402
from parallel_b200.parallel.engine import ParallelEngine  # noqa: E402
from parallel_b200.state import ParallelConfig  # noqa: E402

B, S, PROMPT, TOP_K = 8, 64, 16, 16


def make_engine(device: torch.device, layers: int, seed: int, lr: float):
    cuda = device.type == "cuda"
    cfg = merge(load_cfg(argv=[]), from_dotlist([f"config.device_type={device.type}", f"model.learning_rate={lr}",
                                                 f"config.use_amp={'true' if cuda else 'false'}"]))
    pc = ParallelConfig(cfg)
    pc.set_device_mesh(device.type)
    mcfg = resolve_config("small-qwen3" if cuda else "tiny-qwen3", num_hidden_layers=layers)
    model = build_model(mcfg, device=device, dtype=torch.bfloat16 if cuda else torch.float32, seed=seed)
    return ParallelEngine(model, None, pc, cfg, device), mcfg


def batch(vocab: int, device: torch.device, seed: int = 0):
    """Inputs, the token each position predicts (-100 in the prompt), and the mask of those that count."""
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, vocab, (B, S + 1), generator=gen).to(device)
    targets = tokens[:, 1:].clone()
    targets[:, :PROMPT] = -100
    return tokens[:, :-1].contiguous(), targets, targets >= 0


def run_policy(engine, x, targets, mask, steps):
    with torch.no_grad():
        old = engine.log_probs(x, targets).log_probs  # the policy that sampled is the reference too
    reward = ((targets % 2 == 0) & mask).sum(1).float() / mask.sum(1)
    advantages = (reward - reward.mean()) / (reward.std() + 1e-6)
    for step in range(steps):
        logp = engine.log_probs(x, targets).log_probs
        out = policy_loss(logp, old, advantages, mask=mask, ref_logp=old, clip_low=0.2, clip_high=0.28, kl_coef=0.02,
                          reduction="sequence")
        engine.backward(out.loss)
        engine.step()
        yield dict(step=step, loss=out.loss, clipped=out.clip_fraction, kl=out.kl)


def run_preference(engine, x, targets, mask, steps):
    with torch.no_grad():
        ref = engine.log_probs(x, targets).log_probs
    for step in range(steps):
        logp = engine.log_probs(x, targets).log_probs  # rows [0, B/2) are preferred to rows [B/2, B)
        out = preference_loss(logp, ref_logp=ref, mask=mask, beta=0.1)
        engine.backward(out.loss)
        engine.step()
        gap = (out.rewards[:B // 2] - out.rewards[B // 2:]).mean()
        yield dict(step=step, loss=out.loss, reward_gap=gap)


def run_distill(engine, x, targets, mask, steps, teacher):
    with torch.no_grad():
        logits = teacher(input_ids=x, return_logits=True).logits
    top_logits, top_ids = logits.float().topk(TOP_K, dim=-1)
    for step in range(steps):
        out = engine.distill(x, top_logits, top_ids, mask=mask, temperature=2.0)
        engine.backward(out.loss)
        engine.step()
        yield dict(step=step, loss=out.loss)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("objective", choices=["policy", "preference", "distill"])
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    args = ap.parse_args(argv)
    device = torch.device(args.device)
    engine, mcfg = make_engine(device, args.layers, seed=0, lr=3e-4 if args.objective == "distill" else 2e-5)
    x, targets, mask = batch(mcfg.vocab_size, device)
    if args.objective == "distill":
        dtype = torch.bfloat16 if device.type == "cuda" else torch.float32
        teacher = build_model(mcfg, device=device, dtype=dtype, seed=1)
        run = run_distill(engine, x, targets, mask, args.steps, teacher)
    else:
        run = (run_policy if args.objective == "policy" else run_preference)(engine, x, targets, mask, args.steps)
    history = []
    for row in run:
        row = {k: float(v.detach()) if torch.is_tensor(v) else v for k, v in row.items()}
        history.append(row)
        print("  ".join(f"{k} {v:.4f}" if k != "step" else f"step {int(v):3d}" for k, v in row.items()))
    return history


if __name__ == "__main__":
    main()
