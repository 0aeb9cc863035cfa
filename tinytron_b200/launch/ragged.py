"""Ragged rollouts and packed policy updates, end to end on one device:

    python -m tinytron_b200.launch.ragged --num_prompts 8 --prompt_len 16 200 --num_samples 4 --steps 3

Each step draws seeded prompts of different lengths, prefills them packed, forks every prompt's
pages into ``--num_samples`` answers, decodes them over the paged cache, rewards the answers
(tokens close to a target id, as the RL entry point's rule reward), and takes one AdamW step on
the packed GRPO objective with an entropy bonus.
"""
from __future__ import annotations

import argparse
import time

import torch

from tinytron_b200 import ops
from tinytron_b200.inference import InferenceEngine
from tinytron_b200.models import GPT
from tinytron_b200.models.config import add_model_config_args, build_model_config
from tinytron_b200.rl import group_advantages, make_ragged_rollout, ragged_grpo_loss

from ._presets import expand_preset


def build_parser() -> argparse.ArgumentParser:
    p = add_model_config_args(argparse.ArgumentParser("ragged", allow_abbrev=False))
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--seed", type=int, default=1337)
    p.add_argument("--num_prompts", type=int, default=8)
    p.add_argument("--prompt_len", type=int, nargs=2, default=(16, 256), metavar=("MIN", "MAX"))
    p.add_argument("--num_samples", type=int, default=4)
    p.add_argument("--max_new_tokens", type=int, default=32)
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--eos_token_id", type=int, default=None)
    p.add_argument("--alternatives", type=int, default=4)
    p.add_argument("--steps", type=int, default=2)
    p.add_argument("--lr", type=float, default=1e-5)
    p.add_argument("--entropy_coef", type=float, default=0.0)
    p.add_argument("--kv_cache_page_size", type=int, default=128)
    return p


def main(argv: list[str] | None = None) -> list[dict]:
    args = build_parser().parse_args(expand_preset(argv))
    cfg = build_model_config(args, seed=args.seed)
    engine = InferenceEngine(cfg, device=args.device, kv_cache_page_size=args.kv_cache_page_size)
    actor = GPT(cfg, device=engine.device)
    optim = torch.optim.AdamW(actor.parameters(), lr=args.lr)
    g = torch.Generator().manual_seed(args.seed)
    torch.manual_seed(args.seed)
    log = []
    for step in range(args.steps):
        engine.model.load_state_dict(actor.state_dict())
        lo, hi = args.prompt_len
        prompts = [torch.randint(0, cfg.vocab_size, (int(torch.randint(lo, hi + 1, (1,), generator=g)),), generator=g)
                   for _ in range(args.num_prompts)]
        t0 = time.perf_counter()
        gen = engine.generate_ragged(prompts, args.max_new_tokens, num_samples=args.num_samples,
                                     temperature=args.temperature, eos_token_id=args.eos_token_id,
                                     alternatives=args.alternatives)
        new = int(gen.lengths.sum())
        t1 = time.perf_counter()
        near = 1.0 - gen.new_tokens.float() / max(cfg.vocab_size - 1, 1)
        inside = torch.arange(near.shape[1], device=near.device) < gen.lengths[:, None]
        rewards = (near * inside).sum(1) / gen.lengths
        rollout = make_ragged_rollout(gen)
        out = ragged_grpo_loss(actor, rollout, group_advantages(rewards, args.num_samples), entropy_coef=args.entropy_coef,
                               temperature=args.temperature)
        optim.zero_grad(set_to_none=True)
        out.loss.backward()
        if engine.device.type == "cuda":
            ops.check_status(engine.device)  # no step on gradients of skipped entries
        optim.step()
        loss = float(out.loss.detach())
        t2 = time.perf_counter()
        log.append({"step": step, "loss": loss, "reward": float(rewards.mean()), "entropy": float(out.metrics["entropy"]),
                    "new_tokens": new, "packed_tokens": rollout.tokens.numel(), "rollout_s": t1 - t0, "update_s": t2 - t1})
        print(" ".join(f"{k}: {v:.4f}" if isinstance(v, float) else f"{k}: {v}" for k, v in log[-1].items()), flush=True)
    return log


if __name__ == "__main__":
    main()
