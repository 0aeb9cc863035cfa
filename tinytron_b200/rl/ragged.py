"""Group-relative policy optimisation on answers of different lengths, packed.

``make_ragged_rollout`` lays a ragged generation's sequences end to end (no padding, no
prompt repeated in the cache), ``ragged_grpo_loss`` scores them with the actor in one packed
forward pass: attention within each sequence, and log-probs, entropy and alternatives of the
answer tokens from one pass over the logits.  The objective and its metrics are those of
:func:`tinytron_b200.rl.losses.grpo_loss`.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .losses import grpo_loss
from .types import RLLossOutput


@dataclass
class RaggedRollout:
    """Sequences packed end to end: ``tokens`` [N], ``cu_seqlens`` int32 [S + 1]; ``labels`` [N] is the next token
    where it belongs to the answer (``ignore_index`` elsewhere), ``old_log_probs`` [N] the sampler's log-prob of that
    token, ``sequence`` [N] the row's sequence."""

    tokens: torch.Tensor
    cu_seqlens: torch.Tensor
    labels: torch.Tensor
    old_log_probs: torch.Tensor
    sequence: torch.Tensor
    max_seqlen: int
    ignore_index: int = -100


def make_ragged_rollout(generation, ignore_index: int = -100) -> RaggedRollout:
    """The packed form of a :class:`~tinytron_b200.inference.ragged.RaggedGeneration`."""
    dev = generation.new_tokens.device
    lens = generation.lengths.tolist()
    seqs = generation.sequences()
    labels, old = [], []
    for i, (s, n) in enumerate(zip(seqs, lens)):
        # row t predicts token t + 1: the answer's n tokens are predicted by the n rows before the last
        lab = torch.full_like(s, ignore_index)
        lab[-n - 1:-1] = s[-n:]
        lp = torch.zeros(s.numel(), dtype=torch.float32, device=dev)
        lp[-n - 1:-1] = generation.sampler_log_probs[i, :n]
        labels.append(lab)
        old.append(lp)
    total = [s.numel() for s in seqs]
    cu = torch.tensor([0, *total], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
    owner = torch.arange(len(seqs), device=dev).repeat_interleave(torch.tensor(total, device=dev))
    return RaggedRollout(torch.cat(seqs), cu, torch.cat(labels), torch.cat(old), owner, max(total), ignore_index)


def ragged_grpo_loss(model, rollout: RaggedRollout, advantages: torch.Tensor, clip_range: float = 0.2,
                     entropy_coef: float = 0.0, temperature: float = 1.0) -> RLLossOutput:
    """GRPO objective of the packed answers (``advantages`` [S], one per sequence), less ``entropy_coef`` times the
    mean entropy of the scored positions; metrics also carry that mean.  On CUDA, offsets or labels out of range are found
    on the device: call ``ops.check_status()`` before stepping on the gradients."""
    if tuple(advantages.shape) != (rollout.cu_seqlens.numel() - 1,):
        raise ValueError(f"advantages must have one entry per sequence ({rollout.cu_seqlens.numel() - 1}), got {tuple(advantages.shape)}")
    stats = model.packed_token_stats(rollout.tokens, rollout.labels, rollout.cu_seqlens, max_seqlen=rollout.max_seqlen,
                                     temperature=temperature, ignore_index=rollout.ignore_index)
    mask = rollout.labels.ne(rollout.ignore_index).to(torch.float32)
    adv = advantages.to(stats.log_probs.dtype)[rollout.sequence]
    out = grpo_loss(stats.log_probs, rollout.old_log_probs, adv, mask, clip_range=clip_range)
    entropy = (stats.entropy * mask).sum() / mask.sum().clamp_min(1.0)
    metrics = dict(out.metrics, entropy=entropy.detach())
    return RLLossOutput(loss=out.loss - entropy_coef * entropy if entropy_coef else out.loss, metrics=metrics)
