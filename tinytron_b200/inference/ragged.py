"""A paged KV cache whose sequences have lengths of their own, and generation on it.

One pool of pages ``[layers, pages, page_size, Hkv, D]`` (keys and values apart) and one page
table ``[max_seqs, width]`` serve all layers.  Which page belongs to whom is decided on the
host (free pages, a reference count per page); the data moves on the device:

* prompts of different lengths are prefilled packed, in one forward pass;
* ``fork`` lets several continuations share a prompt's full pages and copies only the page
  that the next token falls into, so a group of answers holds its prompt once;
* ``free`` gives pages back as their last user goes, ``compact`` moves the pages in use to
  the front of the pool, ``resize`` gives the rest back;
* a decode step reads lengths and page table on the device, so it is captured once in a
  CUDA graph however the lengths differ.
"""
from __future__ import annotations

import heapq
from dataclasses import dataclass
from typing import NamedTuple, Sequence

import torch

from tinytron_b200 import ops
from tinytron_b200.parallel import parallel_state


class RaggedStep(NamedTuple):
    """What the layers of one forward pass over ragged tokens read: sequence b's tokens are rows
    [cu_seqlens[b], cu_seqlens[b + 1]), the first at position start[b].  With ``seq_lens`` (one token per
    sequence) attention reads the pages; without, the tokens are whole prompts and attend to each other."""

    cache: "RaggedKVCache"
    page_table: torch.Tensor
    cu_seqlens: torch.Tensor
    start: torch.Tensor
    seq_lens: torch.Tensor | None


class RaggedKVCache:
    def __init__(self, num_layers: int, num_heads: int, head_dim: int, num_pages: int, page_size: int, max_seqs: int,
                 max_seq_len: int, device, dtype):
        if min(num_layers, num_heads, head_dim, page_size, max_seqs, max_seq_len) <= 0 or num_pages < 0:
            raise ValueError("cache sizes must be positive")
        self.page_size = page_size
        self.max_seq_len = max_seq_len
        self.width = -(-max_seq_len // page_size)
        self.device = torch.device(device)
        shape = (num_layers, num_pages, page_size, num_heads, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.page_table = torch.full((max_seqs, self.width), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self._rows: list[list[int] | None] = [None] * max_seqs  # pages of each sequence (None: no sequence)
        self._lens = [0] * max_seqs
        self._refs = [0] * num_pages
        self._free = list(range(num_pages))  # heap: the lowest page first keeps the pool dense
        self._free_seqs = list(range(max_seqs))
        self._dirty = False  # the host's table is ahead of the device's
        self._workspaces: dict = {}

    @classmethod
    def from_model_config(cls, model_config, num_pages: int, page_size: int, max_seqs: int, device, dtype,
                          max_seq_len: int | None = None) -> "RaggedKVCache":
        return cls(model_config.num_layer, model_config.num_key_value_heads,
                   model_config.hidden_size // model_config.num_attention_heads, num_pages, page_size, max_seqs,
                   max_seq_len or model_config.block_size, device, dtype)

    # ------------------------------------------------------------------ bookkeeping
    @property
    def num_pages(self) -> int:
        return self.k_pages.shape[1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        self._check(seq)
        return self._lens[seq]

    def pages_of(self, seq: int) -> list[int]:
        self._check(seq)
        return list(self._rows[seq])

    def _check(self, *seqs: int) -> None:
        for s in seqs:
            if not 0 <= s < len(self._rows) or self._rows[s] is None:
                raise ValueError(f"no sequence {s} in the cache")

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise RuntimeError(f"KV cache page pool exhausted: {n} pages needed, {len(self._free)} free")
        pages = [heapq.heappop(self._free) for _ in range(n)]
        for p in pages:
            self._refs[p] = 1
        return pages

    def _sync(self) -> None:
        if not self._dirty:
            return
        rows = [(r or []) + [-1] * (self.width - len(r or [])) for r in self._rows]
        self.page_table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.seq_lens.copy_(torch.tensor(self._lens, dtype=torch.int32))
        self._dirty = False

    # ------------------------------------------------------------------ sequences
    def add(self, count: int = 1) -> list[int]:
        """Empty sequences; their numbers are rows of ``page_table``."""
        if count > len(self._free_seqs):
            raise RuntimeError(f"KV cache holds at most {len(self._rows)} sequences")
        out = [heapq.heappop(self._free_seqs) for _ in range(count)]
        for s in out:
            self._rows[s], self._lens[s] = [], 0
        self._dirty = True
        return out

    def reserve(self, seqs: Sequence[int], tokens: Sequence[int]) -> None:
        """Map pages for the next ``tokens[i]`` positions of ``seqs[i]`` (all or, if the pool cannot, none)."""
        self._check(*seqs)
        want = []
        for s, n in zip(seqs, tokens, strict=True):
            if n < 0:
                raise ValueError(f"sequence {s}: {n} tokens")
            end = self._lens[s] + n
            if end > self.max_seq_len:
                raise ValueError(f"KV cache overflow: requested sequence length {end}, max supported is {self.max_seq_len}")
            want.append(max(0, -(-end // self.page_size) - len(self._rows[s])))
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        pages = self._take(sum(want))
        for s, n in zip(seqs, want):
            self._rows[s].extend(pages[:n])
            del pages[:n]
            self._dirty |= n > 0

    def advance(self, seqs: Sequence[int], tokens: Sequence[int]) -> None:
        """Commit tokens whose keys and values have been written."""
        self._check(*seqs)
        for s, n in zip(seqs, tokens, strict=True):
            if n < 0:
                raise ValueError(f"sequence {s}: {n} tokens")
            if self._lens[s] + n > len(self._rows[s]) * self.page_size:
                raise ValueError(f"sequence {s}: length {self._lens[s] + n} is past its mapped pages")
            self._lens[s] += n
        self._dirty = True

    def fork(self, parents: Sequence[int]) -> list[int]:
        """A copy of each of ``parents`` (one may be named several times): full pages are shared, a partly filled
        last page is copied.  Pages that a parent has reserved past its length stay the parent's."""
        self._check(*parents)
        if not parents:
            return []
        part = [self._lens[p] % self.page_size for p in parents]
        if sum(1 for x in part if x) > len(self._free) or len(parents) > len(self._free_seqs):
            raise RuntimeError("KV cache page pool or sequence table exhausted")
        kids = self.add(len(parents))
        fresh = [self._take(1)[0] if x else -1 for x in part]
        try:
            self._sync()
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
            ops.fork_pages(self.k_pages, self.v_pages, self.page_table, self.seq_lens, i32(list(parents)), i32(kids), i32(fresh))
        except BaseException:  # nothing was forked: what was taken goes back
            for c, f in zip(kids, fresh):
                self._rows[c] = [f] if f >= 0 else []
            self.free(kids)
            raise
        for p, c, f in zip(parents, kids, fresh):
            full = self._lens[p] // self.page_size
            self._rows[c] = self._rows[p][:full] + ([f] if f >= 0 else [])
            self._lens[c] = self._lens[p]
            for page in self._rows[p][:full]:
                self._refs[page] += 1
            if len(self._rows[p]) > full + (f >= 0):  # the device's row also names pages that are only reserved
                self._dirty = True
        return kids

    def free(self, seqs: Sequence[int]) -> None:
        """Drop sequences; pages that no other sequence shares return to the pool."""
        self._check(*seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is freed twice")
        for s in seqs:
            for page in self._rows[s]:
                self._refs[page] -= 1
                if self._refs[page] == 0:
                    heapq.heappush(self._free, page)
            self._rows[s], self._lens[s] = None, 0
            heapq.heappush(self._free_seqs, s)
        self._dirty = True

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many there are."""
        used = sum(1 for r in self._refs if r)
        src = [p for p in range(used, len(self._refs)) if self._refs[p]]
        if src:
            dst = [p for p in range(used) if not self._refs[p]]
            self._sync()
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
            ops.move_pages(self.k_pages, self.v_pages, self.page_table, i32(src), i32(dst))
            to = dict(zip(src, dst))
            self._rows = [r if r is None else [to.get(p, p) for p in r] for r in self._rows]
            for a, b in to.items():
                self._refs[b], self._refs[a] = self._refs[a], 0
            self._free = list(range(used, len(self._refs)))
        return used

    def resize(self, num_pages: int) -> None:
        """A pool of another size (after :meth:`compact`, at least the pages in use)."""
        if num_pages < 0:
            raise ValueError(f"num_pages must not be negative, got {num_pages}")
        if any(self._refs[num_pages:]):
            raise ValueError(f"pages past {num_pages} are in use: compact() first")
        keep = min(num_pages, self.num_pages)
        pools = []
        for old in (self.k_pages, self.v_pages):
            new = torch.empty((old.shape[0], num_pages, *old.shape[2:]), dtype=old.dtype, device=old.device)
            new[:, :keep] = old[:, :keep]
            pools.append(new)
        self.k_pages, self.v_pages = pools  # both or, where there is no room for the second, neither
        self._refs = self._refs[:num_pages] + [0] * (num_pages - len(self._refs))
        self._free = [p for p in range(num_pages) if not self._refs[p]]

    # ------------------------------------------------------------------ forward passes
    def _rows_of(self, seqs: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
        self._check(*seqs)
        self._sync()
        at = torch.tensor(list(seqs), dtype=torch.long, device=self.device)
        return self.page_table[at], self.seq_lens[at]

    def prefill_step(self, seqs: Sequence[int], tokens: Sequence[int]) -> RaggedStep:
        """A step in which ``seqs[i]``, empty so far, receives ``tokens[i]`` tokens (pages reserved here)."""
        self._check(*seqs)
        if any(self._lens[s] for s in seqs):
            raise ValueError("prefill of a sequence that already holds tokens")
        self.reserve(seqs, tokens)
        table, start = self._rows_of(seqs)
        cu = torch.tensor([0, *tokens], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(self.device)
        return RaggedStep(self, table, cu, start, None)

    def decode_step(self, seqs: Sequence[int]) -> RaggedStep:
        """A step in which each of ``seqs`` receives one token (reserved before); ``start`` and ``seq_lens`` are
        tensors of the step's own, for a caller that replays it to advance."""
        self._check(*seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        for s in seqs:
            if self._lens[s] >= len(self._rows[s]) * self.page_size:
                raise ValueError(f"sequence {s}: its next position {self._lens[s]} has no page, reserve() it first")
        table, start = self._rows_of(seqs)
        cu = torch.arange(len(seqs) + 1, dtype=torch.int32, device=self.device)
        return RaggedStep(self, table, cu, start, start + 1)

    def workspace(self, batch: int, num_heads: int):
        """Decode-attention scratch for this batch, kept: the steps of one cache run one after the other.  Scratch made
        inside a capture is the capture's own: its counters are cleared by the graph's replays, not now."""
        if self.device.type != "cuda":
            return None
        key = (batch, num_heads)
        if key in self._workspaces:
            return self._workspaces[key]
        made = ops.paged_attention_workspace(batch, num_heads, self.k_pages.shape[3], self.k_pages.shape[4],
                                             self.width * self.page_size, self.device)
        if not torch.cuda.is_current_stream_capturing():
            self._workspaces[key] = made
        return made


@dataclass
class RaggedGeneration:
    """Continuations of prompts of different lengths, ``num_samples`` per prompt, prompt by prompt.

    Sequence i answers prompt ``i // num_samples``; its tokens are ``new_tokens[i, :lengths[i]]`` (an EOS is the
    last).  ``sampler_log_probs`` are those of the filtered distribution that the token was drawn from,
    ``log_probs``, ``entropy`` and the alternatives those of the model's own.  Entries past a length are zero
    (ids -1)."""

    prompts: list[torch.Tensor]
    num_samples: int
    new_tokens: torch.Tensor
    lengths: torch.Tensor
    sampler_log_probs: torch.Tensor
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_ids: torch.Tensor

    def sequences(self) -> list[torch.Tensor]:
        n = self.lengths.tolist()
        return [torch.cat([self.prompts[i // self.num_samples], self.new_tokens[i, :n[i]]]) for i in range(len(n))]


class _Draw:
    """Draws a token per sequence and records it with its statistics; everything stays on the device, so the
    draw can be part of a captured step."""

    def __init__(self, n: int, steps: int, device, temperature, top_k, top_p, eos, alternatives, generator):
        self.args = (temperature, top_k, top_p)
        self.eos, self.alternatives, self.generator = eos, alternatives, generator
        f = dict(dtype=torch.float32, device=device)
        self.tokens = torch.zeros(n, steps, dtype=torch.long, device=device)
        self.sampler_lp, self.lp, self.ent = (torch.zeros(n, steps, **f) for _ in range(3))
        self.top_lp = torch.zeros(n, steps, alternatives, **f)
        self.top_ids = torch.full((n, steps, alternatives), -1, dtype=torch.long, device=device)
        self.live = torch.ones(n, dtype=torch.int32, device=device)
        self.token_in = torch.zeros(n, dtype=torch.long, device=device)
        self.cuda = torch.device(device).type == "cuda"
        if self.cuda:
            seed = int(torch.randint(0, 2 ** 62, (1,), generator=generator).item())
            self.rng = torch.tensor([seed, 0], dtype=torch.long, device=device)  # seed, step
            self._next = torch.empty(n, dtype=torch.long, device=device)
            self._next_lp = torch.empty(n, **f)
        else:
            self.rng = torch.zeros(2, dtype=torch.long)

    def __call__(self, logits: torch.Tensor) -> None:
        from .sampler import _cuda_sample, sample_next_token_with_log_prob

        if self.cuda:
            _cuda_sample(logits, *self.args, True, rng=self.rng, out=(self._next, self._next_lp))
            nxt, lp = self._next, self._next_lp
        else:
            nxt, lp = sample_next_token_with_log_prob(logits, *self.args, generator=self.generator)
        at = self.rng[1:]
        # sequences that have ended are not scored
        target = torch.where(self.live > 0, nxt, torch.full_like(nxt, ops.IGNORE_INDEX))
        st = ops.token_stats(logits, target, top_k=self.alternatives)
        self.lp.index_copy_(1, at, st.log_probs[:, None])
        self.ent.index_copy_(1, at, st.entropy[:, None])
        if self.alternatives:
            self.top_lp.index_copy_(1, at, st.top_log_probs[:, None])
            self.top_ids.index_copy_(1, at, st.top_ids[:, None])
        self.sampler_lp.index_copy_(1, at, (lp * self.live)[:, None])
        self.tokens.index_copy_(1, at, (nxt * self.live)[:, None])
        self.token_in.copy_(nxt)
        if self.eos is not None:
            self.live.mul_((nxt != self.eos).to(torch.int32))
        at.add_(1)


def check_ragged_model(config, device) -> None:
    """Ragged generation runs on one rank; on CUDA with the head sizes that the attention kernels have."""
    if parallel_state.get_sep_world_size() > 1:
        raise ValueError("ragged generation does not run sequence/expert parallel (SEP size must be 1)")
    d = config.hidden_size // config.num_attention_heads
    if torch.device(device).type == "cuda" and d not in (64, 128):
        raise ValueError(f"ragged generation needs head_dim 64 or 128 on CUDA, got {d}")


@torch.no_grad()
def generate_ragged(engine, prompts: Sequence[torch.Tensor], max_new_tokens: int, num_samples: int = 1,
                    temperature: float = 1.0, top_k: int | None = None, top_p: float | None = None,
                    eos_token_id: int | None = None, alternatives: int = 0,
                    cache: RaggedKVCache | None = None) -> RaggedGeneration:
    """``InferenceEngine.generate_ragged``; see there."""
    cfg, dev, model = engine.model_config, engine.device, engine.model
    check_ragged_model(cfg, dev)
    lens = [int(p.numel()) for p in prompts]
    if not prompts or min(lens) < 1 or any(p.dim() != 1 for p in prompts):
        raise ValueError("prompts must be a non-empty list of non-empty 1-D token tensors")
    if max_new_tokens < 1 or num_samples < 1:
        raise ValueError(f"max_new_tokens ({max_new_tokens}) and num_samples ({num_samples}) must be positive")
    if max(lens) + max_new_tokens > cfg.block_size:
        raise ValueError(f"Requested total sequence length {max(lens) + max_new_tokens} exceeds block_size {cfg.block_size}")
    if temperature <= 0:
        raise ValueError("temperature must be > 0")
    prompts = [p.to(dev, torch.long) for p in prompts]
    n = len(prompts) * num_samples
    # positions that are written: the prompt and all new tokens but the last
    total = [x + max_new_tokens - 1 for x in lens]
    own = cache is None
    if own:
        page = engine.kv_cache_page_size
        pages = sum(x // page for x in lens) + sum(num_samples * (-(-t // page) - x // page) for x, t in zip(lens, total))
        cache = RaggedKVCache.from_model_config(cfg, pages, page, n, dev, engine.dtype if dev.type == "cuda" else torch.float32,
                                                max_seq_len=max(max(lens), max(total)))
    first = cache.add(len(prompts))
    seqs = list(first)
    try:
        step = cache.prefill_step(first, lens)
        logits = model.forward_ragged(torch.cat(prompts), step, step.cu_seqlens[1:].long() - 1)
        cache.advance(first, lens)
        kids = cache.fork([s for s in first for _ in range(num_samples - 1)])
        seqs = []
        for i, s in enumerate(first):
            seqs += [s, *kids[i * (num_samples - 1):(i + 1) * (num_samples - 1)]]
        logits = logits.repeat_interleave(num_samples, 0)
        draw = _Draw(n, max_new_tokens, dev, temperature, top_k, top_p, eos_token_id, alternatives, None)
        draw(logits)
        if max_new_tokens > 1:
            cache.reserve(seqs, [max_new_tokens - 1] * n)
            step = cache.decode_step(seqs)

            def advance():
                # a sequence that has ended keeps its position and attends to nothing
                step.seq_lens.copy_((step.start + 1) * draw.live)
                out = model.forward_ragged(draw.token_in, step)
                step.start.add_(draw.live)
                return out

            every = engine.eos_check_interval
            graph = None
            if engine.use_cuda_graph and max_new_tokens > 3:
                keep = step.start.clone()
                advance()  # outside the graph: allocations, lazy tables
                step.start.copy_(keep)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    draw(advance())
            for i in range(1, max_new_tokens):
                if eos_token_id is not None and (i - 1) % every == 0 and not bool(draw.live.any()):
                    break
                if graph is not None:
                    graph.replay()
                else:
                    draw(advance())
        if dev.type == "cuda":
            torch.cuda.synchronize()  # before the graph's memory goes
    finally:
        cache.free([s for s in seqs if cache._rows[s] is not None])
    if dev.type == "cuda":
        ops.check_status(dev)  # a skipped entry or a failed wait: the tokens are not to be used
    steps = int(draw.rng[1].item())
    lengths = torch.full((n,), steps, dtype=torch.long, device=dev)
    if eos_token_id is not None:
        hit = draw.tokens[:, :steps] == eos_token_id
        # tokens after an end are stored as 0, which may be the EOS id itself: the first hit counts
        lengths = torch.where(hit.any(1), hit.to(torch.int8).argmax(1) + 1, lengths)
    return RaggedGeneration(prompts, num_samples, draw.tokens[:, :steps], lengths, draw.sampler_lp[:, :steps],
                            draw.lp[:, :steps], draw.ent[:, :steps], draw.top_lp[:, :steps], draw.top_ids[:, :steps])
