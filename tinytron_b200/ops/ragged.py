"""Operators for sequences of different lengths: packed attention, a paged cache whose
sequences have lengths of their own, and statistics of given tokens.

As in :mod:`tinytron_b200.ops`, a CUDA input runs the sm_100a kernels and a CPU input plain
torch math of the same definition; there is no fallback between the two.  Shapes, types and
strides are checked on the host (``ValueError`` here, ``RuntimeError`` at the extension);
index tensors live on the device, and an entry out of range is skipped (its output rows are
zeros; where offsets do not ascend, all of them) and recorded in the status word that
``ops.check_status()`` raises on: call it where the host waits for the device anyway, and before
a step is taken on the results.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

IGNORE_INDEX = -100
MAX_TOP_K = 32


def _C():
    from . import _ext

    return _ext.load()


def _int32(name: str, t: torch.Tensor, device, dim: int = 1) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dim}-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _heads(name: str, t: torch.Tensor, dtype, device, tokens: int | None = None, heads: int | None = None,
           dim: int | None = None) -> None:
    if t.dim() != 3 or (tokens is not None and t.shape[0] != tokens) or (heads is not None and t.shape[1] != heads) \
            or (dim is not None and t.shape[2] != dim):
        want = tuple("*" if x is None else x for x in (tokens, heads, dim))
        raise ValueError(f"{name} must be [tokens, heads, head_dim] = {want}, got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")


def _no_gradient(op: str, *inputs: torch.Tensor) -> None:
    """The serving kernels record no gradient: refuse inputs whose gradient would silently stop here."""
    if torch.is_grad_enabled() and any(x.requires_grad for x in inputs):
        raise ValueError(f"{op} has no gradient on CUDA and its inputs require one: call it under torch.no_grad()"
                         + (" (rotary_packed_attention is differentiable)" if op == "rotary_append" else ""))


def _kernel_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where the kernels can read it in place (head rows contiguous, 16-byte aligned strides),
    else a contiguous copy."""
    per = 16 // t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        n <= 1 or (s > 0 and s % per == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    return t if ok else t.contiguous()


# ----------------------------------------------------------------------------- packed attention
def _offsets_cpu(name: str, cu: torch.Tensor, tokens: int) -> list[int]:
    """The offsets as numbers; on CUDA the kernels make the same test."""
    c = cu.tolist()
    if c[0] != 0 or c[-1] > tokens or any(b < a for a, b in zip(c, c[1:])):
        raise ValueError(f"{name} must ascend from 0 to at most {tokens}, got {c}")
    return c


def _packed_attention_cpu(q, k, v, cu_q, cu_k, scale):
    g = q.shape[1] // k.shape[1]
    out = []
    cq, ck = _offsets_cpu("cu_seqlens", cu_q, q.shape[0]), _offsets_cpu("cu_seqlens_k", cu_k, k.shape[0])
    for b in range(len(cq) - 1):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        qs = q[cq[b]:cq[b + 1]].float().transpose(0, 1)
        ks, vs = (x[ck[b]:ck[b + 1]].float().transpose(0, 1).repeat_interleave(g, 0) for x in (k, v))
        seen = torch.arange(m) <= torch.arange(n)[:, None] + (m - n)
        z = (qs @ ks.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        some = seen.any(-1)  # a query that sees no key gets zeros, not 0 / 0
        p = torch.where(some[:, None], z, torch.zeros((), dtype=z.dtype)).softmax(-1) * some[:, None]
        out.append((p @ vs).transpose(0, 1).to(q.dtype))
    if q.shape[0] > cq[-1]:
        out.append(torch.zeros_like(q[cq[-1]:]))
    return torch.cat(out) if out else torch.zeros_like(q)


def _packed_fwd(q, k, v, cu_q, cu_k, scale, for_backward):
    """(o, (o_lo, lse)): for a backward, what the rounding of o left over and the rows' log-sum-exp."""
    C = _C()
    nq, hq, d = q.shape
    o = torch.empty(nq, hq, d, dtype=q.dtype, device=q.device)
    o_lo = torch.empty_like(o) if for_backward else None
    lse = torch.empty(hq, nq, dtype=torch.float32, device=q.device) if for_backward else None
    sched = torch.empty(C.packed_attn_schedule_numel(nq, k.shape[0], cu_q.numel() - 1), dtype=torch.int32, device=q.device)
    C.packed_attn_fwd(q, k, v, cu_q, cu_k, scale, o, lse, o_lo, sched)
    return o, (o_lo, lse)


def _packed_bwd(q, k, v, o, o_lo, lse, do, cu_q, cu_k, scale, dq, dk, dv):
    C = _C()
    nq, hq, _ = q.shape
    b = cu_q.numel() - 1
    stats = torch.empty(C.packed_attn_stats_numel(nq, hq, b), dtype=torch.float32, device=q.device)
    sched = torch.empty(C.packed_attn_schedule_numel(nq, k.shape[0], b), dtype=torch.int32, device=q.device)
    do = do if do.dtype == torch.bfloat16 else do.to(torch.bfloat16)
    do = do.contiguous()
    if do.data_ptr() % 16:
        do = do.clone()
    C.packed_attn_bwd(q, k, v, o, o_lo, do, lse, cu_q, cu_k, scale, dq, dk, dv, stats, sched)


class PackedAttentionFn(torch.autograd.Function):
    """Forward saves q, k, v, o, what the rounding of o left over, and the log-sum-exp; backward is two kernels (dQ; dK and dV) whose
    sums have a fixed order."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale):
        q, k, v = _kernel_rows(q), _kernel_rows(k), _kernel_rows(v)
        o, saved = _packed_fwd(q, k, v, cu_q, cu_k, scale, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, o, *saved, cu_q, cu_k)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, o_lo, lse, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        _packed_bwd(q, k, v, o, o_lo, lse, do.reshape(o.shape), cu_q, cu_k, ctx.scale, dq, dk, dv)
        return dq, dk, dv, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Causal attention over packed sequences of different lengths, grouped heads.

    q [Nq, Hq, D], k/v [Nk, Hkv, D] bf16, D 64 or 128, Hq a multiple of Hkv, any strides with contiguous
    16-byte-aligned head rows (slices of one packed projection are read in place).  ``cu_seqlens``
    int32 [B + 1] on the same device, ascending from 0: sequence b is rows [cu[b], cu[b + 1]) (lengths of zero are
    allowed).  ``cu_seqlens_k`` gives the keys' rows where they differ: the sequences then end together,
    query i sees keys j <= i + (len_k - len_q).  Queries that see no key, and rows after the last
    sequence, get zeros (and zero gradients).  Returns o [Nq, Hq, D]; differentiable in q, k and v."""
    _heads("q", q, q.dtype, q.device)
    _heads("k", k, q.dtype, q.device, dim=q.shape[2])
    _heads("v", v, q.dtype, q.device, tokens=k.shape[0], heads=k.shape[1], dim=q.shape[2])
    if k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"query heads ({q.shape[1]}) must be a multiple of kv heads ({k.shape[1]})")
    cu_q = _int32("cu_seqlens", cu_seqlens, q.device)
    if cu_seqlens_k is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"q has {q.shape[0]} tokens and k {k.shape[0]}: cu_seqlens_k is needed")
    cu_k = cu_q if cu_seqlens_k is None else _int32("cu_seqlens_k", cu_seqlens_k, q.device)
    if cu_q.numel() < 1 or cu_k.numel() != cu_q.numel():
        raise ValueError(f"cu_seqlens ({cu_q.numel()}) and cu_seqlens_k ({cu_k.numel()}) must have B + 1 entries each")
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if not q.is_cuda:
        return _packed_attention_cpu(q, k, v, cu_q, cu_k, scale)
    if q.dtype != torch.bfloat16 or q.shape[2] not in (64, 128):
        raise ValueError(f"packed_attention runs bf16 with head_dim 64 or 128 on CUDA, got {q.dtype} and {q.shape[2]}")
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return _packed_fwd(_kernel_rows(q), _kernel_rows(k), _kernel_rows(v), cu_q, cu_k, scale, False)[0]
    return PackedAttentionFn.apply(q, k, v, cu_q, cu_k, scale)


class RotaryPackedAttentionFn(torch.autograd.Function):
    """RoPE by position in the sequence (in place on q|k of the packed projection) + packed attention;
    backward writes dq|dk|dv into one buffer of the projection's layout and rotates it back in place."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, cu, hq, hkv, d):
        n = qkv.shape[0]
        qkv = qkv.contiguous()
        x = qkv.view(n, hq + 2 * hkv, d)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        _C().rotary_append(qkv, cos, sin, hq, hkv, d, cu, None, False, q, k, None, None, None)
        scale = 1.0 / math.sqrt(d)
        o, saved = _packed_fwd(q, k, v, cu, cu, scale, ctx.needs_input_grad[0])
        ctx.save_for_backward(qkv, o, *saved, cu, cos, sin)
        ctx.cfg = (hq, hkv, d, scale)
        return o.view(n, hq * d)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        qkv, o, o_lo, lse, cu, cos, sin = ctx.saved_tensors
        hq, hkv, d, scale = ctx.cfg
        n = qkv.shape[0]
        dqkv = torch.empty_like(qkv)
        x, dx = qkv.view(n, hq + 2 * hkv, d), dqkv.view(n, hq + 2 * hkv, d)
        _packed_bwd(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], o, o_lo, lse, do.reshape(n, hq, d), cu, cu, scale,
                    dx[:, :hq], dx[:, hq:hq + hkv], dx[:, hq + hkv:])
        _C().rotary_append(dqkv, cos, sin, hq, hkv, d, cu, None, True, dx[:, :hq], dx[:, hq:hq + hkv], None, None, None)
        return dqkv, None, None, None, None, None, None


def rotary_packed_attention(qkv: torch.Tensor, cu_seqlens: torch.Tensor, num_heads: int, num_kv_heads: int,
                            head_dim: int, theta: float = 10000.0, max_seqlen: int | None = None) -> torch.Tensor:
    """The packed form of ``ops.rotary_attention``: qkv [N, (Hq + 2 Hkv) D] -> o [N, Hq D], positions restart at
    every sequence.  ``max_seqlen`` bounds the longest sequence (default: N).  On CUDA the rotation is done in
    place on ``qkv``, as in ``ops.rotary_attention``."""
    from .rope import rope_tables

    n, w = qkv.shape
    if w != (num_heads + 2 * num_kv_heads) * head_dim:
        raise ValueError(f"qkv must have (Hq + 2 Hkv) * head_dim = {(num_heads + 2 * num_kv_heads) * head_dim} columns, got {w}")
    _int32("cu_seqlens", cu_seqlens, qkv.device)
    cos, sin = rope_tables(head_dim, theta, max(1, n if max_seqlen is None else max_seqlen), qkv.device)
    if qkv.is_cuda:
        return RotaryPackedAttentionFn.apply(qkv, cos, sin, cu_seqlens, num_heads, num_kv_heads, head_dim)
    q, k = rotary_append(qkv, cos, sin, num_heads, num_kv_heads, cu_seqlens)
    v = qkv.view(n, num_heads + 2 * num_kv_heads, head_dim)[:, num_heads + num_kv_heads:]
    return packed_attention(q, k, v, cu_seqlens).reshape(n, num_heads * head_dim)


# ----------------------------------------------------------------------------- pages
def _pool(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor, dims=(4, 5)) -> None:
    if k_pages.dim() not in dims or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype \
            or not k_pages.is_contiguous() or not v_pages.is_contiguous() or v_pages.device != k_pages.device:
        raise ValueError(f"{name}: k_pages and v_pages must be contiguous pools [layers, pages, page_size, Hkv, D] of one "
                         f"shape, type and device ({' or '.join(map(str, dims))} dimensions), got {tuple(k_pages.shape)} "
                         f"and {tuple(v_pages.shape)}")


def rotary_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int, num_kv_heads: int,
                  cu_seqlens: torch.Tensor, start: torch.Tensor | None = None, k_pages: torch.Tensor | None = None,
                  v_pages: torch.Tensor | None = None, page_table: torch.Tensor | None = None, want_k: bool = True):
    """Rotates the q and k heads of packed tokens and writes k and v into their sequences' pages.

    qkv [N, (Hq + 2 Hkv) D] bf16; sequence b is rows [cu_seqlens[b], cu_seqlens[b + 1]), its first token at
    position ``start[b]`` (0 without ``start``; one token per sequence is ``cu_seqlens = arange(B + 1)``).
    cos/sin fp32 [max_pos, D / 2] (``rope_tables``).  With pools [pages, page_size, Hkv, D] and ``page_table`` int32
    [B, width], token t goes to page ``page_table[b, t // page_size]``.  Returns (q [N, Hq, D], k [N, Hkv, D] or None);
    rows of no sequence come back as zeros and are written nowhere.  No gradient on CUDA (refused where one is wanted)."""
    d = 2 * cos.shape[1]
    n = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] < (num_heads + 2 * num_kv_heads) * d:
        raise ValueError(f"qkv must be [N, >= (Hq + 2 Hkv) * D = {(num_heads + 2 * num_kv_heads) * d}], got {tuple(qkv.shape)}")
    cu = _int32("cu_seqlens", cu_seqlens, qkv.device)
    if start is not None and _int32("start", start, qkv.device).numel() != cu.numel() - 1:
        raise ValueError(f"start must have {cu.numel() - 1} entries, got {start.numel()}")
    given = [x is not None for x in (k_pages, v_pages, page_table)]
    if any(given) and not all(given):
        raise ValueError("k_pages, v_pages and page_table go together")
    if k_pages is not None:
        _pool("rotary_append", k_pages, v_pages, (4,))
        _int32("page_table", page_table, qkv.device, 2)
    if qkv.is_cuda:
        _no_gradient("rotary_append", qkv)
        q = torch.empty(n, num_heads, d, dtype=qkv.dtype, device=qkv.device)
        k = torch.empty(n, num_kv_heads, d, dtype=qkv.dtype, device=qkv.device) if want_k else None
        _C().rotary_append(qkv, cos, sin, num_heads, num_kv_heads, d, cu, start, False, q, k, k_pages, v_pages, page_table)
        return q, k
    x = qkv[:, :(num_heads + 2 * num_kv_heads) * d].reshape(n, num_heads + 2 * num_kv_heads, d)
    c = cu.long()
    owner = torch.bucketize(torch.arange(n), c[1:], right=True)
    inside = (owner < cu.numel() - 1) & (torch.arange(n) >= c[0])  # tokens of no sequence: before the first, after the last
    b = owner.clamp(max=max(0, cu.numel() - 2))
    if cu.numel() == 1:
        inside = torch.zeros(n, dtype=torch.bool)
        pos = torch.zeros(n, dtype=torch.long)
    else:
        pos = torch.arange(n) - c[b] + (start.long()[b] if start is not None else 0)
        pos = torch.where(inside, pos, torch.zeros_like(pos))
        if n and (int(pos.min()) < 0 or int(pos.max()) >= cos.shape[0]):
            raise ValueError(f"a position is outside the {cos.shape[0]} rows of the rotation tables")
    cs, sn = cos[pos][:, None], sin[pos][:, None]
    lo, hi = x[:, :num_heads + num_kv_heads, :d // 2].float(), x[:, :num_heads + num_kv_heads, d // 2:].float()
    r = torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1).to(x.dtype)
    r = torch.where(inside[:, None, None], r, torch.zeros((), dtype=r.dtype))
    q, k = r[:, :num_heads], r[:, num_heads:]
    if k_pages is not None and n:
        page = k_pages.shape[1]
        tok = inside.nonzero()[:, 0]
        p = pos[tok]
        if len(tok) and int(p.max()) // page >= page_table.shape[1]:
            raise ValueError(f"a position is past the {page_table.shape[1]} pages of its sequence")
        where = page_table.long()[b[tok], p // page]
        if len(tok) and (int(where.min()) < 0 or int(where.max()) >= k_pages.shape[0]):
            raise ValueError("a token's page is not mapped")
        k_pages[where, p % page] = k[tok].detach().to(k_pages.dtype)
        v_pages[where, p % page] = x[tok, num_heads + num_kv_heads:].detach().to(v_pages.dtype)
    return q, (k if want_k else None)


def fork_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
               parents: torch.Tensor, children: torch.Tensor, fresh: torch.Tensor) -> None:
    """Sequence ``children[i]`` becomes a copy of ``parents[i]``: its row of ``page_table`` [rows, width] and its
    length; full pages are shared, and where ``fresh[i]`` >= 0 the page that the next token falls into is copied, in
    every layer, to page ``fresh[i]``, which takes its place in the child's row (-1: nothing to copy, the parent ends
    with a full page).  Pools [layers, pages, page_size, Hkv, D] or one layer's.  All index tensors are int32 on the
    pools' device; children are no parents, and no page is given twice (one launch copies in no order)."""
    _pool("fork_pages", k_pages, v_pages)
    dev = k_pages.device
    _int32("page_table", page_table, dev, 2)
    for name, t in (("seq_lens", seq_lens), ("parents", parents), ("children", children), ("fresh", fresh)):
        _int32(name, t, dev)
    if seq_lens.numel() != page_table.shape[0] or not parents.numel() == children.numel() == fresh.numel():
        raise ValueError(f"seq_lens needs {page_table.shape[0]} entries (got {seq_lens.numel()}); parents, children and fresh "
                         f"as many as each other (got {parents.numel()}, {children.numel()}, {fresh.numel()})")
    if k_pages.is_cuda:
        _C().fork_pages(k_pages, v_pages, page_table, seq_lens, parents, children, fresh)
        return
    page = k_pages.shape[-3]
    kp, vp = (x if x.dim() == 5 else x.unsqueeze(0) for x in (k_pages, v_pages))
    rows, width = page_table.shape
    for par, kid, new in zip(parents.tolist(), children.tolist(), fresh.tolist()):
        if not (0 <= par < rows and 0 <= kid < rows) or par == kid or new >= kp.shape[1]:
            raise ValueError(f"parent {par}, child {kid} or page {new} is out of range")
        last = int(seq_lens[par]) // page
        old = int(page_table[par, last]) if new >= 0 and 0 <= last < width else -1
        if last < 0 or new >= 0 and (not 0 <= old < kp.shape[1] or old == new):
            raise ValueError(f"sequence {par} has no page to copy to {new}")
    for par, kid, new in zip(parents.tolist(), children.tolist(), fresh.tolist()):
        page_table[kid] = page_table[par]
        seq_lens[kid] = seq_lens[par]
        if new >= 0:
            last = int(seq_lens[par]) // page
            old = int(page_table[par, last])
            kp[:, new] = kp[:, old]
            vp[:, new] = vp[:, old]
            page_table[kid, last] = new


def move_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, src: torch.Tensor,
               dst: torch.Tensor) -> None:
    """Page ``src[i]`` moves to the free page ``dst[i]`` in every layer, and every entry of ``page_table`` that named it
    follows.  ``src`` ascends; no ``dst`` is a ``src`` or given twice.  Pools as in :func:`fork_pages`."""
    _pool("move_pages", k_pages, v_pages)
    dev = k_pages.device
    _int32("page_table", page_table, dev, 2)
    _int32("src", src, dev)
    _int32("dst", dst, dev)
    if src.numel() != dst.numel():
        raise ValueError(f"src ({src.numel()}) and dst ({dst.numel()}) must have as many entries")
    if k_pages.is_cuda:
        _C().move_pages(k_pages, v_pages, page_table, src, dst)
        return
    kp, vp = (x if x.dim() == 5 else x.unsqueeze(0) for x in (k_pages, v_pages))
    s, t = src.long(), dst.long()
    if bool(((s < 0) | (s >= kp.shape[1]) | (t < 0) | (t >= kp.shape[1]) | (s == t)).any()) or bool((s[1:] <= s[:-1]).any()):
        raise ValueError("src must ascend, and src and dst be different pages of the pool")
    kp[:, t] = kp[:, s]
    vp[:, t] = vp[:, s]
    to = torch.arange(kp.shape[1], dtype=torch.int32)
    to[s] = dst
    page_table.copy_(torch.where(page_table >= 0, to[page_table.long().clamp_min(0)], page_table))


# ----------------------------------------------------------------------------- decode
class PagedAttentionWorkspace(NamedTuple):
    """Scratch of :func:`paged_attention`: partials of sequences that span several CTAs, and arrival counters
    (zero between calls).  Calls that share one must run one after the other."""

    partials: torch.Tensor
    counters: torch.Tensor


def paged_attention_workspace(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, max_keys: int,
                              device) -> PagedAttentionWorkspace:
    """Scratch for calls of up to this batch and ``max_keys`` = page_table width * page_size on ``device``."""
    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    part, cnt = _C().paged_attention_workspace(batch, num_heads, num_kv_heads, head_dim, max_keys, index)
    return PagedAttentionWorkspace(torch.empty(part, dtype=torch.float32, device=device),
                                   torch.zeros(cnt, dtype=torch.int32, device=device))


_WORKSPACES: dict = {}  # (device, stream) -> workspace: calls on one stream run one after the other


def _stream_workspace(q, k_pages, page_table) -> PagedAttentionWorkspace:
    args = (q.shape[0], q.shape[1], k_pages.shape[2], q.shape[2], page_table.shape[1] * k_pages.shape[1])
    if torch.cuda.is_current_stream_capturing():  # a graph replays on any stream: scratch of its own
        return paged_attention_workspace(*args, q.device)
    part, cnt = _C().paged_attention_workspace(*args, q.device.index)
    key = (q.device.index, torch.cuda.current_stream(q.device).cuda_stream)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.partials.numel() < part or ws.counters.numel() < cnt:
        ws = paged_attention_workspace(*args, q.device)
        _WORKSPACES[key] = ws
    return ws


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float | None = None,
                    workspace: PagedAttentionWorkspace | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages, every sequence with its own length.

    q [B, Hq, D] bf16 (D 64 or 128, up to 16 query heads per kv head), pools [pages, page_size, Hkv, D] with any page
    size, ``page_table`` int32 [B, width], ``seq_lens`` int32 [B]: query b attends to its first ``seq_lens[b]`` keys
    (0: output zeros; recorded in the status word: a length past the table, cut there, and a key on a page that is not
    mapped, which counts as zeros).  The lengths are read on the device, so a captured call replays with new ones.
    ``workspace`` (:func:`paged_attention_workspace`) is taken from a per-stream cache if not given.  No gradient on
    CUDA (refused where one is wanted)."""
    _pool("paged_attention", k_pages, v_pages, (4,))
    _heads("q", q, k_pages.dtype, k_pages.device, dim=k_pages.shape[3])
    _int32("page_table", page_table, q.device, 2)
    _int32("seq_lens", seq_lens, q.device)
    b, hq, d = q.shape
    hkv = k_pages.shape[2]
    if page_table.shape[0] != b or seq_lens.numel() != b:
        raise ValueError(f"page_table ({page_table.shape[0]} rows) and seq_lens ({seq_lens.numel()}) must match the batch of {b}")
    if hkv < 1 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be a multiple of kv heads ({hkv})")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if q.is_cuda:
        if q.dtype != torch.bfloat16 or d not in (64, 128) or hq // hkv > 16:
            raise ValueError(f"paged_attention runs bf16, head_dim 64 or 128 and up to 16 query heads per kv head on CUDA, got "
                             f"{q.dtype}, {d} and {hq // hkv}")
        _no_gradient("paged_attention", q, k_pages, v_pages)
        out = torch.empty(b, hq, d, dtype=q.dtype, device=q.device)
        ws = workspace if workspace is not None else _stream_workspace(q, k_pages, page_table)
        _C().paged_attention(_kernel_rows(q), k_pages, v_pages, page_table, seq_lens, scale, ws.partials, ws.counters, out)
        return out
    out = torch.zeros_like(q)
    page = k_pages.shape[1]
    for i, n in enumerate(seq_lens.tolist()):
        if n <= 0:
            continue
        rows = page_table[i, :(n + page - 1) // page].long()
        if len(rows) * page < n or int(rows.min()) < 0 or int(rows.max()) >= k_pages.shape[0]:
            raise ValueError(f"sequence {i}: a page within its {n} keys is not mapped")
        ks, vs = (x[rows].reshape(-1, hkv, d)[:n].float().repeat_interleave(hq // hkv, 1) for x in (k_pages, v_pages))
        p = (torch.einsum("hd,nhd->hn", q[i].float(), ks) * scale).softmax(-1)
        out[i] = torch.einsum("hn,nhd->hd", p, vs).to(q.dtype)
    return out


# ----------------------------------------------------------------------------- token statistics
class TokenStats(NamedTuple):
    """log p of the given tokens, entropy of the rows' distributions, and the k largest log-probs with their ids
    (leading shape of the targets; the last two with a trailing k)."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_ids: torch.Tensor


def _token_stats_fwd(logits, targets, top_k, ignore_index, temperature):
    n = logits.shape[0]
    f = dict(dtype=torch.float32, device=logits.device)
    lp, ent, ms, top = torch.empty(n, **f), torch.empty(n, **f), torch.empty(n, 2, **f), torch.empty(n, top_k, **f)
    ids = torch.empty(n, top_k, dtype=torch.long, device=logits.device)
    _C().token_stats_fwd(logits, targets, top_k, ignore_index, temperature, lp, ent, ms, top, ids)
    return lp, ent, top, ids, ms


class TokenStatsFn(torch.autograd.Function):
    """One pass over the logits forward, one read and one write backward (csrc/fused/token_stats.cu)."""

    @staticmethod
    def forward(ctx, logits, targets, *cfg):
        lp, ent, top, ids, ms = _token_stats_fwd(logits, targets, *cfg)
        ctx.save_for_backward(logits, targets, ent, ms, ids)
        ctx.cfg = cfg  # top_k, ignore_index, temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        logits, targets, ent, ms, ids = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        g = [x.float().contiguous() if x is not None else None for x in (g_lp, g_ent, g_top)]
        _C().token_stats_bwd(logits, targets, *ctx.cfg, ent, ms, ids, *g, grad)
        return grad, None, None, None, None


def _ranking(x):
    """Columns of each row by falling logit, equal ones by their index, NaN last.  Not by log-prob: distinct logits
    may round to one."""
    nan = x.isnan()
    order = torch.sort(x.masked_fill(nan, -math.inf), dim=-1, descending=True, stable=True).indices
    last = torch.sort(nan.gather(1, order).to(torch.uint8), dim=-1, stable=True).indices  # NaN behind -inf too
    return order.gather(1, last)


def _token_stats_cpu(logits, targets, top_k, ignore_index, temperature):
    scored = targets != ignore_index
    t = targets.clamp(min=0)
    if bool((scored & ((targets < 0) | (targets >= logits.shape[-1]))).any()):
        raise ValueError("a target is outside the vocabulary")
    zero = torch.zeros((), dtype=torch.float32)
    # rows that are not scored must not reach the gradient, whatever they hold
    y = torch.log_softmax(torch.where(scored[:, None], logits.float() / temperature, zero), -1)
    lp = torch.where(scored, y.gather(1, t[:, None])[:, 0], zero)
    p = y.exp()
    ent = torch.where(scored, -(p * torch.where(p > 0, y, zero)).sum(-1), zero)  # p log p is 0 where p is
    ids = _ranking(logits.detach())[:, :top_k]
    top = torch.where(scored[:, None], y.gather(1, ids), zero)
    return lp, ent, top, torch.where(scored[:, None], ids, torch.full_like(ids, -1))


def token_stats(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, ignore_index: int = IGNORE_INDEX,
                temperature: float = 1.0) -> TokenStats:
    """Statistics of given tokens under softmax(logits / temperature), in fp32 and differentiable in the logits.

    logits [..., V] bf16 or fp32 (rows contiguous; a row stride of its own is fine), targets [...] int64.  Rows whose
    target is ``ignore_index`` are not scored: log-prob, entropy and alternatives 0, ids -1, no gradient.  The ``top_k``
    (at most 32) alternatives are in falling order, equal logits by their index; a NaN ranks below every number.
    A row without a finite logit has no distribution: NaN, as ``log_softmax`` gives."""
    if logits.dim() < 1 or tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError(f"targets {tuple(targets.shape)} must match the leading dimensions of logits {tuple(logits.shape)}")
    if targets.dtype != torch.long or targets.device != logits.device:
        raise ValueError(f"targets must be int64 on {logits.device}, got {targets.dtype} on {targets.device}")
    v = logits.shape[-1]
    if not 0 <= top_k <= min(MAX_TOP_K, v):
        raise ValueError(f"top_k must be between 0 and min({MAX_TOP_K}, {v}), got {top_k}")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    temperature = float(temperature)
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    lead = tuple(targets.shape)
    x = logits.reshape(-1, v)
    t = targets.reshape(-1).contiguous()
    if logits.is_cuda:
        if v and x.stride(-1) != 1:
            x = x.contiguous()
        if torch.is_grad_enabled() and x.requires_grad:
            lp, ent, top, ids = TokenStatsFn.apply(x, t, top_k, ignore_index, temperature)
        else:
            lp, ent, top, ids, _ = _token_stats_fwd(x, t, top_k, ignore_index, temperature)
    else:
        lp, ent, top, ids = _token_stats_cpu(x, t, top_k, ignore_index, temperature)
    return TokenStats(lp.view(lead), ent.view(lead), top.view(*lead, top_k), ids.view(*lead, top_k))
