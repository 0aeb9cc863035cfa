"""Plain definitions in 64 bits of the operators in ``tinytron_b200.ops.ragged``, for their tests.

The error bounds are elementwise and come from what the kernels round: probabilities and dS to bf16
(2^-9 each), outputs to bf16 (2^-9), exponentials to about 2^-12; sums are fp32."""
import math

import torch


def attention_one(q, k, v, do=None, scale=None):
    """One sequence: q [n, Hq, D], k/v [m, Hkv, D] -> dict of fp64 results and elementwise error bounds."""
    n, hq, d = q.shape
    m, hkv, _ = k.shape
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, k, v = q.double().transpose(0, 1), k.double().transpose(0, 1), v.double().transpose(0, 1)
    ke, ve = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
    seen = torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n)
    z = (q @ ke.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    some = seen.any(-1)[None, :, None]
    p = torch.where(some, z, torch.zeros_like(z)).softmax(-1) * some if m else z
    o = p @ ve
    mag = p @ ve.abs()
    out = {"o": o, "o_tol": 2.0 ** -7 * mag + 1e-30}
    if do is not None:
        do = do.double().transpose(0, 1)
        dp = do @ ve.transpose(1, 2)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # P and its exponential, dS's own rounding, and delta taken from the rounded o
        e = 2.0 ** -8 * ds.abs() + p * (2.0 ** -7 * (do.abs() * mag).sum(-1, keepdim=True)) + 2.0 ** -11 * p * (dp - delta).abs()
        fold = lambda x: x.reshape(hkv, g, m, d).sum(1)  # noqa: E731
        dq, dk, dv = scale * ds @ ke, scale * ds.transpose(1, 2) @ q, p.transpose(1, 2) @ do
        out.update(dq=dq, dk=fold(dk), dv=fold(dv))
        out["dq_tol"] = scale * e @ ke.abs() + 2.0 ** -8 * dq.abs() + 1e-30
        out["dk_tol"] = fold(scale * e.transpose(1, 2) @ q.abs()) + 2.0 ** -8 * out["dk"].abs() + 1e-30
        out["dv_tol"] = fold(2.0 ** -7 * p.transpose(1, 2) @ do.abs()) + 2.0 ** -8 * out["dv"].abs() + 1e-30
    return {x: y.transpose(0, 1) for x, y in out.items()}


def packed(q, k, v, cu_q, cu_k=None, do=None, scale=None):
    """All sequences of a packing, rows after the last one zero."""
    cu_k = cu_q if cu_k is None else cu_k
    parts = []
    for b in range(len(cu_q) - 1):
        i, j = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        parts.append(attention_one(q[i], k[j], v[j], None if do is None else do[i], scale))
    res = {}
    for x, like in (("o", q), ("dq", q), ("dk", k), ("dv", v)):
        if x != "o" and do is None:
            continue
        for s in ("", "_tol"):
            full = torch.zeros(like.shape, dtype=torch.float64, device=like.device)
            at = 0
            for part in parts:
                full[at:at + len(part[x + s])] = part[x + s]
                at += len(part[x + s])
            res[x + s] = full
    return res


def token_stats(x, t, top, ignore=-100):
    """fp64 (log-prob, entropy, top log-probs, ids, log softmax) of scored rows, zeros / -1 elsewhere."""
    x = x.double()
    scored = t != ignore
    y = torch.log_softmax(x, -1)
    lp = y.gather(1, t.clamp_min(0)[:, None])[:, 0]
    p = y.exp()
    ent = -torch.where(p > 0, p * y, torch.zeros_like(y)).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    tops = y.gather(1, ids)
    z = torch.zeros((), dtype=torch.float64, device=x.device)
    return (torch.where(scored, lp, z), torch.where(scored, ent, z), torch.where(scored[:, None], tops, z),
            torch.where(scored[:, None], ids, torch.full_like(ids, -1)), y)


def token_stats_grad(x, t, g_lp, g_ent, g_top, ids, ignore=-100):
    """fp64 gradient and the magnitude its rounding errors scale with."""
    y = torch.log_softmax(x.double(), -1)
    p = y.exp()
    h = -torch.where(p > 0, p * y, torch.zeros_like(y)).sum(-1, keepdim=True)
    yy = torch.where(p > 0, y, torch.zeros_like(y))
    scored = (t != ignore).double()[:, None]
    a, b = g_lp.double()[:, None], g_ent.double()[:, None]
    grad = -p * (a + b * (yy + h))
    mag = p * (a.abs() + b.abs() * (yy.abs() + h))
    grad.scatter_add_(1, t.clamp_min(0)[:, None], a)
    mag.scatter_add_(1, t.clamp_min(0)[:, None], a.abs())
    if g_top is not None:
        c = g_top.double()
        grad -= p * c.sum(-1, keepdim=True)
        mag += p * c.abs().sum(-1, keepdim=True)
        grad.scatter_add_(1, ids.clamp_min(0), c)
        mag.scatter_add_(1, ids.clamp_min(0), c.abs())
    return grad * scored, mag * scored
