"""What the operators of ragged generation and packed training are measured on.

Four operators that run one after the other when prompts of different lengths are answered several times each
and the answers are trained on: attention over packed prompts (with its gradients), attention of one new token
over a paged cache, the pages of that cache (rotate-and-append, forking, compacting), and the log-probabilities
of given tokens with entropy and top alternatives (with their gradient).

``listed()`` and ``draw()`` give cases, ``prepare()`` the inputs of one, ``run()`` one pass: the plain form in
32 bits where ``own`` is false, the framework's call where it is true.  ``work()`` is what a pass cannot do
without, ``exact()`` the same outputs from the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
VOCAB = 50304


# ----------------------------------------------------------------------------- lengths
def lengths(case):
    """The case's sequence lengths: log-uniform weights over a range of ``spread``, scaled to ``tokens``."""
    r = random.Random(case["mix"])
    w = [math.exp(r.uniform(0.0, math.log(case["spread"]))) for _ in range(case["seqs"])]
    scale = case["tokens"] / sum(w)
    return [max(1, int(x * scale)) for x in w]


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # a handful of chat-sized prompts at the moment they arrive: latency
        {"name": "prompts_few", "op": "prompts", "seqs": 4, "tokens": 150, "spread": 12.0, "mix": 1,
         "hq": 16, "hkv": 4, "d": 128},
        # a batch of prompts of very different lengths, packed, as a rollout's prefill sees them
        {"name": "prompts_mixed", "op": "prompts", "seqs": 24, "tokens": 16384, "spread": 64.0, "mix": 2,
         "hq": 16, "hkv": 4, "d": 128},
        # one micro-batch of packed sequences of the 1.3B configuration: forward and backward
        {"name": "train_packed", "op": "train", "seqs": 14, "tokens": 16384, "spread": 16.0, "mix": 3,
         "hq": 16, "hkv": 4, "d": 128},
        # long documents with short ones between them, 64-wide heads: forward and backward
        {"name": "train_long_d64", "op": "train", "seqs": 3, "tokens": 17001, "spread": 200.0, "mix": 4,
         "hq": 8, "hkv": 2, "d": 64},
        # the last few unfinished answers of a batch: latency
        {"name": "decode_few", "op": "decode", "seqs": 3, "tokens": 700, "spread": 20.0, "mix": 5,
         "hq": 16, "hkv": 4, "d": 128, "page": 16},
        # the decode benchmark's batch (32 sequences of about 1K tokens), lengths no longer equal
        {"name": "decode_batch", "op": "decode", "seqs": 32, "tokens": 36000, "spread": 6.0, "mix": 6,
         "hq": 16, "hkv": 4, "d": 128, "page": 128},
        # a few long contexts beside short ones, five query heads for each kv head
        {"name": "decode_long", "op": "decode", "seqs": 9, "tokens": 140000, "spread": 300.0, "mix": 7,
         "hq": 40, "hkv": 8, "d": 128, "page": 64},
        # the new prompts of one layer rotated and written into its pages
        {"name": "append_prompts", "op": "append", "seqs": 24, "tokens": 16384, "spread": 64.0, "mix": 2,
         "hq": 16, "hkv": 4, "d": 128, "page": 128},
        # 8 prompts, 8 answers each: every answer shares the prompt's full pages and copies the last one, all layers
        {"name": "fork_groups", "op": "fork", "seqs": 8, "tokens": 6000, "spread": 8.0, "mix": 8, "copies": 8,
         "layers": 16, "hkv": 4, "d": 128, "page": 128},
        # a third of a pool's pages moved down into the holes that finished answers left, all layers
        {"name": "compact_pool", "op": "compact", "seqs": 48, "tokens": 48000, "spread": 12.0, "mix": 9,
         "layers": 16, "hkv": 4, "d": 128, "page": 16, "holes": 0.33},
        # a decode step's logits: log-probs of the drawn tokens, entropy, 8 alternatives
        {"name": "stats_step", "op": "stats", "rows": 32, "vocab": VOCAB, "top": 8, "wide": False, "train": False,
         "unscored": 0.0},
        # a packed micro-batch's logits, the prompts' rows not scored: forward and backward
        {"name": "stats_train", "op": "stats", "rows": 12288, "vocab": VOCAB, "top": 4, "wide": False, "train": True,
         "unscored": 0.25},
    ]


HEADS = [(16, 4, 128), (16, 8, 128), (16, 2, 128), (40, 8, 128), (8, 2, 64), (8, 8, 64)]
CAP_FLOPS = 7.0e11  # of an attention case
CAP_BYTES = 2.0e9  # of a case bound by memory


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompts", "train", "decode", "append", "fork", "compact", "stats"])
    while True:
        case = _draw_one(op, rng)
        w = work(case)
        if w["flops"] <= CAP_FLOPS and w["bytes"] <= CAP_BYTES:
            return case


def _draw_one(op, rng):
    if op == "stats":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "vocab": rng.choice([VOCAB, 8192, _log_int(rng, 500, 60000)]),
                "top": rng.choice([0, 1, 3, 5, 8, 16]), "wide": rng.random() < 0.25, "train": rng.random() < 0.5,
                "unscored": rng.choice([0.0, 0.3])}
    hq, hkv, d = rng.choice(HEADS)
    seqs = _log_int(rng, 1, 64)
    case = {"op": op, "seqs": seqs, "mix": rng.randrange(1 << 30), "spread": rng.choice([1.5, 8.0, 100.0]),
            "hkv": hkv, "d": d}
    if op in ("prompts", "train"):
        case.update(hq=hq, tokens=max(seqs, _log_int(rng, 16, 20000)))
    elif op == "decode":
        case.update(hq=hq, tokens=max(seqs, _log_int(rng, 16, 150000)), page=rng.choice([16, 64, 128, 100]))
    elif op == "append":
        case.update(hq=hq, tokens=max(seqs, _log_int(rng, 1, 20000)), page=rng.choice([16, 64, 128, 100]))
    elif op == "fork":
        case.update(tokens=max(seqs, _log_int(rng, 16, 20000)), copies=rng.choice([1, 2, 7, 16]),
                    layers=rng.choice([6, 12, 24]), page=rng.choice([16, 64, 128]))
    else:
        case.update(tokens=max(4 * seqs, _log_int(rng, 100, 60000)), layers=rng.choice([6, 12, 24]),
                    page=rng.choice([16, 64, 128]), holes=rng.uniform(0.05, 0.6))
    return case


def _pages_of(n, page):
    return (n + page - 1) // page


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype)


def _tables(lens, page, rng, spare=3):
    """A page table whose pages lie in the pool in no order, -1 past each sequence's end; (table rows, pool size)."""
    need = [_pages_of(n, page) for n in lens]
    pool = sum(need) + spare
    ids = list(range(pool))
    rng.shuffle(ids)
    width = max(need) + 1
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return rows, pool, ids[at:]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def _compaction(case):
    """The pool of a case before compaction: every page id in use, and the moves (ascending sources from above the
    line into the holes below it)."""
    rng = random.Random(case["mix"] + 1)
    need = [_pages_of(n, case["page"]) for n in lengths(case)]
    used = sum(need)
    pool = used + max(1, int(used * case["holes"]))
    ids = rng.sample(range(pool), used)
    taken = set(ids)
    src = sorted(i for i in ids if i >= used)
    dst = [i for i in range(used) if i not in taken]
    return need, pool, ids, src, dst


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    op = case["op"]
    if op == "stats":
        n, v = case["rows"], case["vocab"]
        logits = _randn(g, n, v).mul_(2.5)
        tgt = torch.randint(0, v, (n,), generator=g, device=DEVICE)
        # a language model puts much of its mass on few tokens, the given one among them more often than not
        logits[torch.arange(n, device=DEVICE), tgt] += 8.0 * torch.rand(n, generator=g, device=DEVICE).to(logits.dtype)
        if case["unscored"]:
            tgt[torch.rand(n, generator=g, device=DEVICE) < case["unscored"]] = -100
        s["logits"] = (logits.float() if case["wide"] else logits).requires_grad_(case["train"])
        s["targets"] = tgt
        if case["train"]:
            s["grads"] = [_randn(g, n, dtype=torch.float32), _randn(g, n, dtype=torch.float32).mul_(0.01)]
            if case["top"]:
                s["grads"].append(_randn(g, n, case["top"], dtype=torch.float32).mul_(0.1))
        return s
    lens = lengths(case)
    hkv, d = case["hkv"], case["d"]
    rng = random.Random(case["mix"] * 31 + int(seed))
    if op in ("prompts", "train"):
        hq, n = case["hq"], sum(lens)
        # heads lie side by side in one projection's output, as the model has them
        qkv = _randn(g, n, hq + 2 * hkv, d)
        s["q"], s["k"], s["v"] = (x.requires_grad_(op == "train") for x in
                                  (qkv[:, :hq].detach(), qkv[:, hq:hq + hkv].detach(), qkv[:, hq + hkv:].detach()))
        s["cu"] = _i32(offsets(lens))
        s["lens"] = lens
        if op == "train":
            s["do"] = _randn(g, n, hq, d)
    elif op == "decode":
        rows, pool, _ = _tables(lens, case["page"], rng)
        s["q"] = _randn(g, len(lens), case["hq"], d)
        s["kp"], s["vp"] = (_randn(g, pool, case["page"], hkv, d) for _ in range(2))
        s["table"], s["lens"] = _i32(rows), _i32(lens)
    elif op == "append":
        held = random.Random(case["mix"] + 7)
        past = [held.randrange(0, 3 * case["page"]) for _ in lens]  # answers that are already in the cache
        rows, pool, _ = _tables([a + b for a, b in zip(past, lens)], case["page"], rng)
        s["qkv"] = _randn(g, sum(lens), (case["hq"] + 2 * hkv) * d)
        s["kp"], s["vp"] = (_randn(g, pool, case["page"], hkv, d) for _ in range(2))
        s["table"], s["cu"], s["start"] = _i32(rows), _i32(offsets(lens)), _i32(past)
        s["owner"] = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], device=DEVICE)
        m = max(a + b for a, b in zip(past, lens))
        inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32, device=DEVICE) / d))
        ang = torch.arange(m, dtype=torch.float32, device=DEVICE)[:, None] * inv
        s["cos"], s["sin"] = ang.cos(), ang.sin()
    elif op == "fork":
        kids = len(lens) * case["copies"]
        rows, pool, fresh = _tables(lens, case["page"], rng, spare=kids)
        width = len(rows[0])
        s["kp"], s["vp"] = (_randn(g, case["layers"], pool, case["page"], hkv, d) for _ in range(2))
        s["table"] = _i32(rows + [[-1] * width for _ in range(kids)])
        s["lens"] = _i32(lens + [0] * kids)
        s["parents"] = _i32([b for b in range(len(lens)) for _ in range(case["copies"])])
        s["children"] = _i32(list(range(len(lens), len(lens) + kids)))
        s["fresh"] = _i32([f if lens[i // case["copies"]] % case["page"] else -1 for i, f in enumerate(fresh)])
    else:
        need, pool, ids, src, dst = _compaction(case)
        width = max(need) + 1
        rows, at = [], 0
        for n in need:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        s["kp"], s["vp"] = (_randn(g, case["layers"], pool, case["page"], hkv, d) for _ in range(2))
        s["table"], s["src"], s["dst"] = _i32(rows), _i32(src), _i32(dst)
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from tinytron_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "prompts":
        return ops.packed_attention(s["q"], s["k"], s["v"], s["cu"])
    if op == "train":
        o = ops.packed_attention(s["q"], s["k"], s["v"], s["cu"])
        return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]
    if op == "decode":
        return ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"])
    if op == "append":
        q, k = ops.rotary_append(s["qkv"], s["cos"], s["sin"], case["hq"], case["hkv"], s["cu"], s["start"],
                                 s["kp"], s["vp"], s["table"])
        return [q, k, s["kp"], s["vp"]]
    if op == "fork":
        ops.fork_pages(s["kp"], s["vp"], s["table"], s["lens"], s["parents"], s["children"], s["fresh"])
        return [s["kp"], s["vp"], s["table"], s["lens"]]
    if op == "compact":
        ops.move_pages(s["kp"], s["vp"], s["table"], s["src"], s["dst"])
        return [s["kp"], s["vp"], s["table"]]
    st = ops.token_stats(s["logits"], s["targets"], top_k=case["top"])
    outs = [st.log_probs, st.entropy] + ([st.top_log_probs] if case["top"] else [])
    ids = [st.top_ids] if case["top"] else []
    if not case["train"]:
        return outs + ids
    (grad,) = torch.autograd.grad(outs, s["logits"], s["grads"])
    return [x.detach() for x in outs] + ids + [grad]


@torch.no_grad()
def _run_plain(s):
    op = s["case"]["op"]
    return {"prompts": _plain_prompts, "train": _plain_prompts, "decode": _plain_decode, "append": _plain_append,
            "fork": _plain_fork, "compact": _plain_compact, "stats": _plain_stats}[op](s)


def _plain_prompts(s):
    """softmax(q k^T / sqrt(d), keys up to the query) v of each packed sequence, and the gradients by the formula."""
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    train = case["op"] == "train"
    outs, at = [], 0
    for n in s["lens"]:
        q, k, v = (x[at:at + n].detach().float().transpose(0, 1) for x in (s["q"], s["k"], s["v"]))  # [h, n, d]
        k, v = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
        z = (q @ k.transpose(1, 2)).mul_(scale)
        z.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=z.device).triu_(1), -math.inf)
        z.sub_(z.amax(-1, keepdim=True)).exp_()
        p = z.div_(z.sum(-1, keepdim=True))
        o = p @ v
        part = [o.transpose(0, 1).to(s["q"].dtype)]
        if train:
            do = s["do"][at:at + n].float().transpose(0, 1)
            dv = p.transpose(1, 2) @ do
            ds = (do @ v.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            del p, z
            dq, dk = ds @ k, ds.transpose(1, 2) @ q
            del ds
            dk, dv = (x.reshape(hkv, g, n, d).sum(1) for x in (dk, dv))
            part += [x.transpose(0, 1).to(s["q"].dtype) for x in (dq, dk, dv)]
        outs.append(part)
        at += n
    outs = [torch.cat(x) for x in zip(*outs)]
    return outs if train else outs[0]


def _plain_decode(s):
    """The same for one query a sequence, over the keys that its row of the page table leads to."""
    case = s["case"]
    b, hq, d = s["q"].shape
    hkv, page = case["hkv"], case["page"]
    table = s["table"].long().clamp_min(0)
    width = table.shape[1] * page
    k, v = (x[table].reshape(b, width, hkv, d).float() for x in (s["kp"], s["vp"]))
    q = s["q"].float().reshape(b, hkv, hq // hkv, d)
    z = (q @ k.permute(0, 2, 3, 1)) / math.sqrt(d)  # [b, hkv, g, width]
    seen = torch.arange(width, device=z.device) < s["lens"][:, None]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    p = (z - z.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return (p @ v.permute(0, 2, 1, 3)).reshape(b, hq, d).to(s["q"].dtype)


def _plain_append(s):
    """Half-split rotation by each token's position in its sequence; rotated keys and the values into the pages."""
    case = s["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    n = s["qkv"].shape[0]
    x = s["qkv"].view(n, hq + 2 * hkv, d)
    pos = (torch.arange(n, device=x.device) - s["cu"].long()[s["owner"]]) + s["start"].long()[s["owner"]]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :hq + hkv, :d // 2].float(), x[:, :hq + hkv, d // 2:].float()
    r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
    q, k = r[:, :hq].contiguous(), r[:, hq:].contiguous()
    where = s["table"].long()[s["owner"], pos // page]
    s["kp"][where, pos % page] = k
    s["vp"][where, pos % page] = x[:, hq + hkv:]
    return [q, k, s["kp"], s["vp"]]


def _plain_fork(s):
    """Children take their parent's row and length; a page that is not full is copied into one of their own."""
    page = s["case"]["page"]
    par, kid = s["parents"].long(), s["children"].long()
    s["table"][kid] = s["table"][par]
    s["lens"][kid] = s["lens"][par]
    some = s["fresh"] >= 0
    last = (s["lens"].long()[par] // page)[some]
    src, dst = s["table"].long()[par[some], last], s["fresh"].long()[some]
    s["table"][kid[some], last] = s["fresh"][some]
    for x in (s["kp"], s["vp"]):
        x[:, dst] = x[:, src]
    return [s["kp"], s["vp"], s["table"], s["lens"]]


def _plain_compact(s):
    src, dst = s["src"].long(), s["dst"].long()
    for x in (s["kp"], s["vp"]):
        x[:, dst] = x[:, src]
    to = torch.arange(s["kp"].shape[1], dtype=torch.int32, device=src.device)
    to[src] = s["dst"]
    t = s["table"]
    t.copy_(torch.where(t >= 0, to[t.long().clamp_min(0)], t))
    return [s["kp"], s["vp"], t]


def _plain_stats(s):
    """log softmax at the given tokens, its entropy, the largest values (ties to the lowest index), and d/d logits."""
    case = s["case"]
    x = s["logits"].detach().float()
    n, v = x.shape
    scored = s["targets"] != -100
    t = s["targets"].clamp_min(0)
    m = x.amax(-1, keepdim=True)
    logp = x - m
    logp = logp - logp.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    ent = -(p * logp).sum(-1)
    lp = logp.gather(1, t[:, None])[:, 0]
    outs = [lp * scored, ent * scored]
    ids = []
    if case["top"]:
        bits = x.view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))  # in the order of the values
        key = key * (1 << 20) + ((1 << 20) - 1 - torch.arange(v, device=x.device))
        at = (1 << 20) - 1 - (key.topk(case["top"], -1).values & ((1 << 20) - 1))
        del bits, key
        outs.append(logp.gather(1, at) * scored[:, None])
        ids = [torch.where(scored[:, None], at, torch.full_like(at, -1))]
    if not case["train"]:
        return outs + ids
    ga, gb = s["grads"][0] * scored, s["grads"][1] * scored
    pull = ga[:, None] + gb[:, None] * (logp + ent[:, None])
    if case["top"]:
        pull = pull + (s["grads"][2] * scored[:, None]).sum(-1, keepdim=True)
    grad = -p * pull
    grad.scatter_add_(1, t[:, None], ga[:, None])
    if case["top"]:
        grad.scatter_add_(1, at, s["grads"][2] * scored[:, None])
    return outs + ids + [grad.to(s["logits"].dtype)]


# ----------------------------------------------------------------------------- floors
def work(case):
    op = case["op"]
    if op == "stats":
        n, v, size = case["rows"], case["vocab"], 4 if case["wide"] else 2
        scored = n * (1.0 - case["unscored"])
        table = scored * v * size + (n * v * size if case["train"] else 0)
        return {"bytes": table + n * (8 + 8 + 12 * case["top"]), "flops": scored * v * (12 if case["train"] else 5)}
    lens = lengths(case)
    hkv, d, n = case["hkv"], case["d"], sum(lens)
    if op in ("prompts", "train"):
        pairs = sum(t * (t + 1) // 2 for t in lens)
        io = n * d * 2 * (2 * case["hq"] + 2 * hkv)  # q, k, v, o; the gradients once more as many, q, k, v and do
        return {"bytes": io * (2 if op == "train" else 1),
                "flops": (14.0 if op == "train" else 4.0) * pairs * case["hq"] * d}
    if op == "decode":
        return {"bytes": n * hkv * d * 4 + len(lens) * case["hq"] * d * 4, "flops": 4.0 * n * case["hq"] * d}
    if op == "append":
        return {"bytes": n * d * 2 * ((case["hq"] + 2 * hkv) + (case["hq"] + hkv) + 2 * hkv),
                "flops": 6.0 * n * (case["hq"] + hkv) * d / 2}
    page_bytes = 2 * case["layers"] * case["page"] * hkv * d * 2  # keys and values of every layer
    if op == "fork":
        part = sum(1 for t in lens if t % case["page"]) * case["copies"]
        rows = len(lens) * case["copies"] * (max(_pages_of(t, case["page"]) for t in lens) + 1) * 4
        return {"bytes": 2.0 * part * page_bytes + 2 * rows + 16, "flops": 0}
    need, _, _, src, _ = _compaction(case)
    return {"bytes": 2.0 * len(src) * page_bytes + 8 * len(need) * (max(need) + 1), "flops": 0}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    if op == "stats":
        return _exact_stats(s)
    if op == "append":
        return _exact_append(s)
    if op == "decode":
        return _exact_decode(s)
    return _exact_prompts(s)


def _exact_prompts(s):
    case = s["case"]
    train, g = case["op"] == "train", case["hq"] // case["hkv"]
    ins = [s[x].detach().double() for x in "qkv"]
    outs = [torch.zeros_like(ins[0])] + [torch.zeros_like(x) for x in ins]
    at = 0
    for n in s["lens"]:
        see = torch.tril(torch.ones(n, n, dtype=torch.bool, device=DEVICE))
        for h in range(case["hq"]):  # one head at a time: the longest would not fit otherwise
            leaf = [x[at:at + n, i].clone().requires_grad_(train) for x, i in zip(ins, (h, h // g, h // g))]
            w = torch.where(see, leaf[0] @ leaf[1].T / case["d"] ** 0.5, -math.inf).softmax(-1)
            o = w @ leaf[2]
            outs[0][at:at + n, h] = o.detach()
            if train:
                grads = torch.autograd.grad(o, leaf, s["do"][at:at + n, h].double())
                for out, grad, i in zip(outs[1:], grads, (h, h // g, h // g)):
                    out[at:at + n, i] += grad
            del w, o
        at += n
    return outs if train else outs[0]


def _exact_decode(s):
    case = s["case"]
    page, g = case["page"], case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["lens"].tolist()):
        rows = s["table"][b, :_pages_of(n, page)].long()
        k, v = (x[rows].flatten(0, 1)[:n].double() for x in (s["kp"], s["vp"]))
        for h in range(case["hq"]):
            w = torch.softmax(k[:, h // g] @ s["q"][b, h].double() / case["d"] ** 0.5, 0)
            out[b, h] = w @ v[:, h // g]
    return out


def _exact_append(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, 2, d // 2)[:, :hq + hkv]
    pos = torch.cat([torch.arange(n, device=DEVICE) + p for n, p in zip(lengths(case), s["start"].tolist())])
    z = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    r = torch.complex(x[:, :, 0], x[:, :, 1]) * z
    r = torch.cat([r.real, r.imag], -1)
    return [r[:, :hq].contiguous(), r[:, hq:].contiguous(), None, None]


def _exact_stats(s):
    case = s["case"]
    n, top = case["rows"], case["top"]
    lp, ent = (torch.zeros(n, dtype=torch.float64, device=DEVICE) for _ in range(2))
    tops = torch.zeros(n, top, dtype=torch.float64, device=DEVICE)
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device=DEVICE) if case["train"] else None
    for r0 in range(0, n, 2048):
        rows = (s["targets"][r0:r0 + 2048] != -100).nonzero()[:, 0] + r0
        if not len(rows):
            continue
        x = s["logits"].detach()[rows].double().requires_grad_(case["train"])
        y = torch.log_softmax(x, -1)
        a = y.gather(1, s["targets"][rows][:, None])[:, 0]
        e = -(y.exp() * y).sum(-1)
        outs, grads = [a, e], [gr[rows].double() for gr in s.get("grads", [])]
        if top:  # the values do not depend on which of two equal logits is taken, and the gradient takes the lower index
            order = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top]
            outs.append(y.gather(1, order))
            tops[rows] = outs[2].detach()
        lp[rows], ent[rows] = a.detach(), e.detach()
        if case["train"]:
            (gx,) = torch.autograd.grad(outs, x, grads)
            grad[rows] = gx
    outs = [lp, ent] + ([tops, None] if top else [])
    return outs + ([grad] if case["train"] else [])
