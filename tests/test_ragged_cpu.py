"""Ragged operators on CPU against their 64-bit definitions, the cache's bookkeeping, and the path that runs
them together: ragged generation, packed scoring, a packed policy update."""
import math
import random

import pytest
import torch

import ragged_oracle as oracle
from tinytron_b200 import ops
from tinytron_b200.inference import InferenceEngine, RaggedKVCache
from tinytron_b200.models import GPT, ModelConfig
from tinytron_b200.rl import group_advantages, make_ragged_rollout, ragged_grpo_loss


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def cu_of(lens):
    return i32([0, *torch.tensor(lens).cumsum(0).tolist()])


def cfg(**kw):
    base = dict(block_size=128, vocab_size=120, num_layer=2, num_attention_heads=4, num_key_value_heads=2, hidden_size=64,
                intermediate_size=96, init_std=0.05, seed=3)
    base.update(kw)
    return ModelConfig(**base)


# ----------------------------------------------------------------------------- operators
@pytest.mark.parametrize("lens,lens_k", [([5, 1, 12], None), ([0, 7, 0], None), ([4, 9], [11, 3])], ids=str)
def test_packed_attention(lens, lens_k):
    g = torch.Generator().manual_seed(0)
    n, m = sum(lens) + 2, sum(lens_k or lens) + 2
    q, k, v = (torch.randn(a, h, 16, generator=g) for a, h in ((n, 4), (m, 2), (m, 2)))
    do = torch.randn(n, 4, 16, generator=g)
    leaf = [x.clone().requires_grad_(True) for x in (q, k, v)]
    o = ops.packed_attention(*leaf, cu_of(lens), None if lens_k is None else cu_of(lens_k))
    grads = torch.autograd.grad(o, leaf, do)
    ref = oracle.packed(q, k, v, cu_of(lens).tolist(), None if lens_k is None else cu_of(lens_k).tolist(), do=do)
    for x, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv")):
        assert torch.allclose(x.double(), ref[name], atol=1e-5), name


def test_rotary_append_paged_attention_and_rope_positions():
    from tinytron_b200.ops.rope import rope_reference, rope_tables

    g = torch.Generator().manual_seed(1)
    hq, hkv, d, page, lens, past = 4, 2, 8, 4, [3, 1, 6], [0, 5, 2]
    qkv = torch.randn(sum(lens) + 1, (hq + 2 * hkv) * d, generator=g)
    cos, sin = rope_tables(d, 10000.0, 64, "cpu")
    kp, vp = torch.zeros(12, page, hkv, d), torch.zeros(12, page, hkv, d)
    table = i32([[7, 2, -1], [1, 4, -1], [3, 9, 11]])
    q, k = ops.rotary_append(qkv, cos, sin, hq, hkv, cu_of(lens), i32(past), kp, vp, table)
    at = 0
    for b, n in enumerate(lens):
        x = qkv[at:at + n].view(1, n, -1, d).transpose(1, 2)
        pos = torch.arange(past[b], past[b] + n)
        qr, kr = rope_reference(x[:, :hq], x[:, hq:hq + hkv], pos)
        assert torch.allclose(q[at:at + n], qr[0].transpose(0, 1), atol=1e-6)
        assert torch.allclose(k[at:at + n], kr[0].transpose(0, 1), atol=1e-6)
        for i, p in enumerate(pos.tolist()):
            assert torch.equal(kp[table[b, p // page], p % page], k[at + i])
            assert torch.equal(vp[table[b, p // page], p % page], qkv[at + i].view(-1, d)[hq + hkv:])
        at += n
    assert bool((q[at:] == 0).all()) and bool((k[at:] == 0).all())
    n = i32([3, 0, 8])
    out = ops.paged_attention(q[:3], kp, vp, table, n)
    for b, m in enumerate(n.tolist()):
        if m == 0:
            assert bool((out[b] == 0).all())
            continue
        keys, vals = (x[table[b, :(m + page - 1) // page].long()].reshape(-1, hkv, d)[:m] for x in (kp, vp))
        assert torch.allclose(out[b].double(), oracle.attention_one(q[b:b + 1], keys, vals)["o"][0], atol=1e-6)
    for bad in (lambda: ops.rotary_append(qkv, cos, sin, hq, hkv, cu_of(lens), i32([0, cos.shape[0], 0])),
                lambda: ops.rotary_append(qkv, cos, sin, hq, hkv, cu_of(lens), i32([0, 8, 0]), kp, vp, table),
                lambda: ops.paged_attention(q[:3], kp, vp, table, i32([3, 0, 13])),
                lambda: ops.paged_attention(q[:3], kp, vp, table.long(), n)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("v,top", [(1, 1), (17, 5), (400, 32)])
def test_token_stats(v, top):
    g = torch.Generator().manual_seed(v)
    x = torch.randn(6, v, generator=g).mul(3)
    x[2] = 0.5
    if v > 2:
        x[3, ::2] = -math.inf
    t = torch.randint(0, v, (6,), generator=g)
    t[3] = min(1, v - 1)
    t[1] = -100
    leaf = x.clone().requires_grad_(True)
    st = ops.token_stats(leaf, t, top_k=top)
    lp, ent, tops, ids, _ = oracle.token_stats(x, t, top)
    assert torch.allclose(st.log_probs.double(), lp, atol=1e-5) and torch.allclose(st.entropy.double(), ent, atol=1e-5)
    assert torch.equal(st.top_ids, ids)
    assert torch.allclose(st.top_log_probs.double(), tops, atol=1e-5)
    ga, gb, gc = torch.randn(6, generator=g), torch.randn(6, generator=g), torch.randn(6, top, generator=g)
    (grad,) = torch.autograd.grad([st.log_probs, st.entropy, st.top_log_probs], leaf, [ga, gb, gc])
    want, _ = oracle.token_stats_grad(x, t, ga, gb, gc, ids)
    assert torch.allclose(grad.double(), want, atol=1e-5)
    for bad in ((x, t[:2]), (x, t.int()), (x.half(), t)):
        with pytest.raises(ValueError):
            ops.token_stats(*bad)
    with pytest.raises(ValueError):
        ops.token_stats(x, t, top_k=min(v, 32) + 1)


# ----------------------------------------------------------------------------- the cache
def test_cache_fork_free_compact_keep_every_sequence():
    """Random sequence of operations against a plain list of each sequence's tokens."""
    rnd = random.Random(0)
    page, layers = 4, 2
    cache = RaggedKVCache(layers, 1, 2, 40, page, 12, 40, "cpu", torch.float32)
    model: dict[int, list[float]] = {}
    stamp = 0.0
    for _ in range(400):
        op = rnd.choice(["add", "append", "append", "fork", "free", "compact", "resize"])
        live = sorted(model)
        if op == "add" and len(model) < 12:
            (s,) = cache.add()
            model[s] = []
        elif op == "append" and live:
            s, n = rnd.choice(live), rnd.randrange(1, 6)
            need = -(-(len(model[s]) + n) // page) - len(cache.pages_of(s))
            if len(model[s]) + n > 40 or need > cache.free_pages:
                with pytest.raises((ValueError, RuntimeError)):
                    cache.reserve([s], [n])
                continue
            cache.reserve([s], [n])
            for i in range(n):
                stamp += 1.0
                p = cache.pages_of(s)[len(model[s]) // page]
                for x in (cache.k_pages, cache.v_pages):
                    x[:, p, len(model[s]) % page] = stamp
                model[s].append(stamp)
            cache.advance([s], [n])
        elif op == "fork" and live and len(model) < 11:
            par = [rnd.choice(live) for _ in range(rnd.randrange(1, 3))]
            if sum(1 for p in par if len(model[p]) % page) > cache.free_pages:
                with pytest.raises(RuntimeError):
                    cache.fork(par)
                continue
            for p, c in zip(par, cache.fork(par)):
                model[c] = list(model[p])
        elif op == "free" and live:
            s = rnd.choice(live)
            cache.free([s])
            del model[s]
        elif op == "compact":
            used = cache.compact()
            assert used == cache.num_pages - cache.free_pages
            assert all(p < used for s in model for p in cache.pages_of(s))
        elif op == "resize":
            used = cache.compact()
            cache.resize(max(used, rnd.choice([30, 40, 50])))
        cache._sync()
        for s, toks in model.items():
            assert cache.length(s) == len(toks) == int(cache.seq_lens[s])
            for i, x in enumerate(toks):
                p = int(cache.page_table[s, i // page])
                assert p == cache.pages_of(s)[i // page]
                assert bool((cache.k_pages[:, p, i % page] == x).all()) and bool((cache.v_pages[:, p, i % page] == x).all())
    for s in list(model):
        cache.free([s])
    assert cache.free_pages == cache.num_pages


def test_cache_refusals():
    cache = RaggedKVCache(1, 1, 2, 3, 4, 2, 16, "cpu", torch.float32)
    a, b = cache.add(2)
    with pytest.raises(RuntimeError):
        cache.add()
    with pytest.raises(ValueError):
        cache.reserve([a], [17])
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.reserve([a, b], [8, 8])
    assert cache.free_pages == 3 and cache.pages_of(a) == []
    with pytest.raises(ValueError):
        cache.advance([a], [1])
    with pytest.raises(ValueError):
        cache.reserve([a, a], [1, 1])
    with pytest.raises(ValueError):
        cache.free([a, a])
    cache.free([a])
    for f in (cache.length, lambda s: cache.free([s]), lambda s: cache.fork([s])):
        with pytest.raises(ValueError):
            f(a)
    cache.reserve([b], [9])
    with pytest.raises(ValueError):
        cache.resize(2)
    with pytest.raises(ValueError):
        RaggedKVCache(1, 1, 2, 3, 0, 2, 16, "cpu", torch.float32)


# ----------------------------------------------------------------------------- the path
@pytest.mark.parametrize("moe", [False, True])
def test_ragged_generation_is_greedy_decoding_of_each_prompt(moe):
    c = cfg(use_moe=moe, num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32)
    eng = InferenceEngine(c, device="cpu", dtype=torch.float32, kv_cache_page_size=4)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, c.vocab_size, (n,), generator=g) for n in (3, 8, 1, 17)]
    out = eng.generate_ragged(prompts, 6, num_samples=2, top_k=1, alternatives=3)
    assert out.new_tokens.shape == (8, 6) and out.lengths.tolist() == [6] * 8
    for i, p in enumerate(prompts):
        seq = p.clone()
        for j in range(6):
            with torch.no_grad():
                logits = eng.model(seq[None])[0, -1]
            y = logits.float().log_softmax(-1)
            t = int(logits.argmax())
            for s in (2 * i, 2 * i + 1):
                assert int(out.new_tokens[s, j]) == t
                assert abs(float(out.log_probs[s, j] - y[t])) < 1e-4
                assert abs(float(out.entropy[s, j] + (y.exp() * y).sum())) < 1e-4
                assert out.top_ids[s, j, 0] == t and torch.allclose(out.top_log_probs[s, j], y.topk(3).values, atol=1e-4)
            seq = torch.cat([seq, torch.tensor([t])])
        assert torch.equal(out.sequences()[2 * i], seq)


def test_ragged_generation_stops_at_eos_and_reuses_a_cache():
    c = cfg()
    eng = InferenceEngine(c, device="cpu", dtype=torch.float32, kv_cache_page_size=4, eos_check_interval=2)
    prompts = [torch.tensor([5, 9]), torch.tensor([7])]
    free = eng.generate_ragged(prompts, 12, top_k=1)
    eos = int(free.new_tokens[0, 3])
    stop = [row.index(eos) + 1 if eos in row else 12 for row in free.new_tokens.tolist()]
    cache = RaggedKVCache.from_model_config(c, 20, 4, 2, "cpu", torch.float32)
    for _ in range(2):
        out = eng.generate_ragged(prompts, 12, top_k=1, eos_token_id=eos, cache=cache)
        assert out.lengths.tolist() == [min(x, 12) for x in stop]
        for i, n in enumerate(out.lengths.tolist()):
            assert torch.equal(out.new_tokens[i, :n], free.new_tokens[i, :n])
            assert bool((out.log_probs[i, n:] == 0).all())
        assert cache.free_pages == 20
    small = RaggedKVCache.from_model_config(c, 2, 4, 2, "cpu", torch.float32)
    with pytest.raises(RuntimeError, match="exhausted"):
        eng.generate_ragged(prompts, 12, cache=small)
    assert small.free_pages == 2  # what the failed call held is back
    for bad in (dict(prompts=[]), dict(prompts=[torch.tensor([], dtype=torch.long)]), dict(max_new_tokens=0),
                dict(max_new_tokens=1000), dict(num_samples=0), dict(temperature=0.0)):
        with pytest.raises(ValueError):
            eng.generate_ragged(**{"prompts": prompts, "max_new_tokens": 4, **bad})


def test_packed_scores_are_the_padded_scores_and_train():
    c = cfg()
    model = GPT(c, device="cpu")
    g = torch.Generator().manual_seed(4)
    seqs = [torch.randint(0, c.vocab_size, (n,), generator=g) for n in (5, 2, 11)]
    labels = [torch.cat([s[1:], torch.tensor([-100])]) for s in seqs]
    st = model.packed_token_stats(torch.cat(seqs), torch.cat(labels), cu_of([len(s) for s in seqs]), top_k=2)
    want = torch.cat([model.token_log_probs(s[None], t[None])[0] for s, t in zip(seqs, labels)])
    assert torch.allclose(st.log_probs, want, atol=1e-5)
    ga = torch.autograd.grad(st.log_probs.sum(), list(model.parameters()))
    gb = torch.autograd.grad(want.sum(), list(model.parameters()))
    assert all(torch.allclose(a, b, atol=1e-4) for a, b in zip(ga, gb))


def test_ragged_rollout_and_grpo_loss():
    c = cfg()
    eng = InferenceEngine(c, device="cpu", dtype=torch.float32, kv_cache_page_size=4)
    torch.manual_seed(0)
    prompts = [torch.tensor([3, 4, 5]), torch.tensor([6])]
    gen = eng.generate_ragged(prompts, 5, num_samples=3, eos_token_id=11)
    ro = make_ragged_rollout(gen)
    lens = [len(s) for s in gen.sequences()]
    assert ro.cu_seqlens.tolist() == cu_of(lens).tolist() and ro.max_seqlen == max(lens)
    at = 0
    for i, s in enumerate(gen.sequences()):
        p, n = len(prompts[i // 3]), int(gen.lengths[i])
        lab = ro.labels[at:at + len(s)].tolist()
        assert lab == [-100] * (p - 1) + s[p:].tolist() + [-100]
        assert torch.equal(ro.old_log_probs[at + p - 1:at + p - 1 + n], gen.sampler_log_probs[i, :n])
        at += len(s)
    actor = GPT(c, device="cpu")
    actor.load_state_dict(eng.model.state_dict())
    adv = group_advantages(torch.arange(6.0), 3)
    out = ragged_grpo_loss(actor, ro, adv, entropy_coef=0.1)
    # the actor is the sampler: every ratio is one, the surrogate is the mean advantage of the answer tokens
    mean = float((adv * gen.lengths).sum() / gen.lengths.sum())
    assert abs(float(out.metrics["mean_ratio"]) - 1) < 1e-4 and float(out.metrics["clip_frac"]) == 0
    assert abs(float(out.loss.detach()) + mean + 0.1 * float(out.metrics["entropy"])) < 1e-4
    out.loss.backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in actor.parameters())
    with pytest.raises(ValueError):
        ragged_grpo_loss(actor, ro, adv[:2])


def test_launcher_runs_a_step():
    from tinytron_b200.launch.ragged import main

    log = main(["--device", "cpu", "--num_layer", "1", "--hidden_size", "32", "--num_attention_heads", "2",
                "--num_key_value_heads", "1", "--intermediate_size", "48", "--vocab_size", "64", "--block_size", "64",
                "--prompt_len", "2", "20", "--max_new_tokens", "4", "--num_prompts", "3", "--num_samples", "2",
                "--steps", "1", "--kv_cache_page_size", "4"])
    assert len(log) == 1 and log[0]["new_tokens"] == 24 and math.isfinite(log[0]["loss"])
