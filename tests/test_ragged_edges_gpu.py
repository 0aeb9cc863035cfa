"""Edges of the ragged operators on the GPU: values that are not finite, rejected entries, temperatures, lost
gradients, accuracy by norms."""
import math

import pytest
import torch

import ragged_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
K_BAD_INDEX = 8


def ops():
    from tinytron_b200 import ops

    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cu_of(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def status_and_clear():
    from tinytron_b200.ops import _ext

    d = torch.cuda.current_device()
    code = int(_ext.load().status_read(d))
    _ext.load().status_clear(d)
    return code


def within(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got.double() - want).abs().max()))


def dirty_memory(mb=64):
    """Freed blocks full of NaN: what torch.empty returns next is not zero by luck."""
    blocks = [torch.full((n,), math.nan, device=DEV) for n in (64, 1024, 65536, 1 << 20, mb << 18) for _ in range(8 if n < 1 << 20 else 1)]
    del blocks


@pytest.fixture(autouse=True)
def _healthy():
    yield
    if torch.cuda.is_available():
        assert status_and_clear() == 0


# ----------------------------------------------------------------------------- packed attention
def packed_inputs(lens, hq, hkv, d, seed):
    g = gen(seed)
    n = sum(lens)
    return randn(g, n, hq, d), randn(g, n, hkv, d), randn(g, n, hkv, d), randn(g, n, hq, d)


def run_packed(q, k, v, do, cu):
    leaf = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = ops().packed_attention(*leaf, i32(cu))
    return [o.detach(), *torch.autograd.grad(o, leaf, do)]


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_keeps_a_keys_nan(poison, d):
    """A key whose scores are NaN or +inf makes the rows that see it NaN, whichever column of its tile it falls into,
    and with them the gradients of every key that those rows see; rows before it and other sequences stay."""
    lens = [40, 200, 30]
    q, k, v, do = packed_inputs(lens, 4, 2, d, seed=1)
    q[40:240, :, 0] = q[40:240, :, 0].abs() + 0.5  # a key of +inf there scores +inf, not NaN by another element's sign
    clean = run_packed(q, k, v, do, cu_of(lens))
    for at in [*range(64, 72), *range(136, 144)]:
        bad = k.clone()
        bad[40 + at, :, 0] = poison
        o, dq, dk, dv = run_packed(q, bad, v, do, cu_of(lens))
        assert torch.equal(o[:40 + at], clean[0][:40 + at]), at
        for x in (o, dq):
            assert bool(x[40 + at:240].isnan().all()), at
        for x in (dk, dv):
            assert bool(x[40:240].isnan().all()), at
        for x, y in zip((o, dq, dk, dv), clean):
            assert torch.equal(x[:40], y[:40]) and torch.equal(x[240:], y[240:]), at


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_key_of_minus_infinity_weighs_nothing(d):
    lens = [40, 200, 30]
    q, k, v, _ = packed_inputs(lens, 4, 2, d, seed=2)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    for at in range(64, 72):
        bad = k.clone()
        bad[40 + at, :, 0] = -math.inf
        o = ops().packed_attention(q, bad, v, i32(cu_of(lens)))
        ref = oracle.packed(q, bad, v, cu_of(lens))
        within(o, ref["o"], ref["o_tol"], at)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_unseen_values_weigh_nothing(d):
    """Values of 3e38 (finite) at keys that a row does not see leave its output and gradient bit for bit."""
    lens = [40, 200, 30]
    q, k, v, do = packed_inputs(lens, 4, 2, d, seed=3)
    clean = run_packed(q, k, v, do, cu_of(lens))
    for at in (64, 139):
        bad = v.clone()
        bad[40 + at:240] = 3e38
        got = run_packed(q, k, bad, do, cu_of(lens))
        for x, y in zip(got[:2], clean[:2]):
            assert torch.equal(x[:40 + at], y[:40 + at]) and torch.equal(x[240:], y[240:])


# ----------------------------------------------------------------------------- token statistics
def check_tempered(x, t, top, temp):
    z = x.double() / temp
    leaf = x.detach().requires_grad_(True)
    st = ops().token_stats(leaf, t, top_k=top, temperature=temp)
    lp, ent, tops, _, y = oracle.token_stats(z, t, top)
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(st.top_ids, torch.where((t != -100)[:, None], ids, torch.full_like(ids, -1)))
    # a scaled difference d is off by a few roundings of itself (1 / T, log2 e / T, the product): 2^-21 |d|
    d = (z - z.amax(-1, keepdim=True)).abs()
    near = d.gather(1, t.clamp_min(0)[:, None])[:, 0]
    scored = (t != -100).double()
    within(st.log_probs, lp, scored * (1e-5 + 2.0 ** -21 * near + 2.0 ** -21 * lp.abs()), "log-probs")
    within(st.entropy, ent, 4e-5 * (1 + ent), "entropy")
    within(st.top_log_probs, tops, 1e-5 + 2.0 ** -20 * tops.abs(), "top")
    g = gen(9)
    n = x.shape[0]
    ga, gb, gc = randn(g, n, dtype=torch.float32), randn(g, n, dtype=torch.float32), randn(g, n, top, dtype=torch.float32)
    (grad,) = torch.autograd.grad([st.log_probs, st.entropy, st.top_log_probs], leaf, [ga, gb, gc])
    want, mag = oracle.token_stats_grad(z, t, ga, gb, gc, ids)
    far = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y))  # a probability is off by its exponent's error
    tol = (3e-5 + 2.0 ** -20 * far) * mag / temp + (2.0 ** -8 * want.abs() / temp if x.dtype == torch.bfloat16 else 0)
    within(grad, want / temp, tol + 1e-30, "gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temp", [0.7, 1.3, 0.05, 30.0, 1e-4, 1e4])
def test_token_stats_temperature(dtype, temp):
    g = gen(11)
    x = randn(g, 8, 3001, dtype=torch.float32).mul(3)
    x[1, ::3] = -math.inf
    x[2, 9:] = torch.finfo(dtype).min
    x[3] += 500.0
    x[4] = 1.25
    x = x.to(dtype)
    t = torch.tensor([5, 1, 3, 2999, 17, -100, 0, 3000], device=DEV)
    check_tempered(x, t, 5, temp)


@pytest.mark.parametrize("temp", [0.7, 1.4])
def test_token_stats_scores_what_the_sampler_drew(temp):
    """Log-prob of the drawn tokens under the distribution they were drawn from, from the same bf16 logits."""
    from tinytron_b200.inference.sampler import sample_next_token_with_log_prob

    torch.manual_seed(3)
    x = randn(gen(12), 64, 8000).mul_(2.5)
    tok, lp = sample_next_token_with_log_prob(x, temp)
    st = ops().token_stats(x, tok, temperature=temp)
    assert float((st.log_probs - lp).abs().max()) < 1e-4


def test_packed_scores_at_a_temperature_round_the_logits_once(monkeypatch):
    """packed_token_stats at T != 1 is log softmax(logits / T) of the LM head's own logits."""
    from tinytron_b200.models import GPT, ModelConfig

    c = ModelConfig(block_size=512, vocab_size=512, num_layer=1, num_attention_heads=4, num_key_value_heads=2, hidden_size=256,
                    intermediate_size=512, init_std=0.2, seed=5)
    m = GPT(c, device=DEV)
    g = torch.Generator().manual_seed(0)
    idx = torch.randint(0, 512, (300,), generator=g).to(DEV)
    labels = torch.randint(0, 512, (300,), generator=g).to(DEV)
    real, seen = ops().linear, []

    def linear(x, *w):
        y = real(x, *w)
        if w[0] is m.lm_head.weight:
            seen.append(y.detach())
        return y

    monkeypatch.setattr(ops(), "linear", linear)
    with torch.no_grad():
        st = m.packed_token_stats(idx, labels, i32([0, 100, 300]), temperature=0.7)
    assert len(seen) == 1 and seen[0].dtype == torch.bfloat16
    want = torch.log_softmax(seen[0].double() / 0.7, -1).gather(1, labels[:, None])[:, 0]
    assert float(want.abs().max()) > 1
    within(st.log_probs, want, 1e-4 + 2.0 ** -20 * want.abs(), "log-probs")


# ----------------------------------------------------------------------------- gradients that the kernels do not have
def test_serving_operators_refuse_to_lose_gradients():
    from tinytron_b200.inference import RaggedKVCache
    from tinytron_b200.models import GPT, ModelConfig
    from tinytron_b200.ops.rope import rope_tables

    g = gen(13)
    kp, vp = randn(g, 4, 16, 2, 64), randn(g, 4, 16, 2, 64)
    q, table, n = randn(g, 1, 4, 64), i32([[0, 1]]), i32([20])
    for i in range(3):
        args = [q, kp, vp]
        args[i] = args[i].clone().requires_grad_(True)
        with pytest.raises(ValueError, match="gradient"):
            ops().paged_attention(*args, table, n)
        with torch.no_grad():
            ops().paged_attention(*args, table, n)
    qkv = randn(g, 3, 8 * 64).requires_grad_(True)
    cos, sin = rope_tables(64, 10000.0, 64, DEV)
    with pytest.raises(ValueError, match="gradient"):
        ops().rotary_append(qkv, cos, sin, 4, 2, i32([0, 3]))
    with torch.no_grad():
        ops().rotary_append(qkv, cos, sin, 4, 2, i32([0, 3]))
    c = ModelConfig(block_size=64, vocab_size=128, num_layer=1, num_attention_heads=4, num_key_value_heads=2, hidden_size=256,
                    intermediate_size=256, seed=5)
    model, cache = GPT(c, device=DEV), RaggedKVCache.from_model_config(c, 4, 16, 2, DEV, torch.bfloat16)
    (s,) = cache.add()
    step = cache.prefill_step([s], [5])
    assert not model.forward_ragged(torch.arange(5, device=DEV), step).requires_grad


# ----------------------------------------------------------------------------- rejected entries
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cu", [[0, 301], [1, 300], [0, 200, 150, 300], [0, -2, 300]], ids=str)
def test_packed_attention_with_bad_offsets_gives_zeros(cu, d):
    q, k, v, do = packed_inputs([300], 4, 2, d, seed=4)
    dirty_memory()
    qkv = torch.cat([q, k, v], 1)  # gradients of views too
    got = run_packed(q, k, v, do, cu)
    assert status_and_clear() == K_BAD_INDEX
    for x in got:
        assert bool((x == 0).all())
    leaf = qkv.view(300, -1).clone().requires_grad_(True)
    dirty_memory()
    o = ops().rotary_packed_attention(leaf * 1, i32(cu), 4, 2, d)
    (grad,) = torch.autograd.grad(o, leaf, do.view(300, -1))
    assert status_and_clear() == K_BAD_INDEX
    assert bool((o == 0).all()) and bool((grad == 0).all())


def test_rotary_append_gives_zeros_at_bad_positions_and_the_rest_right():
    from tinytron_b200.ops.rope import rope_tables

    hq, hkv, d, page = 2, 1, 64, 16
    qkv = randn(gen(5), 9, (hq + 2 * hkv) * d)
    cos, sin = rope_tables(d, 10000.0, 64, DEV)
    cos, sin = cos[:64].contiguous(), sin[:64].contiguous()
    kp = torch.zeros(8, page, hkv, d, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    table = i32([[0, 1, 2, 3], [4, 5, -1, -1], [6, -1, -1, -1]])
    want = ops().rotary_append(qkv, cos, sin, hq, hkv, i32([0, 3, 6, 9]), i32([62, 4, 0]), want_k=True)
    assert status_and_clear() == K_BAD_INDEX  # the third token of the first sequence is at position 64
    dirty_memory()
    q, k = ops().rotary_append(qkv, cos, sin, hq, hkv, i32([0, 3, 6, 9]), i32([62, 4, 15]), kp, vp, table)
    assert status_and_clear() == K_BAD_INDEX
    assert bool((q[2] == 0).all()) and bool((k[2] == 0).all())
    for i in (0, 1, 3, 4, 5):
        assert torch.equal(q[i], want[0][i]) and torch.equal(k[i], want[1][i])
    at = [(3, 14), (3, 15), None, (4, 4), (4, 5), (4, 6), (6, 15), None, None]  # the last two fall onto no page
    kw, vw = torch.zeros_like(kp), torch.zeros_like(vp)
    for i, where in enumerate(at):
        if where is not None:
            kw[where], vw[where] = k[i], qkv[i].view(-1, d)[hq + hkv:]
    assert torch.equal(kp, kw) and torch.equal(vp, vw)


def test_bad_entries_leave_the_other_sequences_right():
    """A page that is not mapped, a length past the table, a target outside the vocabulary: the rows beside them hold."""
    g = gen(17)
    q, kp, vp = randn(g, 3, 4, 64), randn(g, 9, 16, 2, 64), randn(g, 9, 16, 2, 64)
    table, n = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), i32([40, 33, 48])
    want = ops().paged_attention(q, kp, vp, table, n)
    assert status_and_clear() == 0
    for t, m in ((i32([[0, 1, 2], [3, -1, 5], [6, 7, 8]]), n), (i32([[0, 1, 2], [3, 99, 5], [6, 7, 8]]), n), (table, i32([40, 1000, 48])),
                 (table, i32([40, -5, 48]))):
        got = ops().paged_attention(q, kp, vp, t, m)
        assert status_and_clear() == K_BAD_INDEX
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and bool(got.isfinite().all())
    x = randn(g, 3, 500, dtype=torch.float32).requires_grad_(True)
    good = ops().token_stats(x, torch.tensor([4, 7, 9], device=DEV), top_k=2)
    (ref,) = torch.autograd.grad(good.log_probs.sum() + good.entropy.sum(), x)
    st = ops().token_stats(x, torch.tensor([4, 500, 9], device=DEV), top_k=2)
    (grad,) = torch.autograd.grad(st.log_probs.sum() + st.entropy.sum(), x)
    assert status_and_clear() == K_BAD_INDEX
    for a, b in ((st.log_probs, good.log_probs), (st.entropy, good.entropy), (st.top_ids, good.top_ids), (grad, ref)):
        assert torch.equal(a[[0, 2]], b[[0, 2]])
    assert bool((grad[1] == 0).all()) and float(st.log_probs[1].detach()) == 0 and st.top_ids[1].tolist() == [-1, -1]


def test_a_recorded_bad_index_does_not_stop_later_kernels():
    """An index out of range costs its own entry only: kernels that run before the host looks are whole."""
    lens = [3000, 500, 45]
    q, k, v, do = packed_inputs(lens, 8, 2, 128, seed=6)
    clean = run_packed(q, k, v, do, cu_of(lens))
    a, b = randn(gen(7), 4096, 2048), randn(gen(8), 2048, 2048)
    prod = ops().linear(a, b)
    assert status_and_clear() == 0
    ops().token_stats(torch.zeros(1, 8, device=DEV), torch.tensor([8], device=DEV))
    got = run_packed(q, k, v, do, cu_of(lens))
    assert all(torch.equal(x, y) for x, y in zip(got, clean))
    assert torch.equal(ops().linear(a, b), prod)
    assert status_and_clear() == K_BAD_INDEX


# ----------------------------------------------------------------------------- errors reach the caller
def _cfg():
    from tinytron_b200.models import ModelConfig

    return ModelConfig(block_size=256, vocab_size=256, num_layer=1, num_attention_heads=4, num_key_value_heads=2, hidden_size=256,
                       intermediate_size=256, init_std=0.05, seed=5)


def test_ragged_generation_raises_on_a_recorded_error(monkeypatch):
    from tinytron_b200.inference import InferenceEngine, RaggedKVCache

    eng = InferenceEngine(_cfg(), device=DEV, kv_cache_page_size=16)
    cache = RaggedKVCache.from_model_config(_cfg(), 20, 16, 4, eng.device, torch.bfloat16)
    prompts = [torch.tensor([5, 9, 3]), torch.tensor([7])]
    real = RaggedKVCache.prefill_step
    with monkeypatch.context() as m:  # a prompt's page that is not mapped
        m.setattr(RaggedKVCache, "prefill_step", lambda self, *a: (lambda s: s._replace(page_table=torch.full_like(s.page_table, -1)))(real(self, *a)))
        with pytest.raises(RuntimeError, match="index"):
            eng.generate_ragged(prompts, 4, cache=cache)
    assert cache.free_pages == 20
    out = eng.generate_ragged(prompts, 4, cache=cache)
    assert out.lengths.tolist() == [4, 4]


def test_a_token_outside_the_vocabulary_reads_nothing():
    from tinytron_b200.inference import InferenceEngine

    table = randn(gen(16), 50, 64, dtype=torch.float32)
    got = ops().embedding(torch.tensor([3, -1, 49, 50, 1 << 40], device=DEV), table)
    assert status_and_clear() == K_BAD_INDEX
    assert torch.equal(got[[0, 2]], table[[3, 49]]) and bool((got[[1, 3, 4]] == 0).all())
    eng = InferenceEngine(_cfg(), device=DEV, kv_cache_page_size=16)
    with pytest.raises(RuntimeError, match="index"):
        eng.generate_ragged([torch.tensor([5, 256]), torch.tensor([7])], 4)


def test_launcher_does_not_step_on_a_recorded_error(monkeypatch):
    from tinytron_b200.launch import ragged as launch

    real, steps = launch.make_ragged_rollout, []

    def bad(gen):
        ro = real(gen)
        ro.cu_seqlens = ro.cu_seqlens + torch.tensor([0] * (ro.cu_seqlens.numel() - 1) + [5], dtype=torch.int32, device=DEV)
        return ro

    class Sgd(torch.optim.AdamW):
        def step(self, *a, **k):
            steps.append(1)
            return super().step(*a, **k)

    monkeypatch.setattr(launch, "make_ragged_rollout", bad)
    monkeypatch.setattr(torch.optim, "AdamW", Sgd)
    with pytest.raises(RuntimeError, match="index"):
        launch.main(["--device", "cuda", "--num_layer", "1", "--hidden_size", "256", "--num_attention_heads", "4",
                     "--num_key_value_heads", "2", "--intermediate_size", "256", "--vocab_size", "256", "--block_size", "256",
                     "--prompt_len", "2", "40", "--max_new_tokens", "4", "--num_prompts", "2", "--num_samples", "2", "--steps", "1"])
    assert not steps


# ----------------------------------------------------------------------------- fork and move
def test_fork_and_move_leave_rejected_entries_alone():
    g = gen(14)
    kp, vp = randn(g, 2, 8, 4, 1, 8), randn(g, 2, 8, 4, 1, 8)
    table, n = i32([[0, 1, 5], [-1, -1, -1], [2, -1, -1], [-1, -1, -1], [-1, -1, -1]]), i32([6, 0, 4, 0, 0])

    def after(f):
        x = [y.clone() for y in (kp, vp, table, n)]
        f(*x)
        assert status_and_clear() == K_BAD_INDEX
        return x

    def same(got, want=(kp, vp, table, n)):
        return all(torch.equal(a, b) for a, b in zip(got, want))

    for par, kid, new in ((5, 1, 3), (0, 7, 3), (0, 0, 3), (0, 1, 8), (-1, 1, 3), (2, 1, 3), (0, 1, 1)):
        got = after(lambda k, v, t, s: ops().fork_pages(k, v, t, s, i32([par]), i32([kid]), i32([new])))
        assert same(got), (par, kid, new)
        # beside a good entry, which is done
        want = [y.clone() for y in (kp, vp, table, n)]
        ops().fork_pages(*want, i32([0]), i32([4]), i32([6]))
        got = after(lambda k, v, t, s: ops().fork_pages(k, v, t, s, i32([par, 0]), i32([kid, 4]), i32([new, 6])))
        assert same(got, want), (par, kid, new)
    for src, dst in (([8], [3]), ([5], [-1]), ([5], [8]), ([5, 2], [3, 4]), ([2, 2], [3, 4]), ([5], [5]), ([-1], [3])):
        got = after(lambda k, v, t, s: ops().move_pages(k, v, t, i32(src), i32(dst)))
        if src == [2, 2]:  # the first is taken, the second is not ascending
            want = [y.clone() for y in (kp, vp, table, n)]
            ops().move_pages(*want[:3], i32([2]), i32([3]))
            assert same(got, want)
        else:
            assert same([x for x in got]), (src, dst)
    # the entries that are in order among some that are not: data and table agree
    src, dst = [0, 5, 1, 2], [3, 4, 6, 7]
    k, v, t, s = after(lambda k, v, t, s: ops().move_pages(k, v, t, i32(src), i32(dst)))
    for old, new in zip(src, dst):
        moved = bool((t == new).any())
        assert bool((t == old).any()) != moved
        for x, x0 in ((k, kp), (v, vp)):
            assert torch.equal(x[:, new], x0[:, old] if moved else x0[:, new])


# ----------------------------------------------------------------------------- accuracy by norms
# A rounding to bf16 errs by ulp / sqrt(12) in the root mean square; over mantissas m spread evenly in log m that is
# 2^-7 sqrt(E[1 / m^2] / 12) = 2^-7 sqrt(0.375 / ln 2 / 12) = 0.00166 of the value.  An output of independent terms, each with
# one such rounding inside (P, or dS), and its own rounding: sqrt(2) of it; the short rows at a sequence's start, whose terms
# are few, add delta's share: at most another 0.3 of its square.  With a tenth for the draw: 0.00166 sqrt(2.3) 1.1.
ROUND = 0.00166
NORM_BOUND = ROUND * math.sqrt(2.3) * 1.1


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 2, 64), (4, 4, 128)])
def test_packed_attention_accuracy_by_norm(hq, hkv, d):
    lens = [700, 45, 300, 1000]
    q, k, v, do = packed_inputs(lens, hq, hkv, d, seed=21)
    got = run_packed(q, k, v, do, cu_of(lens))
    ref = oracle.packed(q, k, v, cu_of(lens), do=do)
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        assert rel(x, ref[name]) < NORM_BOUND, (name, rel(x, ref[name]))


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_keeps_what_the_outputs_rounding_left(d):
    """o + o_lo, which delta = dO . O is taken from, carries P's rounding only; o alone has its own besides."""
    from tinytron_b200.ops import ragged

    lens = [700, 45, 300, 1000]
    q, k, v, _ = packed_inputs(lens, 8, 2, d, seed=22)
    cu = i32(cu_of(lens))
    o, (o_lo, _) = ragged._packed_fwd(q, k, v, cu, cu, 1.0 / math.sqrt(d), True)
    ref = oracle.packed(q, k, v, cu_of(lens))["o"]
    assert rel(o.double() + o_lo.double(), ref) < ROUND * 1.1
    assert rel(o, ref) > ROUND * 1.1  # the bound tells them apart


def test_packed_attention_directional_derivatives():
    """Derivatives along random directions against central differences in 64 bits, within the gradients' relative error
    (NORM_BOUND of the gradient's norm a direction, four sigma for eight of them together); a zero and a negated gradient fail."""
    lens, dirs, eps = [150, 9, 300], 8, 1e-5
    q, k, v, do = packed_inputs(lens, 2, 1, 64, seed=23)
    grads = run_packed(q, k, v, do, cu_of(lens))[1:]
    g = gen(24)
    for i, grad in enumerate(grads):
        want, got = [], []
        for _ in range(dirs):
            base = [x.double() for x in (q, k, v)]
            step = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
            f = []
            for s in (eps, -eps):
                x = list(base)
                x[i] = x[i] + s * step
                f.append(float((oracle.packed(*x, cu_of(lens))["o"] * do.double()).sum()))
            want.append((f[0] - f[1]) / (2 * eps))
            got.append(float((grad.double() * step).sum()))
        want, got = torch.tensor(want, dtype=torch.float64), torch.tensor(got, dtype=torch.float64)
        bound = 4 * NORM_BOUND * math.sqrt(dirs) * float(grad.double().norm())
        assert float((got - want).norm()) < bound
        assert float(want.norm()) > bound and float((got + want).norm()) > bound
