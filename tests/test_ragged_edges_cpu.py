"""Edges of the ragged operators on the host: ids of near ties and NaN, bad offsets and entries, the cache's states
after an error, arguments that lie elsewhere."""
import math

import pytest
import torch

import ragged_oracle as oracle
from tinytron_b200 import ops
from tinytron_b200.inference import InferenceEngine, RaggedKVCache
from tinytron_b200.models import GPT, ModelConfig
from tinytron_b200.rl import group_advantages, make_ragged_rollout, ragged_grpo_loss


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


# ----------------------------------------------------------------------------- token statistics
def test_token_stats_ids_follow_the_logits():
    """Logits that differ by less than a log-prob's rounding are in their own order; a NaN is below every number."""
    x = torch.zeros(4, 50)
    x[0, 40], x[0, 10], x[0, 20] = 18.0, 1e-3, 1e-3 + 1.2e-10
    assert float(x[0, 20]) > float(x[0, 10])
    x[1, 3], x[1, 7] = math.nan, 1.0
    x[2] = -math.inf
    x[2, 5], x[2, 6] = math.nan, 2.0
    x[3, 0], x[3, 1], x[3, 2] = -0.0, math.inf, 1.0
    st = ops.token_stats(x, torch.tensor([40, 7, 6, 1]), top_k=4)
    assert st.top_ids.tolist() == [[40, 20, 10, 0], [7, 0, 1, 2], [6, 0, 1, 2], [1, 2, 0, 3]]
    last = ops.token_stats(x[1:2, :20], torch.tensor([7]), top_k=20).top_ids[0]
    assert int(last[-1]) == 3


def test_token_stats_temperature():
    """Log-probs, entropy, alternatives and gradients of softmax(logits / T)."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 300, generator=g).mul(3)
    t = torch.randint(0, 300, (6,), generator=g)
    t[2] = -100
    for temp in (0.7, 2.5):
        leaf = x.clone().requires_grad_(True)
        st = ops.token_stats(leaf, t, top_k=3, temperature=temp)
        z = x.double() / temp
        lp, ent, tops, ids, _ = oracle.token_stats(z, t, 3)
        assert torch.equal(st.top_ids, ids)
        for a, b in ((st.log_probs, lp), (st.entropy, ent), (st.top_log_probs, tops)):
            assert torch.allclose(a.double(), b, atol=1e-5)
        ga, gb, gc = torch.randn(6, generator=g), torch.randn(6, generator=g), torch.randn(6, 3, generator=g)
        (grad,) = torch.autograd.grad([st.log_probs, st.entropy, st.top_log_probs], leaf, [ga, gb, gc])
        want, _ = oracle.token_stats_grad(z, t, ga, gb, gc, ids)
        assert torch.allclose(grad.double(), want / temp, atol=1e-5)
    for bad in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            ops.token_stats(x, t, temperature=bad)


def test_policy_ratio_is_one_at_a_temperature():
    """The actor is the sampler at T != 1 too."""
    c = cfg()
    eng = InferenceEngine(c, device="cpu", dtype=torch.float32, kv_cache_page_size=4)
    torch.manual_seed(1)
    gen = eng.generate_ragged([torch.tensor([3, 4, 5]), torch.tensor([6])], 6, num_samples=3, temperature=0.6)
    actor = GPT(c, device="cpu")
    actor.load_state_dict(eng.model.state_dict())
    out = ragged_grpo_loss(actor, make_ragged_rollout(gen), group_advantages(torch.arange(6.0), 3), temperature=0.6)
    assert abs(float(out.metrics["mean_ratio"]) - 1) < 1e-4 and float(out.metrics["clip_frac"]) == 0


# ----------------------------------------------------------------------------- offsets and entries
def cfg(**kw):
    base = dict(block_size=128, vocab_size=120, num_layer=2, num_attention_heads=4, num_key_value_heads=2, hidden_size=64,
                intermediate_size=96, init_std=0.05, seed=3)
    base.update(kw)
    return ModelConfig(**base)


@pytest.mark.parametrize("cu", [[0, 11], [1, 10], [0, 7, 5, 10], [0, -2, 10]], ids=str)
def test_packed_attention_refuses_bad_offsets(cu):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(10, h, 16, generator=g) for h in (4, 2, 2))
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.packed_attention(q, k, v, i32(cu))
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.packed_attention(q, k, v, i32([0] + [10] * (len(cu) - 1)), i32(cu))


def test_rotary_append_tokens_before_the_first_sequence_belong_to_none():
    from tinytron_b200.ops.rope import rope_tables

    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(7, 8 * 8, generator=g)
    cos, sin = rope_tables(8, 10000.0, 64, "cpu")
    kp, vp = torch.zeros(3, 4, 2, 8), torch.zeros(3, 4, 2, 8)
    q, k = ops.rotary_append(qkv, cos, sin, 4, 2, i32([2, 5]), None, kp, vp, i32([[1]]))
    want = ops.rotary_append(qkv[2:5], cos, sin, 4, 2, i32([0, 3]))
    assert torch.equal(q[2:5], want[0]) and torch.equal(k[2:5], want[1])
    for x in (q, k):
        assert bool((x[:2] == 0).all()) and bool((x[5:] == 0).all())
    assert bool((kp[0] == 0).all()) and bool((kp[2] == 0).all()) and torch.equal(kp[1, :3], want[1])


def test_fork_and_move_refuse_bad_entries_and_change_nothing():
    g = torch.Generator().manual_seed(2)
    kp, vp = torch.randn(2, 8, 4, 1, 8, generator=g), torch.randn(2, 8, 4, 1, 8, generator=g)
    table, n = i32([[0, 1, 5], [-1, -1, -1], [2, -1, -1], [-1, -1, -1]]), i32([6, 0, 4, 0])
    was = [x.clone() for x in (kp, vp, table, n)]
    for par, kid, new in ((5, 1, 3), (0, 7, 3), (0, 0, 3), (0, 1, 8), (-1, 1, 3), (2, 1, 3), (0, 1, 1)):
        with pytest.raises(ValueError):
            ops.fork_pages(kp, vp, table, n, i32([0, par]), i32([3, kid]), i32([6, new]))
    for src, dst in (([8], [3]), ([5], [-1]), ([5], [8]), ([5, 2], [3, 4]), ([2, 2], [3, 4]), ([5], [5]), ([-1], [3])):
        with pytest.raises(ValueError):
            ops.move_pages(kp, vp, table, i32(src), i32(dst))
    assert all(torch.equal(a, b) for a, b in zip((kp, vp, table, n), was))


# ----------------------------------------------------------------------------- the cache after an error
def state(cache):
    return (list(map(lambda r: None if r is None else list(r), cache._rows)), list(cache._lens), list(cache._refs),
            sorted(cache._free), sorted(cache._free_seqs))


def test_fork_that_fails_gives_back_what_it_took(monkeypatch):
    cache = RaggedKVCache(1, 1, 2, 10, 4, 6, 16, "cpu", torch.float32)
    a, b = cache.add(2)
    cache.reserve([a, b], [6, 4])
    cache.advance([a, b], [6, 4])
    before = state(cache)

    def fail(*_):
        raise RuntimeError("no launch")

    with monkeypatch.context() as m:
        m.setattr(ops, "fork_pages", fail)
        with pytest.raises(RuntimeError, match="no launch"):
            cache.fork([a, a, b])
    assert state(cache) == before
    kids = cache.fork([a, a, b])  # and it works afterwards
    cache._sync()
    assert [cache.length(k) for k in kids] == [6, 6, 4]
    assert cache.page_table[kids[0]].tolist()[0] == cache.pages_of(a)[0]
    cache.free([a, b, *kids])
    assert cache.free_pages == 10


def test_resize_that_runs_out_of_memory_changes_nothing(monkeypatch):
    cache = RaggedKVCache(1, 1, 2, 10, 4, 6, 16, "cpu", torch.float32)
    real, calls = torch.empty, []

    def empty(*a, **k):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("out of memory")
        return real(*a, **k)

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        with pytest.raises(RuntimeError, match="out of memory"):
            cache.resize(5)
    assert cache.k_pages.shape == cache.v_pages.shape and cache.num_pages == len(cache._refs) == 10
    cache.resize(5)
    assert cache.k_pages.shape[1] == cache.v_pages.shape[1] == 5 and cache.free_pages == 5
    with pytest.raises(ValueError):
        cache.resize(-1)


def test_decode_step_needs_its_pages():
    """A step whose token has no mapped page, or that names a sequence twice, is refused on the host."""
    cache = RaggedKVCache(1, 1, 2, 10, 4, 6, 8, "cpu", torch.float32)
    a, b = cache.add(2)
    cache.reserve([a, b], [4, 3])
    cache.advance([a, b], [4, 3])
    with pytest.raises(ValueError, match="reserve"):
        cache.decode_step([a, b])
    with pytest.raises(ValueError, match="twice"):
        cache.decode_step([b, b])
    cache.reserve([a], [1])
    step = cache.decode_step([a, b])
    assert step.seq_lens.tolist() == [5, 4]
    for f in (cache.reserve, cache.advance):
        with pytest.raises(ValueError):
            f([a], [-1])
    with pytest.raises(ValueError):
        cache.prefill_step([99], [2])


def test_a_workspace_made_in_a_capture_stays_there(monkeypatch):
    """Scratch that is cleared by a captured step holds nothing valid outside of it."""
    cache = RaggedKVCache(1, 1, 2, 4, 4, 2, 16, "cpu", torch.float32)
    cache.device = torch.device("cuda")
    capturing, made = [True], []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(ops, "paged_attention_workspace", lambda *a: made.append(object()) or made[-1])
    inside = cache.workspace(2, 4)
    capturing[0] = False
    outside = cache.workspace(2, 4)
    assert outside is not inside and cache.workspace(2, 4) is outside
    capturing[0] = True
    assert cache.workspace(2, 4) is outside  # cleared before the capture: shared with it


# ----------------------------------------------------------------------------- the policy loss
def test_ignore_index_of_a_rollout_is_the_losss():
    c = cfg()
    eng = InferenceEngine(c, device="cpu", dtype=torch.float32, kv_cache_page_size=4)
    torch.manual_seed(0)
    gen = eng.generate_ragged([torch.tensor([3, 4, 5]), torch.tensor([6])], 5, num_samples=3)
    actor = GPT(c, device="cpu")
    actor.load_state_dict(eng.model.state_dict())
    adv = group_advantages(torch.arange(6.0), 3)
    outs = []
    for ignore in (-100, -7):
        ro = make_ragged_rollout(gen, ignore_index=ignore)
        assert int((ro.labels == ignore).sum()) == ro.labels.numel() - int(gen.lengths.sum())
        outs.append(ragged_grpo_loss(actor, ro, adv, entropy_coef=0.1))
    assert torch.equal(outs[0].loss, outs[1].loss)
    assert abs(float(outs[1].metrics["mean_ratio"]) - 1) < 1e-4
