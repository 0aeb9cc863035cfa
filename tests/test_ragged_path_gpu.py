"""Ragged generation and packed scoring on the GPU, against the engine's own one-prompt generation and the CPU model."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    from tinytron_b200.models import ModelConfig

    base = dict(block_size=512, vocab_size=512, num_layer=2, num_attention_heads=4, num_key_value_heads=2, hidden_size=256,
                intermediate_size=512, init_std=0.05, seed=5)
    base.update(kw)
    return ModelConfig(**base)


def _prompts(c, lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, c.vocab_size, (n,), generator=g) for n in lens]


def _score(model_cpu, seq, start):
    """log softmax of the CPU model at the positions that predict seq[start:], and which of them have routed clearly: where
    the k-th and the next router logit are closer than bf16 resolves, bf16 and fp32 run different experts, and there is no
    common value to compare."""
    clear = torch.ones(len(seq), dtype=torch.bool)

    def look(mlp, _, out):
        top = out[1][0].float().topk(mlp.top_k + 1, -1).values
        clear.logical_and_(top[:, -2] - top[:, -1] > 2.0 ** -5 * out[1][0].float().abs().amax(-1))

    hooks = [b.mlp.register_forward_hook(look) for b in model_cpu.blocks if model_cpu.use_moe]
    with torch.no_grad():
        y = model_cpu(seq[None])[0, start - 1:-1].float().log_softmax(-1)
    for h in hooks:
        h.remove()
    return y, clear[start - 1:-1]


@pytest.mark.parametrize("moe", [False, True])
@pytest.mark.parametrize("page", [16, 7])
def test_ragged_generation_follows_the_model(moe, page):
    """Every drawn token's statistics are those of the fp32 CPU model on the sequence so far, with bf16's distance;
    graph replay and eager steps agree exactly."""
    from tinytron_b200.inference import InferenceEngine
    from tinytron_b200.models import GPT
    from tinytron_b200.ops import check_status

    c = _cfg(use_moe=moe, num_experts=8, num_experts_per_tok=2, moe_intermediate_size=128)
    prompts = _prompts(c, [1, 40, 130, 17])
    outs = []
    for graph in (True, False):
        eng = InferenceEngine(c, device="cuda", kv_cache_page_size=page, use_cuda_graph=graph)
        torch.manual_seed(7)
        outs.append(eng.generate_ragged(prompts, 12, num_samples=3, temperature=0.8, top_k=20, alternatives=4))
    a, b = outs
    for name in ("new_tokens", "lengths", "log_probs", "entropy", "top_ids", "sampler_log_probs"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    cpu = GPT(c, device="cpu").eval()
    cpu.load_state_dict({k: v.cpu() for k, v in eng.model.state_dict().items()})
    checked = 0
    for i, seq in enumerate(a.sequences()):
        p = len(prompts[i // 3])
        y, clear = _score(cpu, seq.cpu(), p)
        got = a.log_probs[i].cpu()
        want = y.gather(1, seq.cpu()[p:, None])[:, 0]
        checked += int(clear.sum())
        assert float(((got - want).abs() * clear).max()) < 0.08
        assert float(((a.entropy[i].cpu() + (y.exp() * y).sum(-1)).abs() * clear).max()) < 0.08
    assert checked >= 72  # at least half of the tokens
    # answers of one prompt differ from each other, and all tokens are in the vocabulary
    assert len({tuple(r) for r in a.new_tokens.tolist()}) == 12
    check_status()


def test_greedy_ragged_generation_matches_one_prompt_at_a_time():
    """The same greedy tokens as ``generate`` of each prompt alone, up to a near-tie of bf16 logits."""
    from tinytron_b200.inference import InferenceEngine

    c = _cfg(init_std=0.2)
    eng = InferenceEngine(c, device="cuda", kv_cache_page_size=32)
    prompts = _prompts(c, [5, 100, 64, 33, 1])
    out = eng.generate_ragged(prompts, 10, top_k=1, alternatives=2)
    for i, p in enumerate(prompts):
        alone = eng.generate(p[None], 10, top_k=1)[0, len(p):].cpu()
        got = out.new_tokens[i].cpu()
        differ = (alone != got).nonzero()
        if len(differ):
            j = int(differ[0])
            gap = float(out.top_log_probs[i, j, 0] - out.top_log_probs[i, j, 1])
            assert gap < 0.1, (i, j, gap)


def test_ragged_generation_with_eos_in_a_shared_cache():
    from tinytron_b200.inference import InferenceEngine, RaggedKVCache

    c = _cfg(init_std=0.2)
    eng = InferenceEngine(c, device="cuda", kv_cache_page_size=16, eos_check_interval=3)
    prompts = _prompts(c, [9, 30])
    free = eng.generate_ragged(prompts, 16, num_samples=2, top_k=1)
    eos = int(free.new_tokens[0, 4])
    cache = RaggedKVCache.from_model_config(c, 40, 16, 4, eng.device, torch.bfloat16)
    out = eng.generate_ragged(prompts, 16, num_samples=2, top_k=1, eos_token_id=eos, cache=cache)
    for i in range(4):
        row = free.new_tokens[i].tolist()
        n = row.index(eos) + 1 if eos in row else 16
        assert int(out.lengths[i]) == min(n, out.new_tokens.shape[1])
        assert out.new_tokens[i, :n].tolist() == row[:n]
    assert cache.free_pages == 40


def test_packed_scores_and_gradients_match_cpu():
    from tinytron_b200.models import GPT

    c = _cfg()
    cpu = GPT(c, device="cpu")
    gpu = GPT(c, device="cuda")
    gpu.load_state_dict(cpu.state_dict())
    lens = [200, 3, 129, 64]
    seqs = _prompts(c, lens, seed=3)
    labels = torch.cat([torch.cat([s[1:], torch.tensor([-100])]) for s in seqs])
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    idx = torch.cat(seqs)
    outs = []
    for m, dev in ((cpu, "cpu"), (gpu, "cuda")):
        st = m.packed_token_stats(idx.to(dev), labels.to(dev), cu.to(dev), top_k=3, max_seqlen=200)
        w = torch.linspace(-1, 1, len(idx), device=dev)
        ((st.log_probs * w).sum() + 0.1 * st.entropy.sum()).backward()
        outs.append(st)
    assert float((outs[0].log_probs - outs[1].log_probs.cpu()).abs().max()) < 0.08
    assert float((outs[0].entropy - outs[1].entropy.cpu()).abs().max()) < 0.08
    for (name, a), (_, b) in zip(cpu.named_parameters(), gpu.named_parameters()):
        rel = float((b.grad.cpu() - a.grad).norm() / a.grad.norm())
        assert rel < 6e-2, (name, rel)  # the bound of the flagship smoke test's gradients


def test_launcher_on_the_gpu():
    from tinytron_b200.launch.ragged import main

    log = main(["--device", "cuda", "--num_layer", "2", "--hidden_size", "256", "--num_attention_heads", "4",
                "--num_key_value_heads", "2", "--intermediate_size", "512", "--vocab_size", "512", "--block_size", "512",
                "--prompt_len", "2", "200", "--max_new_tokens", "8", "--num_prompts", "5", "--num_samples", "3", "--steps", "2"])
    assert [x["new_tokens"] for x in log] == [120, 120] and all(abs(x["loss"]) < 10 for x in log)
