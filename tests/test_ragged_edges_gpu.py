"""Edges of the ragged operators on the GPU: values that are not finite, rejected entries, temperatures, lost
gradients, accuracy by norms."""
import math

import pytest
import torch

import ragged_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


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
