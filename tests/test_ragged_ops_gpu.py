"""sm_100a kernels of the ragged operators against their definitions in 64 bits, at the sizes and masks where
they can go wrong.  Bounds are elementwise (tests/ragged_oracle.py)."""
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


@pytest.fixture(autouse=True)
def _healthy():
    yield
    if torch.cuda.is_available():
        assert status_and_clear() == 0


# ----------------------------------------------------------------------------- packed attention
PACKINGS = [
    [1], [2, 1, 3], [127, 128, 129], [256, 0, 257], [0, 0, 5, 0], [64] * 9, [513, 33, 1, 300, 129], [1000, 1],
]


def packed_case(lens, hq, hkv, d, seed=0, tail=0, lens_k=None):
    g = gen(seed)
    n = sum(lens) + tail
    m = n if lens_k is None else sum(lens_k) + tail
    return (randn(g, n, hq, d), randn(g, m, hkv, d), randn(g, m, hkv, d), randn(g, n, hq, d))


def run_packed(q, k, v, do, cu, cu_k=None, scale=None):
    leaf = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = ops().packed_attention(*leaf, i32(cu), None if cu_k is None else i32(cu_k), scale)
    return [o.detach(), *torch.autograd.grad(o, leaf, do)]


@pytest.mark.parametrize("lens", PACKINGS, ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (3, 1, 64), (5, 5, 128)])
def test_packed_attention(lens, hq, hkv, d):
    q, k, v, do = packed_case(lens, hq, hkv, d, seed=len(lens))
    got = run_packed(q, k, v, do, cu_of(lens))
    ref = oracle.packed(q, k, v, cu_of(lens), do=do)
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        within(x, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("lens,lens_k", [([5, 3], [300, 3]), ([1, 1, 1], [1, 128, 257]), ([200, 130], [70, 130]),
                                         ([300, 4, 0], [0, 4, 9]), ([129, 384], [500, 300])], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_keys_of_their_own(lens, lens_k, d):
    """Sequences end together: more keys than queries (a cached context), or fewer (rows that see nothing)."""
    q, k, v, do = packed_case(lens, 4, 2, d, seed=7, lens_k=lens_k)
    got = run_packed(q, k, v, do, cu_of(lens), cu_of(lens_k), scale=0.2)
    ref = oracle.packed(q, k, v, cu_of(lens), cu_of(lens_k), do=do, scale=0.2)
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        within(x, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_rows_after_the_last_sequence_are_zero(d):
    lens = [130, 20]
    q, k, v, do = packed_case(lens, 2, 1, d, tail=300)
    got = run_packed(q, k, v, do, cu_of(lens))
    ref = oracle.packed(q, k, v, cu_of(lens), do=do)
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        assert bool((x[150:] == 0).all())
        within(x, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("poison", [math.nan, math.inf, -3.3e38])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_neighbours_do_not_leak(poison, d):
    """A sequence of infinities and NaN leaves the sequences beside it, and their gradients, as they are."""
    lens = [100, 60, 200]
    q, k, v, do = packed_case(lens, 4, 2, d, seed=3)
    clean = run_packed(q, k, v, do, cu_of(lens))
    bad = [x.clone() for x in (q, k, v, do)]
    for x in bad:
        x[100:160] = poison
    got = run_packed(*bad, cu_of(lens))
    for x, y in zip(got, clean):
        assert torch.equal(x[:100], y[:100]) and torch.equal(x[160:], y[160:])


def test_packed_attention_sharp_and_shifted_scores():
    """Scores far apart (the running maximum jumps by hundreds within a tile) and all far below zero."""
    lens = [300, 200]
    q, k, v, do = packed_case(lens, 2, 2, 128, seed=5)
    k = k * torch.linspace(0.1, 30, 500, device=DEV)[:, None, None].to(k.dtype)
    k[300:] = -k[300:].abs()
    q[300:] = q[300:].abs()
    got = run_packed(q, k, v, do, cu_of(lens))
    ref = oracle.packed(q, k, v, cu_of(lens), do=do)
    # scores reach hundreds: fp32 accumulation error of a score (2^-24 * sum |q k|) is no longer far below 2^-12
    s = float((q.double().abs().sum(-1).max() * k.double().abs().max()) / math.sqrt(128)) * 2.0 ** -22
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        within(x, ref[name], ref[name + "_tol"] * (1 + 256 * s), name)


@pytest.mark.parametrize("layout", ["qkv", "heads_first", "wide"])
def test_packed_attention_strides(layout):
    lens, hq, hkv, d = [77, 140], 4, 2, 128
    q, k, v, do = packed_case(lens, hq, hkv, d, seed=9)
    want = run_packed(q, k, v, do, cu_of(lens))
    n = q.shape[0]
    if layout == "qkv":
        x = torch.cat([q, k, v], 1)
        ins = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    elif layout == "heads_first":
        ins = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    else:  # an odd row stride that cannot be read in place: copied
        ins = []
        for x in (q, k, v):
            y = torch.zeros(n, x.shape[1], d + 3, dtype=x.dtype, device=DEV)
            y[:, :, :d] = x
            ins.append(y[:, :, :d])
    got = run_packed(*ins, do, cu_of(lens))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    # an expanded upstream gradient (of a sum) has no strides of its own
    leaf = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = ops().packed_attention(*leaf, i32(cu_of(lens)))
    a = torch.autograd.grad(o.sum(), leaf)
    b = run_packed(q, k, v, torch.ones_like(do), cu_of(lens))[1:]
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_packed_attention_repeats_bit_for_bit_and_in_a_batch():
    """No atomics in any sum: the same inputs give the same bits, and so does a sequence alone."""
    lens = [700, 45, 300]
    q, k, v, do = packed_case(lens, 8, 2, 128, seed=11)
    a, b = run_packed(q, k, v, do, cu_of(lens)), run_packed(q, k, v, do, cu_of(lens))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    i = slice(700, 745)
    alone = run_packed(q[i], k[i], v[i], do[i], [0, 45])
    assert all(torch.equal(x[i], y) for x, y in zip(a, alone))


def test_packed_attention_gradient_against_differences():
    lens = [150, 9]
    q, k, v, do = packed_case(lens, 2, 1, 64, seed=13)
    _, dq, dk, dv = run_packed(q, k, v, do, cu_of(lens))
    ref = oracle.packed(q, k, v, cu_of(lens), do=do)
    g = gen(14)
    for i, grad, tol in ((0, dq, "dq_tol"), (1, dk, "dk_tol"), (2, dv, "dv_tol")):
        base = [x.double() for x in (q, k, v)]
        step = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-5
        f = []
        for s in (eps, -eps):
            x = list(base)
            x[i] = x[i] + s * step
            f.append(float((oracle.packed(*x, cu_of(lens))["o"] * do.double()).sum()))
        want = (f[0] - f[1]) / (2 * eps)
        assert abs(float((grad.double() * step).sum()) - want) <= float((ref[tol] * step.abs()).sum()) + 1e-5 * abs(want)


def test_packed_attention_refusals_and_bad_offsets():
    q, k, v, _ = packed_case([10], 4, 2, 64)
    f = ops().packed_attention
    for args in [(q, k[:, :, :32], v[:, :, :32], i32([0, 10])), (q, k, v[:5], i32([0, 10])),
                 (q[:, :3], k, v, i32([0, 10])), (q, k, v, torch.tensor([0, 10], device=DEV)), (q, k, v, i32([[0, 10]])),
                 (q, k, v, torch.tensor([0, 10], dtype=torch.int32)), (q, k[:5], v[:5], i32([0, 10])),
                 (q.float(), k.float(), v.float(), i32([0, 10])), (q, k, v.float(), i32([0, 10]))]:
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError):
        f(q, k, v, i32([0, 10]), i32([0, 5, 10]))
    with pytest.raises(ValueError):
        f(q, k, v, i32([0, 10]), scale=0.0)
    wide = torch.zeros(10, 2, 96, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        f(wide, wide, wide, i32([0, 10]))
    assert status_and_clear() == 0
    for cu in ([0, 11], [1, 10], [0, 7, 5, 10], [0, -2, 10]):  # found on the device: nothing is read, the status tells
        run_packed(q, k, v, torch.zeros_like(q), cu)
        assert status_and_clear() == K_BAD_INDEX
    assert f(q[:0], k[:0], v[:0], i32([0, 0])).shape == (0, 4, 64)
    assert bool((f(q, k, v, i32([0])) == 0).all())


def test_packed_attention_first_call_of_a_thread():
    """A thread that has made no CUDA call yet has no context bound to it."""
    import threading

    q, k, v, do = packed_case([40, 7], 4, 2, 64, seed=1)
    want = run_packed(q, k, v, do, cu_of([40, 7]))
    cu, got = i32(cu_of([40, 7])), []

    def work():
        from tinytron_b200.ops import ragged

        o, saved = ragged._packed_fwd(q, k, v, cu, cu, 0.125, True)
        d = [torch.empty_like(x) for x in (q, k, v)]
        ragged._packed_bwd(q, k, v, o, *saved, do, cu, cu, 0.125, *d)
        got.extend([o, *d])

    torch.cuda.synchronize()
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 4 and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("d", [64, 128])
def test_rotary_packed_attention_matches_its_parts(d):
    from tinytron_b200.ops.rope import rope_tables

    lens, hq, hkv = [40, 1, 200], 4, 2
    n = sum(lens)
    g = gen(21)
    qkv = randn(g, n, (hq + 2 * hkv) * d)
    do = randn(g, n, hq * d)
    cu = i32(cu_of(lens))
    leaf = qkv.clone().requires_grad_(True)
    o = ops().rotary_packed_attention(leaf * 1, cu, hq, hkv, d, max_seqlen=max(lens))
    (grad,) = torch.autograd.grad(o, leaf, do)
    cos, sin = rope_tables(d, 10000.0, max(lens), DEV)
    q, k = ops().rotary_append(qkv, cos, sin, hq, hkv, cu)
    v = qkv.view(n, -1, d)[:, hq + hkv:]
    want = run_packed(q, k, v, do.view(n, hq, d), cu_of(lens))
    assert torch.equal(o.detach().view(n, hq, d), want[0])
    # the inverse rotation is the transpose: rotate the gradients of q and k back by hand, in 64 bits
    pos = torch.cat([torch.arange(x, device=DEV) for x in lens])
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    gr = grad.view(n, -1, d)
    for got, ref in ((gr[:, :hq], want[1]), (gr[:, hq:hq + hkv], want[2])):
        a, b = ref.double()[..., :d // 2], ref.double()[..., d // 2:]
        back = torch.cat([a * c + b * s, b * c - a * s], -1)
        within(got, back, 2.0 ** -8 * back.abs() + 2.0 ** -20 * ref.double().abs().amax(), "rotated gradient")
    assert torch.equal(gr[:, hq + hkv:], want[3])


# ----------------------------------------------------------------------------- decode
def paged_case(lens, hq, hkv, d, page, seed=0, width_extra=1, poison=math.nan):
    """Pages in no order; everything that no key of a sequence lies in is ``poison``."""
    g = gen(seed)
    need = [(n + page - 1) // page for n in lens]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(need + [0]) + width_extra
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    kp, vp = randn(g, pool, page, hkv, d), randn(g, pool, page, hkv, d)
    used = torch.zeros(pool, page, dtype=torch.bool, device=DEV)
    for r, n in zip(rows, lens):
        for j in range((n + page - 1) // page):
            used[r[j], :min(page, n - j * page)] = True
    for x in (kp, vp):
        x[~used] = poison
    return randn(g, len(lens), hq, d), kp, vp, i32(rows).reshape(len(lens), width), i32(lens)


def check_decode(q, kp, vp, table, lens, got):
    page, hkv, d = kp.shape[1:]
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            assert bool((got[b] == 0).all())
            continue
        rows = table[b, :(n + page - 1) // page].long()
        k, v = (x[rows].reshape(-1, hkv, d)[:n] for x in (kp, vp))
        ref = oracle.attention_one(q[b:b + 1], k, v)
        within(got[b:b + 1], ref["o"], ref["o_tol"], f"sequence {b} of {n}")


@pytest.mark.parametrize("page", [1, 16, 24, 128, 700])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (10, 2, 128), (8, 1, 64), (16, 1, 128), (16, 4, 128)])
def test_paged_attention(page, hq, hkv, d):
    lens = [1, 0, 63, 64, 65, 700, 17, 128, 3]
    case = paged_case(lens, hq, hkv, d, page, seed=page + hq)
    check_decode(*case, ops().paged_attention(*case))


@pytest.mark.parametrize("lens", [[5], [0], [9000], [20000, 1, 1, 1], [300] * 70, [0] * 200 + [65] * 3, [1] * 333], ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attention_batches(lens, d):
    """One long sequence over every CTA, many short ones, more sequences than a scan step."""
    case = paged_case(lens, 4, 2, d, 64, seed=len(lens))
    got = ops().paged_attention(*case)
    check_decode(*case, got)
    assert torch.equal(got, ops().paged_attention(*case))  # the join's order is fixed


def test_paged_attention_lengths_are_read_on_the_device():
    """A captured call replays with new lengths, on another stream than the eager calls."""
    lens = [100, 900, 0, 31]
    q, kp, vp, table, n = paged_case([1024] * 4, 8, 2, 128, 32, seed=2)
    n.copy_(i32(lens))
    ws = ops().paged_attention_workspace(4, 8, 2, 128, table.shape[1] * 32, DEV)
    ops().paged_attention(q, kp, vp, table, n, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops().paged_attention(q, kp, vp, table, n, workspace=ws)
    for new in (lens, [1024, 1, 5, 0], [64, 64, 64, 64]):
        n.copy_(i32(new))
        graph.replay()
        torch.cuda.synchronize()
        check_decode(q, kp, vp, table, n, got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops().paged_attention(q, kp, vp, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)


def test_paged_attention_strided_queries_and_scale():
    q, kp, vp, table, n = paged_case([77, 200], 4, 2, 128, 16, seed=4)
    wide = torch.zeros(2, 9, 128, dtype=q.dtype, device=DEV)
    wide[:, 2:6] = q
    got = ops().paged_attention(wide[:, 2:6], kp, vp, table, n, scale=0.3)
    ref = oracle.attention_one(q[1:2], kp[table[1, :13].long()].reshape(-1, 2, 128)[:200],
                               vp[table[1, :13].long()].reshape(-1, 2, 128)[:200], scale=0.3)
    within(got[1:2], ref["o"], ref["o_tol"], "strided")


def test_paged_attention_offsets_past_32_bits():
    """A pool whose last pages lie more than 2^32 bytes (and 2^31 elements) into it."""
    page, hkv, d = 128, 8, 128
    pages = (1 << 31) // (page * hkv * d) + 40
    kp = torch.zeros(pages, page, hkv, d, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    g = gen(6)
    ids = [pages - 1, 5, pages - 7]
    for i in ids:
        kp[i], vp[i] = randn(g, page, hkv, d), randn(g, page, hkv, d)
    q = randn(g, 1, 16, d)
    table, n = i32([ids]), i32([300])
    check_decode(q, kp, vp, table, n, ops().paged_attention(q, kp, vp, table, n))


def test_paged_attention_refusals_and_bad_entries():
    q, kp, vp, table, n = paged_case([50, 20], 4, 2, 64, 16, poison=0.0)
    f = ops().paged_attention
    for args in [(q[:1], kp, vp, table, n), (q, kp[:, :, :1], vp, table, n), (q, kp, vp, table.long(), n), (q, kp, vp, table, n.float()),
                 (q, kp, vp, table[:, :2], n), (q[:, :3], kp, vp, table, n), (q.float(), kp, vp, table, n), (q, kp, vp, table, n[:1])]:
        with pytest.raises(ValueError):
            f(*args)
    big = torch.zeros(2, 34, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        f(big, kp, vp, table, n)  # 17 query heads per kv head
    small = ops().paged_attention_workspace(1, 4, 2, 64, 16, DEV)
    with pytest.raises(RuntimeError, match="too small"):
        f(q, kp, vp, table, n, workspace=small)
    assert status_and_clear() == 0
    for bad in (-1, 1 << 20):
        t = table.clone()
        t[0, 1] = bad
        f(q, kp, vp, t, n)
        assert status_and_clear() == K_BAD_INDEX
    for wrong in ([-3, 20], [50, 10 ** 6]):  # a negative length, one past the table
        t = table.clamp_min(0)
        f(q, kp, vp, t, i32(wrong))
        assert status_and_clear() == K_BAD_INDEX
    assert f(q[:0], kp, vp, table[:0], n[:0]).shape == (0, 4, 64)


# ----------------------------------------------------------------------------- pages
@pytest.mark.parametrize("lens,past", [([1], [0]), ([5, 0, 130, 1], [3, 9, 0, 127]), ([1] * 40, list(range(40)))], ids=["one", "mixed", "step"])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 128, 16), (3, 1, 64, 100), (2, 2, 32, 1)])
def test_rotary_append(lens, past, hq, hkv, d, page):
    from tinytron_b200.ops.rope import rope_tables

    g = gen(1)
    n, tail = sum(lens), 2
    qkv = randn(g, n + tail, (hq + 2 * hkv) * d + 8)[:, :(hq + 2 * hkv) * d]  # a row stride of its own
    _, kp, vp, table, _ = paged_case([a + b for a, b in zip(past, lens)], hq, hkv, d, page, seed=5)
    cos, sin = rope_tables(d, 10000.0, 512, DEV)
    k0, v0 = kp.clone(), vp.clone()
    q, k = ops().rotary_append(qkv, cos, sin, hq, hkv, i32(cu_of(lens)), i32(past), kp, vp, table)
    owner = torch.tensor([b for b, x in enumerate(lens) for _ in range(x)], device=DEV, dtype=torch.long)
    pos = torch.tensor([p + i for p, x in zip(past, lens) for i in range(x)], device=DEV, dtype=torch.long)
    x = qkv[:n].view(n, -1, d) if qkv.is_contiguous() else qkv[:n].reshape(n, -1, d)
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x[:, :hq + hkv, :d // 2].double(), x[:, :hq + hkv, d // 2:].double()
    want = torch.cat([a * c - b * s, b * c + a * s], -1)
    got = torch.cat([q, k], 1)
    within(got[:n], want, 2.0 ** -8 * want.abs() + 2.0 ** -22 * (a.abs() + b.abs()).repeat(1, 1, 2), "rotation")
    assert bool((got[n:] == 0).all())
    where = table[owner, pos // page].long()
    k0[where, pos % page] = k[:n]
    v0[where, pos % page] = x[:, hq + hkv:]
    assert torch.equal(kp.view(torch.int16), k0.view(torch.int16)) and torch.equal(vp.view(torch.int16), v0.view(torch.int16))
    only_q, none = ops().rotary_append(qkv, cos, sin, hq, hkv, i32(cu_of(lens)), i32(past), want_k=False)
    assert none is None and torch.equal(only_q, q)


def test_rotary_append_bad_positions_and_pages():
    from tinytron_b200.ops.rope import rope_tables

    hq, hkv, d, page = 2, 1, 64, 16
    qkv = randn(gen(2), 3, (hq + 2 * hkv) * d)
    cos, sin = rope_tables(d, 10000.0, 64, DEV)
    kp = torch.zeros(4, page, hkv, d, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    f = lambda table, start: ops().rotary_append(qkv, cos, sin, hq, hkv, i32([0, 3]), i32(start), kp, vp, i32(table))  # noqa: E731
    for table, start in (([[0, -1]], [15]), ([[0, 9]], [15]), ([[0, 1]], [32]), ([[0, 1]], [-1]), ([[0, 1]], [10 ** 9])):
        f(table, start)
        assert status_and_clear() == K_BAD_INDEX
    with pytest.raises(ValueError):
        ops().rotary_append(qkv[:, :-d], cos, sin, hq, hkv, i32([0, 3]))
    with pytest.raises(ValueError):
        ops().rotary_append(qkv, cos, sin, hq, hkv, i32([0, 3]), i32([0, 0]))
    with pytest.raises(ValueError):
        ops().rotary_append(qkv, cos, sin, hq, hkv, i32([0, 3]), None, kp, vp)


@pytest.mark.parametrize("layers,page,hkv,d", [(None, 16, 2, 64), (3, 5, 1, 8), (2, 128, 8, 128)])
def test_fork_pages(layers, page, hkv, d):
    g = gen(3)
    lens = [page * 2 + 1, page, 0, 3 * page - 1]
    rows = [[7, 2, 9, -1], [4, -1, -1, -1], [-1] * 4, [1, 11, 3, -1]] + [[5] * 4 for _ in range(6)]
    lead = () if layers is None else (layers,)
    kp, vp = randn(g, *lead, 20, page, hkv, d), randn(g, *lead, 20, page, hkv, d)
    table, n = i32(rows), i32(lens + [99] * 6)
    parents, children, fresh = [0, 1, 0, 3, 2], [4, 5, 8, 6, 9], [12, -1, 13, 14, -1]
    k0, v0, t0, n0 = kp.clone(), vp.clone(), table.clone(), n.clone()
    ops().fork_pages(kp, vp, table, n, i32(parents), i32(children), i32(fresh))
    for p, c, f in zip(parents, children, fresh):
        t0[c], n0[c] = t0[p], n0[p]
        if f >= 0:
            last = lens[p] // page
            for x in (k0, v0):
                x[..., f, :, :, :] = x[..., rows[p][last], :, :, :]
            t0[c, last] = f
    for x, y in ((kp, k0), (vp, v0), (table, t0), (n, n0)):
        assert torch.equal(x, y)


def test_fork_and_move_refusals_and_bad_entries():
    kp = torch.zeros(2, 6, 4, 1, 8, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    table, n = i32([[0, 1], [-1, -1], [2, -1]]), i32([6, 0, 4])
    f = lambda p, c, x: ops().fork_pages(kp, vp, table, n, i32(p), i32(c), i32(x))  # noqa: E731
    for bad in (([5], [1], [3]), ([0], [7], [3]), ([0], [0], [3]), ([0], [1], [6]), ([-1], [1], [3]), ([2], [1], [3])):
        f(*bad)
        assert status_and_clear() == K_BAD_INDEX
    with pytest.raises(ValueError):
        f([0], [1, 2], [3])
    with pytest.raises(ValueError):
        ops().fork_pages(kp, vp[:, :3], table, n, i32([0]), i32([1]), i32([3]))
    with pytest.raises(ValueError):
        ops().move_pages(kp, vp, table, i32([3, 4]), i32([1]))
    with pytest.raises(ValueError):
        ops().move_pages(kp, vp, table.long(), i32([3]), i32([1]))
    for src, dst in (([6], [1]), ([4], [-1]), ([4, 3], [0, 1]), ([3], [3])):
        ops().move_pages(kp, vp, table, i32(src), i32(dst))
        assert status_and_clear() == K_BAD_INDEX


@pytest.mark.parametrize("pool,moves,page,hkv,d", [(9, 1, 1, 1, 8), (300, 100, 16, 2, 64), (40, 17, 128, 4, 128)])
def test_move_pages(pool, moves, page, hkv, d):
    g = gen(4)
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(1))
    src, dst = perm[:moves].sort().values, perm[moves:2 * moves]
    kp, vp = randn(g, 2, pool, page, hkv, d), randn(g, 2, pool, page, hkv, d)
    table = torch.full((7, pool // 2), -1, dtype=torch.int32)
    at = torch.randint(0, table.numel(), (pool,), generator=torch.Generator().manual_seed(2))
    table.view(-1)[at] = torch.arange(pool, dtype=torch.int32)
    k0, v0 = kp.clone(), vp.clone()
    for x in (k0, v0):
        x[:, dst.cuda()] = x[:, src.cuda()]
    to = torch.arange(pool, dtype=torch.int32)
    to[src] = dst.int()
    want = torch.where(table >= 0, to[table.long().clamp_min(0)], table)
    t = table.cuda()
    ops().move_pages(kp, vp, t, src.int().cuda(), dst.int().cuda())
    assert torch.equal(kp, k0) and torch.equal(vp, v0) and torch.equal(t.cpu(), want)


# ----------------------------------------------------------------------------- token statistics
def check_stats(x, t, top, ignore=-100, grads=True):
    leaf = x.detach().requires_grad_(True)
    st = ops().token_stats(leaf, t, top_k=top, ignore_index=ignore)
    lp, ent, tops, ids, y = oracle.token_stats(x, t, top, ignore)
    d = (x.double() - x.double().amax(-1, keepdim=True)).abs()
    near = d.gather(1, t.clamp_min(0)[:, None])[:, 0]
    within(st.log_probs, lp, 1e-5 + 2.0 ** -22 * near + 2.0 ** -22 * lp.abs(), "log-probs")
    within(st.entropy, ent, 2e-5 * (1 + ent), "entropy")
    assert torch.equal(st.top_ids, ids)
    within(st.top_log_probs, tops, 1e-5 + 2.0 ** -21 * tops.abs(), "top")
    if not grads:
        return
    g = gen(9)
    n = x.shape[0]
    ga, gb, gc = randn(g, n, dtype=torch.float32), randn(g, n, dtype=torch.float32), randn(g, n, top, dtype=torch.float32)
    outs = [st.log_probs, st.entropy] + ([st.top_log_probs] if top else [])
    (grad,) = torch.autograd.grad(outs, leaf, [ga, gb, gc][:len(outs)])
    want, mag = oracle.token_stats_grad(x, t, ga, gb, gc if top else None, ids, ignore)
    # the exponent's error is relative to |log p| (2^-23 each way); bf16 gradients are rounded once
    within(grad, want, 3e-5 * mag + (2.0 ** -8 * want.abs() if x.dtype == torch.bfloat16 else 0) + 1e-30, "gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (3, 2, 2), (5, 31, 7), (4, 512, 32), (7, 1001, 3), (2, 8192, 16), (33, 50304, 8), (2, 50257, 0)])
def test_token_stats(dtype, n, v, top):
    g = gen(n + v)
    x = randn(g, n, v, dtype=torch.float32).mul(3).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device=DEV)
    if n > 2:
        t[1] = -100
    check_stats(x, t, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_stats_masked_shifted_and_tied_logits(dtype):
    g = gen(5)
    v = 3000
    x = randn(g, 8, v, dtype=torch.float32).mul(2)
    low = torch.finfo(dtype).min
    x[0, ::2] = -math.inf      # half the vocabulary masked
    x[1, 7:] = low             # all but a few at the type's lowest value
    x[2] += 1000.0             # a large common offset
    x[3] = 1.5                 # one value: the alternatives are the lowest indices
    x[4, 100:] = -math.inf
    x[4, :100] = 2.0
    x[5] = low                 # nothing but the lowest value: uniform
    x[6, :] = -30.0
    x[6, 17] = 40.0            # all the mass on one token
    x = x.to(dtype)
    t = torch.tensor([1, 2, 5, 2999, 3, 0, 17, 11], device=DEV)
    check_stats(x, t, 5)


def test_token_stats_all_rows_tied_take_the_slow_path():
    x = torch.zeros(3, 20000, device=DEV, dtype=torch.bfloat16)
    x[1, 5::3] = 1.0
    x[2, -1] = 1.0
    check_stats(x, torch.tensor([4, 19999, 19999], device=DEV), 32)


def test_token_stats_without_a_distribution():
    x = torch.zeros(4, 700, device=DEV)
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2, 9] = math.inf
    st = ops().token_stats(x, torch.tensor([5, 6, 7, 8], device=DEV), top_k=3)
    want = torch.log_softmax(x.double(), -1)[torch.arange(4), torch.tensor([5, 6, 7, 8])]
    assert torch.equal(st.log_probs.isnan(), want.isnan()) and torch.equal(st.entropy.isnan(), want.isnan())
    assert st.top_ids[1].tolist() == [0, 1, 2] and st.top_ids[2].tolist() == [9, 0, 1] and st.top_ids[0].tolist() == [0, 1, 2]
    # the same rows, not scored: zeros and no gradient
    leaf = x.clone().requires_grad_(True)
    st = ops().token_stats(leaf, torch.tensor([-100, -100, -100, 8], device=DEV), top_k=3)
    (st.log_probs.sum() + st.entropy.sum() + st.top_log_probs.sum()).backward()
    assert bool((st.log_probs[:3] == 0).all()) and bool((st.top_ids[:3] == -1).all()) and bool((leaf.grad[:3] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_stats_strides_and_shapes(dtype):
    g = gen(8)
    wide = randn(g, 2, 5, 1011, dtype=torch.float32).to(dtype)
    x = wide[:, :, 3:1004]  # rows that start at no 16-byte boundary
    t = torch.randint(0, 1001, (2, 5), generator=g, device=DEV)
    st = ops().token_stats(x, t, top_k=4)
    flat = ops().token_stats(x.reshape(10, 1001).contiguous(), t.reshape(10), top_k=4)
    assert st.log_probs.shape == (2, 5) and st.top_log_probs.shape == (2, 5, 4)
    assert torch.equal(st.top_ids.reshape(10, 4), flat.top_ids)
    check_stats(wide.reshape(10, 1011)[:, 3:1004], t.reshape(10), 4)
    check_stats(wide.reshape(10, 1011)[:, 8:1009], t.reshape(10), 4)  # input and gradient rows aligned differently
    tr = wide.reshape(10, 1011).t().contiguous().t()
    check_stats(tr, t.reshape(10), 4)


def test_token_stats_partial_gradients_differences_and_refusals():
    g = gen(10)
    x = randn(g, 4, 600, dtype=torch.float32).requires_grad_(True)
    t = torch.randint(0, 600, (4,), generator=g, device=DEV)
    for pick in range(3):
        st = ops().token_stats(x, t, top_k=2)
        w = randn(g, *st[pick].shape, dtype=torch.float32)
        (grad,) = torch.autograd.grad((st[pick] * w).sum(), x)
        step = torch.randn(x.shape, generator=g, device=DEV, dtype=torch.float64)
        f = [float((oracle.token_stats(x.detach().double() + e * step, t, 2)[pick] * w.double()).sum()) for e in (1e-6, -1e-6)]
        want = (f[0] - f[1]) / 2e-6
        assert abs(float((grad.double() * step).sum()) - want) < 1e-4 * (1 + abs(want))
    f = ops().token_stats
    for args in [(x, t[:2]), (x, t.int()), (x.half(), t), (x, t.cpu())]:
        with pytest.raises(ValueError):
            f(*args)
    for k in (-1, 33):
        with pytest.raises(ValueError):
            f(x, t, top_k=k)
    with pytest.raises(ValueError):
        f(x[:, :4], t % 4, top_k=5)
    assert status_and_clear() == 0
    st = f(x, torch.tensor([600, -1, 3, 4], device=DEV), top_k=2)  # outside the vocabulary: not scored, and told
    assert status_and_clear() == K_BAD_INDEX
    assert bool((st.log_probs[:2] == 0).all()) and st.top_ids[:2].tolist() == [[-1, -1]] * 2
    assert f(x[:0], t[:0], top_k=2).top_ids.shape == (0, 2)
