"""Operators of drafted-token trees and of logits before sampling on the GPU, against 64-bit loops (``tree_oracle``)."""

import math

import pytest
import torch
import tree_oracle as oracle

pytestmark = pytest.mark.gpu

F32, BF16 = 2.0**-24, 2.0**-8  # half a step


@pytest.fixture(scope="module", autouse=True)
def _built(kernels):
    yield


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def attention_case(sizes, ctx, heads, page, seed=0, holes=0.0, shape="random", dtype=torch.bfloat16, packed=False, spare=0):
    """Caches are NaN wherever no token stands; the page table points far away behind a request's pages; ``spare`` rows of q follow the
    last tree. ``packed``: q is a column range of a wider matrix, the caches are two halves of one tensor."""
    Hq, Hkv, D = heads
    g = torch.Generator().manual_seed(seed)
    cu, parents = oracle.make_trees(sizes, seed, holes, shape)
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, sizes)], page, seed)
    T = int(cu[-1]) + spare
    kv = torch.full((slots, 2, Hkv, D), math.nan).to(dtype)
    for b, (c, n) in enumerate(zip(ctx, sizes)):
        at = torch.tensor([oracle.slot(table, b, p, page) for p in range(c + n)], dtype=torch.long)
        kv[at] = torch.randn(c + n, 2, Hkv, D, generator=g).to(dtype)
    wide = (2 * torch.randn(T, Hq + 2, D, generator=g)).to(dtype)
    if packed:
        wide, kv = wide.cuda(), kv.cuda()
        q, k, v = wide[:, 1:-1], kv[:, 0], kv[:, 1]
    else:
        q, k, v = wide[:, 1:-1].contiguous().cuda(), kv[:, 0].contiguous().cuda(), kv[:, 1].contiguous().cuda()
    parents = torch.cat([parents, torch.zeros(spare, dtype=torch.int32)])
    return q, k, v, *cuda(table, torch.tensor(ctx, dtype=torch.int32), cu, parents)


def bound(want, mass, dtype, D):
    """Scores are sums of D products, off by D roundings of fp32 of some 14 on this scale (1e-4) and by that factor in the weights; bf16 kernels round the weights
    to bf16, and every kernel its output."""
    weights = 1e-4 + (BF16 if dtype == torch.bfloat16 else 0)
    return weights * mass + (BF16 if dtype == torch.bfloat16 else F32) * want.abs() + 1e-6


SIZES = [
    ([1], [0]),
    ([1], [1]),
    ([8], [1023]),
    ([3, 1, 0, 17], [127, 128, 5, 129]),
    ([16, 16, 16], [112, 0, 500]),
    ([64, 5], [1000, 64]),
    ([31, 61, 2], [97, 3, 255]),
    ([128, 100], [40, 300]),
    ([2] * 40, list(range(40))),
]
HEADS = [(14, 2, 64), (4, 4, 64), (32, 8, 128), (16, 1, 128), (8, 1, 128), (2, 2, 128)]


@pytest.mark.parametrize("sizes, ctx", SIZES)
@pytest.mark.parametrize("heads", HEADS)
def test_attention_bf16(sizes, ctx, heads):
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case(sizes, ctx, heads, 16, seed=len(sizes), holes=0.1 if len(sizes) > 1 else 0.0)
    got = ops.tree_attention(q, k, v, table, c, cu, parents, 16, max(sizes))
    want, mass = oracle.attention(q, k, v, table, c, cu, parents, 16, heads[2] ** -0.5)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound(want, mass, torch.bfloat16, heads[2])).all(), float((err / (mass + 1e-9)).max())


@pytest.mark.parametrize("heads, page", [((4, 2, 8), 4), ((6, 2, 80), 16), ((2, 1, 256), 32), ((3, 3, 5), 1), ((14, 2, 64), 16), ((8, 2, 128), 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_every_width_and_page(heads, page, dtype):
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([3, 1, 0, 17], [127, 128, 5, 40], heads, page, holes=0.1, dtype=dtype)
    got = ops.tree_attention(q, k, v, table, c, cu, parents, page, 17)
    want, mass = oracle.attention(q, k, v, table, c, cu, parents, page, heads[2] ** -0.5)
    assert ((got.double().cpu() - want).abs() <= bound(want, mass, dtype, heads[2])).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 48])
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
def test_attention_strides_sinks_factors_and_pages(page, heads):
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([9, 1, 33], [300, 17, 65], heads, page, packed=True, spare=3)
    sinks = torch.randn(heads[0], device="cuda")
    for scale, s in ((None, sinks), (0.3, None), (-0.05, sinks), (0.0, None)):
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        assert ops.tree_attention(q, k, v, table, c, cu, parents, page, 33, scale=scale, sinks=s, out=out) is out
        f = heads[2] ** -0.5 if scale is None else scale
        want, mass = oracle.attention(q, k, v, table, c, cu, parents, page, f, s)
        # (a factor of 0.3 makes scores of up to a hundred: their sums are off by as much more)
        slack = 1 + abs(f) / heads[2] ** -0.5
        n = int(cu[-1])
        assert ((out[:n].double().cpu() - want[:n]).abs() <= slack * bound(want, mass, torch.bfloat16, heads[2])[:n]).all()
        assert (out[n:] == 7).all()


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (16, 1, 128), (8, 1, 128), (2, 2, 64), (4, 2, 8)])
@pytest.mark.parametrize("sizes, ctx", [([8, 1], [120, 16]), ([31, 61, 2], [97, 3, 255]), ([128, 100, 9], [40, 300, 2000])])
@pytest.mark.parametrize("what", ["keys", "values", "one value"])
def test_attention_beside_numbers_that_are_not_finite(heads, sizes, ctx, what):
    """NaN in nodes of no tree and in one node of each tree, infinities in a cached token of the last request: rows that see none of them are as ever, the others not finite."""
    from slime_b200 import ops

    page = 16
    q, k, v, table, c, cu, parents = attention_case(sizes, ctx, heads, page, seed=3, holes=0.15)
    par, starts = parents.tolist(), cu.tolist()
    x = k if what == "keys" else v
    last = slice(0, 1) if what == "one value" else slice(None)
    for b, n in enumerate(sizes):
        for i in range(n):
            if i == n // 2 or (i > 0 and not oracle.way_up(par[starts[b] : starts[b + 1]], i)):
                x[oracle.slot(table, b, ctx[b] + i, page), :, last] = math.nan
    if len(sizes) > 2:
        x[oracle.slot(table, 2, ctx[2] // 3, page), :, last] = math.inf
    got = ops.tree_attention(q, k, v, table, c, cu, parents, page, max(sizes)).double().cpu()
    want, mass = oracle.attention(q, k, v, table, c, cu, parents, page, heads[2] ** -0.5)
    fine = want.isfinite()
    assert not got[~fine].isfinite().any() and (~fine).any()
    rows = fine.all(2) & mass.isfinite().all(2)
    assert rows.any() and ((got - want).abs() <= bound(want, mass, torch.bfloat16, heads[2]))[rows].all()


@pytest.mark.parametrize("heads", [(8, 2, 64), (16, 4, 128), (6, 2, 40)])
def test_attention_of_caches_laid_out_otherwise(heads):
    """Heads outside slots, one head for all, a head of its own whose pitch means nothing, keys and values of other pitches, queries with heads outside rows."""
    from slime_b200 import ops

    Hq, Hkv, D = heads
    q, k, v, table, c, cu, parents = attention_case([9, 1, 33], [300, 17, 65], heads, 16)
    rest = (table, c, cu, parents, 16, 33)
    turned = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    want = ops.tree_attention(q, k, v, *rest)
    assert torch.equal(want, ops.tree_attention(turned(q), turned(k), v, *rest))
    assert torch.equal(want, ops.tree_attention(q, torch.cat([k, k], 1)[:, :Hkv], turned(v), *rest))
    one = [x[:, :1].contiguous() for x in (k, v)]
    same = ops.tree_attention(q, *(x.repeat(1, Hkv, 1) for x in one), *rest)
    assert torch.equal(same, ops.tree_attention(q, *(x.expand(-1, Hkv, -1) for x in one), *rest))
    lone = ops.tree_attention(q, *one, *rest)
    odd = [x.as_strided(x.shape, (D, 3, 1)) for x in one]  # (the pitch of a single head)
    want, mass = oracle.attention(q, *one, table, c, cu, parents, 16, D**-0.5)
    for got in (lone, ops.tree_attention(q, *odd, *rest)):
        assert ((got.double().cpu() - want).abs() <= bound(want, mass, torch.bfloat16, D)).all()


@pytest.mark.parametrize("shape", ["chain", "star"])
def test_attention_of_chains_and_stars(shape):
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([70, 20], [60, 2000], (32, 8, 128), 16, shape=shape)
    got = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 70)
    want, mass = oracle.attention(q, k, v, table, c, cu, parents, 16, 128**-0.5)
    assert ((got.double().cpu() - want).abs() <= bound(want, mass, torch.bfloat16, 128)).all()


def test_attention_of_a_long_cache_and_empty_calls():
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([6, 12], [20011, 9000], (8, 2, 128), 16)
    got = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 12)
    want, mass = oracle.attention(q, k, v, table, c, cu, parents, 16, 128**-0.5)
    assert ((got.double().cpu() - want).abs() <= bound(want, mass, torch.bfloat16, 128)).all()
    assert ops.tree_attention(q[:0], k, v, table, c, torch.zeros_like(cu), parents[:0], 16, 12).shape == (0, 8, 128)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.tree_attention(q[:0], k, v, table[:0], c[:0], none, parents[:0], 16, 12).shape == (0, 8, 128)


@pytest.mark.parametrize("page", [16, 24])
def test_caches_of_more_than_32_bits(page):
    """The rows in use stand behind 2^31 elements, 2^32 bytes."""
    from slime_b200 import ops

    heads, sizes, ctx = (16, 8, 64), [9, 17], [150, 33]
    q, k, v, table, c, cu, parents = attention_case(sizes, ctx, heads, page)
    first = -(-(1 << 22) // page) * page
    big = torch.empty(2, 1, first + k.shape[0], 8, 64, dtype=torch.bfloat16, device="cuda")
    big[0, 0, first:], big[1, 0, first:] = k, v
    far = table + first // page
    got = ops.tree_attention(q, big[0, 0], big[1, 0], far, c, cu, parents, page, 17)
    assert torch.equal(got, ops.tree_attention(q, k, v, table, c, cu, parents, page, 17))
    sampled, drafted, parents, cu = accept_case(sizes, 2, 1.0)
    want = oracle.accepted(sampled, drafted, parents, cu, 17)
    after = oracle.moved([k.cpu()[None], v.cpu()[None]], table.cpu(), ctx, [w[0] for w in want], [w[2] for w in want], page)
    ops.accept_tree(*cuda(sampled, drafted, parents, cu), 17, k_caches=big[0], v_caches=big[1], block_table=far, context_lens=c, page_size=page)
    for x, y in zip(big[:, 0, first:].cpu(), after):
        torch.testing.assert_close(x, y[0], rtol=0, atol=0, equal_nan=True)


def test_attention_is_the_same_every_time_and_with_other_requests_beside_it_where_asked():
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([9] * 12, [400 + 37 * i for i in range(12)], (14, 2, 64), 16)
    a = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 9)
    for _ in range(3):
        assert torch.equal(a, ops.tree_attention(q, k, v, table, c, cu, parents, 16, 9))
    ops.set_batch_invariant(True)
    try:
        a = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 9)
        for b in (0, 7):
            lone = ops.tree_attention(q[9 * b : 9 * b + 9], k, v, table[b : b + 1], c[b : b + 1], cu[:2], parents[9 * b : 9 * b + 9], 16, 9)
            assert torch.equal(lone, a[9 * b : 9 * b + 9])
    finally:
        ops.set_batch_invariant(False)


def test_attention_on_another_stream_and_in_a_graph():
    from slime_b200 import ops

    q, k, v, table, c, cu, parents = attention_case([9, 30], [400, 77], (32, 8, 128), 16)
    want = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 30)
    side.synchronize()
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 30)
    # other lengths and trees of the same packed rows
    c.copy_(torch.tensor([390, 80], dtype=torch.int32))
    cu[1] = 20
    parents[9:20] = torch.arange(8, 19, dtype=torch.int32, device="cuda")
    parents[20] = -1
    q2 = q.clone()
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    table_full = table.clone()
    del q2
    fresh = ops.tree_attention(q, k.nan_to_num(0.0), v.nan_to_num(0.0), table_full.clamp(max=k.shape[0] // 16 - 1), c, cu, parents, 16, 30)
    assert fresh.isfinite().all()
    assert torch.equal(held.nan_to_num(5.0)[:20], ops.tree_attention(q, k, v, table, c, cu, parents, 16, 30).nan_to_num(5.0)[:20])


# -------------------------------------------------------------------------------------------------------------- logits
def logits_case(S, V, sizes=None, seed=0, L=23, K=5, dtype=torch.float32, parts=("repetition", "frequency", "presence", "bias", "allowed")):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, dtype=torch.int32)  # noqa: E731
    R = S if sizes is None else sum(sizes)
    kw = dict(tokens=ints(-2, V + 2, S, L) // 3, lengths=ints(0, L + 1, S), prompt_lens=ints(0, L + 1, S))
    if "repetition" in parts:
        kw["repetition"] = 0.5 + rnd(S)
    if "frequency" in parts:
        kw["frequency"] = rnd(S) - 0.3
    if "presence" in parts:
        kw["presence"] = rnd(S) - 0.3
    if "bias" in parts:
        kw["bias_ids"], kw["bias_values"] = ints(-3, V + 3, S, K) // 2, torch.randn(S, K, generator=g)
    if "allowed" in parts:
        kw["allowed"] = torch.randint(-(1 << 31), 1 << 31, (R, -(-V // 32)), generator=g).to(torch.int32)
        kw["allowed"][R // 2] = 0
    if sizes is not None:
        cu, parents = oracle.make_trees(sizes, seed, holes=0.1)
        kw["tree"] = (ints(0, V, R), parents, cu)
    x = 3 * torch.randn(R, V, generator=g)
    x[0, 0], x[-1, V // 2], x[R // 2, -1] = 0.0, -math.inf, math.nan
    dev = {n: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for n, v in kw.items()}
    return x.to(dtype), kw, dev


def same_logits(got, want, dtype, spread=40):
    # five roundings of fp32 of values below ``spread``, and of the result
    half = BF16 if dtype == torch.bfloat16 else F32
    torch.testing.assert_close(got.double().cpu(), want, rtol=half + 8 * F32, atol=8 * F32 * spread, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S, V, sizes, L, K", [(1, 1, None, 1, 1), (3, 31, None, 5, 40), (4, 4096, None, 300, 64), (3, 4097, [3, 0, 9], 1000, 7),
                                               (2, 9001, [1, 128], 77, 1), (5, 12345, None, 4099, 700)])  # fmt: skip
def test_logits(dtype, S, V, sizes, L, K):
    from slime_b200 import ops

    x, kw, dev = logits_case(S, V, sizes, L=L, K=K, dtype=dtype)
    want, _ = oracle.adjusted(x, **kw)
    y = x.cuda()
    same_logits(ops.adjust_logits(y, **dev), want, dtype, spread=40 + K)
    assert torch.equal(y.nan_to_num(9.0).cpu(), x.nan_to_num(9.0))
    assert ops.adjust_logits(y, **dev, out=y) is y  # in place
    same_logits(y, want, dtype, spread=40 + K)


@pytest.mark.parametrize("parts", [(), ("repetition",), ("frequency",), ("presence",), ("bias",), ("allowed",)])
def test_logits_parts_alone(parts):
    from slime_b200 import ops

    x, kw, dev = logits_case(6, 5003, parts=parts)
    want, _ = oracle.adjusted(x, **kw)
    same_logits(ops.adjust_logits(x.cuda(), **dev), want, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_strided_rows_and_rows_behind_the_last_tree(dtype):
    from slime_b200 import ops

    x, kw, dev = logits_case(3, 5003, [2, 3, 1], dtype=dtype)
    drafted, parents, cu = dev["tree"]
    pad = lambda t: torch.cat([t, t[:2]])  # noqa: E731
    dev["tree"], dev["allowed"] = (pad(drafted), pad(parents), cu), pad(dev["allowed"])
    want, _ = oracle.adjusted(x, **kw)
    for left, right in ((1, 4), (0, 5), (3, 8)):  # rows that start and end off every boundary
        wide = torch.full((8, left + 5003 + right), 7.0, dtype=dtype, device="cuda")
        wide[:, left : left + 5003] = pad(x.cuda())
        out = torch.full((8, 5003 + 2 * left), 5.0, dtype=dtype, device="cuda")[:, left : left + 5003]
        ops.adjust_logits(wide[:, left : left + 5003], **dev, out=out)
        same_logits(out[:6], want, dtype)
        assert (out[6:] == 5).all()
        ops.adjust_logits(wide[:, left : left + 5003], **dev, out=wide[:, left : left + 5003])
        same_logits(wide[:6, left : left + 5003], want, dtype)
        assert (wide[:, :left] == 7).all() and (wide[:, left + 5003 :] == 7).all()


def test_logits_of_a_whole_vocabulary_in_a_graph():
    from slime_b200 import ops

    V, S = 151936, 3
    x, kw, dev = logits_case(S, V, L=2000, parts=("repetition", "frequency", "presence", "bias"))
    y = x.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adjust_logits(y, **dev)
    dev["tokens"].add_(11)
    kw["tokens"] += 11
    graph.replay()
    want, _ = oracle.adjusted(x, **kw)
    same_logits(out, want, torch.float32)
    assert ops.adjust_logits(y[:0], allowed=torch.zeros(0, -(-V // 32), dtype=torch.int32, device="cuda")).shape == (0, V)


# (rows times pieces of 2048 logits are more than the GPU holds at once: texts are counted by a kernel of their own)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S, V, sizes, L, K", [(600, 4200, None, 70, 3), (40, 4099, [13, 0, 30, 75] * 10, 200, 5), (7, 6145, [128, 0, 90, 128, 1, 128, 128], 500, 300)])
def test_logits_of_many_rows(dtype, S, V, sizes, L, K):
    from slime_b200 import ops

    x, kw, dev = logits_case(S, V, sizes, L=L, K=K, dtype=dtype)
    want, _ = oracle.adjusted(x, **kw)
    y = x.cuda()
    a = ops.adjust_logits(y, **dev)
    same_logits(a, want, dtype, spread=40 + K)
    assert torch.equal(a.nan_to_num(9.0), ops.adjust_logits(y, **dev).nan_to_num(9.0))
    assert torch.equal(y.nan_to_num(9.0).cpu(), x.nan_to_num(9.0))
    assert ops.adjust_logits(y, **dev, out=y) is y
    assert torch.equal(a.nan_to_num(9.0), y.nan_to_num(9.0))


@pytest.mark.parametrize("parts", [(), ("repetition",), ("frequency",), ("presence",), ("bias",), ("allowed",), ("repetition", "allowed")])
@pytest.mark.parametrize("sizes", [None, [2, 0, 100, 57] * 4])
def test_logits_parts_alone_of_many_rows(parts, sizes):
    from slime_b200 import ops

    x, kw, dev = logits_case(640 if sizes is None else len(sizes), 4101, sizes, parts=parts)
    want, _ = oracle.adjusted(x, **kw)
    same_logits(ops.adjust_logits(x.cuda(), **dev), want, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [6143, 6145, 12289, 40000])
def test_logits_of_long_texts(dtype, L):
    """Texts of every length up to L, tokens from the whole vocabulary and from a few; the same token all along; no text; a bias at either end, one of them twice."""
    from slime_b200 import ops

    S, V, sizes = 6, 20011, [40, 1, 0, 50, 24, 10]
    x, kw, dev = logits_case(S, V, sizes, L=L, K=9, dtype=dtype)
    g = torch.Generator().manual_seed(L)
    kw["tokens"] = torch.randint(-1, V + 1, (S, L), generator=g, dtype=torch.int32)
    kw["tokens"][1] %= 64
    kw["tokens"][3] = 77
    kw["tokens"][4, 1:] = V - 1
    kw["lengths"] = torch.tensor([L, L - 1, 5, L, L // 2, 0], dtype=torch.int32)
    kw["prompt_lens"] = torch.tensor([L // 3, 0, 5, L - 2, L, 0], dtype=torch.int32)
    kw["bias_ids"][0, :3] = torch.tensor([V - 1, 0, V - 1])
    dev = {n: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for n, v in kw.items()}
    want, _ = oracle.adjusted(x, **kw)
    # (a frequency below one times up to L answers: one rounding of the product, one of the difference)
    same_logits(ops.adjust_logits(x.cuda(), **dev), want, dtype, spread=40 + L)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_many_strided_rows_in_a_graph(dtype):
    from slime_b200 import ops

    sizes, V = [60, 128, 0, 128, 3, 100, 128], 4097
    x, kw, dev = logits_case(7, V, sizes, dtype=dtype, L=90)
    R = sum(sizes)
    drafted, parents, cu = dev["tree"]
    pad = lambda t: torch.cat([t, t[:2]])  # noqa: E731
    dev["tree"], dev["allowed"] = (pad(drafted), pad(parents), cu), pad(dev["allowed"])
    for left, right in ((1, 4), (0, 5), (3, 8)):
        wide = torch.full((R + 2, left + V + right), 7.0, dtype=dtype, device="cuda")
        wide[:, left : left + V] = pad(x.cuda())
        out = torch.full((R + 2, V + 2 * left), 5.0, dtype=dtype, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.adjust_logits(wide[:, left : left + V], **dev, out=out[:, left : left + V])
            ops.adjust_logits(wide[:, left : left + V], **dev, out=wide[:, left : left + V])
        # the graph reads texts, lengths and trees as they are when it runs
        cu_then = cu.clone()
        for step in (0, 1):
            if step:
                wide[:, left : left + V] = pad(x.cuda())
                out.fill_(5.0)
                dev["tokens"].add_(3)
                dev["lengths"].clamp_(max=60)
            now = {**kw, "tokens": dev["tokens"].cpu(), "lengths": dev["lengths"].cpu()}
            graph.replay()
            want, _ = oracle.adjusted(x, **now)
            for t in (out, wide):
                same_logits(t[:R, left : left + V], want, dtype)
            assert (out[R:] == 5).all() and (out[:, :left] == 5).all() and (out[:, left + V :] == 5).all()
            assert (wide[:, :left] == 7).all() and (wide[:, left + V :] == 7).all()
        assert torch.equal(cu, cu_then)


def test_captured_logits_share_a_workspace():
    """Two captured calls of other sizes, one replayed after the other, in memory that is full of something else; neither allocates any of its own. A smaller one is refused."""
    from slime_b200 import ops

    cases = [logits_case(R, V, L=L, K=K, parts=("repetition", "frequency", "presence", "bias")) for R, V, L, K in ((600, 4200, 70, 3), (130, 20011, 7000, 9))]
    sizes = [ops.adjust_logits_workspace(*x.shape, "cuda", text=kw["tokens"].shape[1], biases=kw["bias_ids"].shape[1]) for x, kw, _ in cases]
    assert min(sizes) > 0
    work = torch.full((max(sizes),), 0x7F, dtype=torch.uint8, device="cuda")
    held = []
    for x, _, dev in cases:
        y, out = x.cuda(), torch.empty(x.shape, device="cuda")
        ops.adjust_logits(y, **dev, out=out, workspace=work)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.max_memory_allocated()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.adjust_logits(y, **dev, out=out, workspace=work)
        assert torch.cuda.max_memory_allocated() - before < min(sizes)
        held.append((graph, out, y))
    want = [oracle.adjusted(x, **kw)[0] for x, kw, _ in cases]
    for i in (0, 1, 1, 0):
        held[i][1].fill_(5.0)
        work.fill_(0x55)
        held[i][0].replay()
        same_logits(held[i][1], want[i], torch.float32, spread=7040)
    with pytest.raises(ValueError, match="workspace"):
        ops.adjust_logits(held[0][2], **cases[0][2], workspace=work[: sizes[0] - 16])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [2, 125])  # one launch, two
@pytest.mark.parametrize("K", [37, 2999, 20011])
@pytest.mark.parametrize("what", ["distinct", "one twice", "all twice", "all the same", "last place"])
def test_logits_of_long_lists_of_biases(dtype, R, K, what):
    """Whole numbers as biases, so that sums of them are exact; beside penalties of a text that shares tokens with the list."""
    from slime_b200 import ops

    V = 20011
    x, kw, _ = logits_case(R, V, L=50, K=K, dtype=dtype, parts=("repetition", "frequency", "bias"))
    g = torch.Generator().manual_seed(K)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]).int()
    if what == "one twice":
        ids[:, K // 2] = ids[:, 1]
    elif what == "all twice":
        ids[:, K // 2 :] = ids[:, : K - K // 2].flip(1)
    elif what == "all the same":
        ids[:] = V - 1
    elif what == "last place":
        ids[:, -1] = ids[:, 0]
    kw["bias_ids"], kw["bias_values"] = ids, torch.randint(-8, 9, (R, K), generator=g).float()
    kw["tokens"][:, ::2] = ids[:, : 1].expand(-1, 25)
    dev = {n: v.cuda() for n, v in kw.items()}
    y = x.cuda()
    want, _ = oracle.adjusted(x, **kw)
    got = ops.adjust_logits(y, **dev)
    same_logits(got, want, dtype, spread=90 + float(kw["bias_values"].sum(1).abs().max()))
    for _ in range(2):
        assert torch.equal(got.nan_to_num(9.0), ops.adjust_logits(y, **dev).nan_to_num(9.0))


def test_a_token_listed_twice_does_not_cost_every_entry_a_look_at_the_list():
    from slime_b200 import ops

    x = torch.randn(64, 151936, device="cuda")
    ids = (7 * torch.arange(12000, dtype=torch.int32, device="cuda")).repeat(64, 1)
    twice, values = ids.clone(), torch.ones(64, 12000, device="cuda")
    twice[:, 5000] = twice[:, 3]

    def best(i):
        ends = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)) for _ in range(8)]
        for a, b in ends:
            a.record()
            ops.adjust_logits(x, bias_ids=i, bias_values=values, out=x)
            b.record()
        torch.cuda.synchronize()
        return min(a.elapsed_time(b) for a, b in ends)

    assert best(twice) < 5 * best(ids)  # (once 100 times as much)


# ------------------------------------------------------------------------------------------------------------- accept
def accept_case(sizes, seed=0, share=0.8, holes=0.0):
    g = torch.Generator().manual_seed(seed)
    cu, parents = oracle.make_trees(sizes, seed, holes)
    T = int(cu[-1])
    drafted = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32)
    sampled = torch.randint(100, 200, (T,), generator=g, dtype=torch.int32)
    for b in range(len(sizes)):
        for i in range(1, sizes[b]):
            up = int(parents[cu[b] + i])
            if 0 <= up < i and torch.rand((), generator=g) < share:
                sampled[cu[b] + up] = drafted[cu[b] + i]
    return sampled, drafted, parents, cu


@pytest.mark.parametrize("sizes", [[1], [8], [0, 5, 1, 0], [31, 32, 33], [128, 2], [3, 7] * 100])
@pytest.mark.parametrize("shape", [(2, 1, 4), (3, 8, 128), (1, 3, 5), (2, 1, 3)])
def test_acceptance(sizes, shape):
    from slime_b200 import ops

    layers, H, D = shape
    for seed, share, holes in ((0, 1.0, 0.0), (1, 0.7, 0.2)):
        ctx = [(7 * b + seed) % 40 for b in range(len(sizes))]
        sampled, drafted, parents, cu = accept_case(sizes, seed, share, holes)
        table, slots = oracle.make_pages([c + n for c, n in zip(ctx, sizes)], 16, seed)
        caches = [torch.randn(layers, slots, H, D).bfloat16(), torch.randn(layers, slots, H, 2 * D).bfloat16()]
        want = oracle.accepted(sampled, drafted, parents, cu, max(sizes))
        after = oracle.moved(caches, table, ctx, [w[0] for w in want], [w[2] for w in want], 16)
        dev = cuda(sampled, drafted, parents, cu)
        at = dict(block_table=table.cuda(), context_lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"), page_size=16)
        for split in (False, True):
            k, v = cuda(*caches)
            path, tokens, count = ops.accept_tree(*dev, max(sizes), k_caches=list(k) if split else k, v_caches=list(v) if split else v, **at)
            assert path.tolist() == [w[0] for w in want] and tokens.tolist() == [w[1] for w in want] and count.tolist() == [w[2] for w in want]
            assert torch.equal(k.cpu(), after[0]) and torch.equal(v.cpu(), after[1])
        alone = ops.accept_tree(*dev, max(sizes))
        assert all(torch.equal(a, b) for a, b in zip(alone, (path, tokens, count)))


def test_acceptance_of_many_layers_in_a_list_and_empty_values():
    from slime_b200 import ops

    sampled, drafted, parents, cu = accept_case([9, 12], 3, 1.0)
    ctx = [15, 2]
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, [9, 12])], 16, 0)
    caches = [torch.randn(150, slots, 2, 8)]
    want = oracle.accepted(sampled, drafted, parents, cu, 12)
    after = oracle.moved(caches, table, ctx, [w[0] for w in want], [w[2] for w in want], 16)
    k = caches[0].cuda()
    ops.accept_tree(*cuda(sampled, drafted, parents, cu), 12, k_caches=list(k), v_caches=[torch.empty(slots, 1, 0, device="cuda")] * 150,
                    block_table=table.cuda(), context_lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"), page_size=16)  # fmt: skip
    assert torch.equal(k.cpu(), after[0])
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    path, tokens, count = ops.accept_tree(none, none, none, torch.zeros(1, dtype=torch.int32, device="cuda"), 4)
    assert path.shape == (0, 4) and count.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float8_e4m3fn])
@pytest.mark.parametrize("H, D, left", [(1, 1, 0), (1, 3, 0), (2, 4, 0), (3, 16, 0), (1, 6, 1), (3, 5, 2), (1, 16, 4)])
def test_acceptance_of_one_byte_caches(dtype, H, D, left):
    """Rows of odd and even numbers of bytes, from odd and even addresses (``left`` bytes into a wider row): only the rows of the path change, and nothing
    between or behind them."""
    from slime_b200 import ops

    sizes, ctx = [9, 1, 40], [15, 3, 2]
    sampled, drafted, parents, cu = accept_case(sizes, 4, 1.0)
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, sizes)], 16, 1)
    want = oracle.accepted(sampled, drafted, parents, cu, 40)
    g = torch.Generator().manual_seed(D)
    for wide in (H * D + left, H * D + left + 3):  # a row's pitch
        store = torch.randint(0, 120, (2, 3, slots, wide), generator=g, dtype=torch.uint8)
        view = lambda t: t[..., left : left + H * D].unflatten(-1, (H, D))  # noqa: E731
        after = store.clone()
        for s in range(2):
            moved = oracle.moved([view(store[s]).contiguous()], table, ctx, [w[0] for w in want], [w[2] for w in want], 16)[0]
            view(after[s]).copy_(moved)
        for split in (False, True):
            dev = store.cuda()
            k, v = (view(dev[s]).view(dtype) for s in range(2))
            ops.accept_tree(*cuda(sampled, drafted, parents, cu), 40, k_caches=list(k) if split else k, v_caches=list(v) if split else v,
                            block_table=table.cuda(), context_lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"), page_size=16)  # fmt: skip
            assert torch.equal(dev.cpu(), after)


@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 8)])
@pytest.mark.parametrize("copies", [1, 300])  # logits in one launch, in two
def test_a_tree_that_begins_in_front_of_the_rows_is_none(heads, copies):
    """A first number below zero: nothing in front of the packed rows is read, and the other trees are what they are. (Checks of indices refuse such a call.)"""
    from slime_b200 import ops

    sizes, ctx = [2] + [4, 1] * copies, [9] + [5, 30] * copies
    q, k, v, table, c, cu, parents = attention_case(sizes, ctx, heads, 16, seed=2)
    bad = cu.clone()
    bad[0] = -3
    want = ops.tree_attention(q, k, v, table, c, cu, parents, 16, 4)
    got = ops.tree_attention(q, k, v, table, c, bad, parents, 16, 4, out=torch.full_like(q, 7.0))
    assert torch.equal(got[2:], want[2:]) and (got[:2] == 7).all()
    x, _, dev = logits_case(len(sizes), 4100, sizes, L=40)
    drafted = dev["tree"][0]
    want = ops.adjust_logits(x.cuda(), **{**dev, "tree": (drafted, parents, cu)})
    got = ops.adjust_logits(x.cuda(), **{**dev, "tree": (drafted, parents, bad)})
    assert torch.equal(got[2:].nan_to_num(9.0), want[2:].nan_to_num(9.0))
    sampled = drafted.roll(-1)
    want = ops.accept_tree(sampled, drafted, parents, cu, 4)
    got = ops.accept_tree(sampled, drafted, parents, bad, 4)
    assert all(torch.equal(a[1:], b[1:]) for a, b in zip(got, want)) and int(got[2][0]) == 0


# ------------------------------------------------------------------------------------------------------- a whole round
def test_a_round_of_drafted_trees_is_ordinary_decoding():
    """One attention layer with a vocabulary behind it, in fp32 (close calls of the sampler aside, both forms then draw the same tokens): two rounds of trees, penalties included,
    give the tokens that single steps give, and leave the cache that they leave."""
    from slime_b200 import ops

    g = torch.Generator().manual_seed(5)
    V, Hq, Hkv, D, page, B = 97, 4, 2, 16, 16, 3
    wq, wk, wv = (torch.randn(V, h * D, generator=g).cuda() for h in (Hq, Hkv, Hkv))
    head = torch.randn(Hq * D, V, generator=g).cuda() * 0.4
    ctx0 = [21, 3, 40]
    texts = [torch.randint(0, V, (c + 1,), generator=g).tolist() for c in ctx0]
    pens = dict(repetition=torch.tensor([1.3, 1.0, 0.8]).cuda(), frequency=torch.tensor([0.2, 0.0, 0.1]).cuda(), presence=torch.tensor([0.1, 0.0, 0.3]).cuda())
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, slots = oracle.make_pages([c + 64 for c in ctx0], page, 0)
    dev_table = table.cuda()
    prompts, seeds, temp = i32([c + 1 for c in ctx0]), torch.tensor([11, 12, 13], device="cuda"), torch.ones(B, device="cuda")

    def fresh_cache():
        k, v = torch.zeros(1, slots, Hkv, D, device="cuda"), torch.zeros(1, slots, Hkv, D, device="cuda")
        for b in range(B):
            at = torch.tensor([oracle.slot(table, b, p, page) for p in range(ctx0[b])], device="cuda")
            ids = torch.tensor(texts[b][:-1], device="cuda")
            k[0, at], v[0, at] = wk[ids].view(-1, Hkv, D), wv[ids].view(-1, Hkv, D)
        return k, v

    def step(k, v, text, ctx, sizes, parents, drafted):
        """Feed the nodes, adjust and sample every row."""
        cu = i32([0] + torch.tensor(sizes).cumsum(0).tolist())
        ids, par, where = torch.tensor(drafted, device="cuda"), i32(parents), i32(ctx)
        at = torch.tensor([oracle.slot(table, b, ctx[b] + i, page) for b in range(B) for i in range(sizes[b])], device="cuda")
        k[0, at], v[0, at] = wk[ids].view(-1, Hkv, D), wv[ids].view(-1, Hkv, D)
        o = ops.tree_attention(wq[ids].view(-1, Hq, D), k[0], v[0], dev_table, where, cu, par, page, max(sizes))
        tokens = torch.zeros(B, 128, dtype=torch.int32)
        for b in range(B):
            tokens[b, : len(text[b])] = torch.tensor(text[b])
        tree = (ids.int(), par, cu)
        logits = ops.adjust_logits(o.view(-1, Hq * D) @ head, tokens.cuda(), i32([len(t) for t in text]), prompts, tree=tree, **pens)
        # a node's place in the answer: behind the text, plus its depth
        depth = [len(oracle.way_up(parents[int(cu[b]) : int(cu[b + 1])], i)) - 1 for b in range(B) for i in range(sizes[b])]
        owner = [b for b in range(B) for _ in range(sizes[b])]
        pos = i32([len(text[b]) - ctx0[b] - 1 + d for b, d in zip(owner, depth)])
        rows = torch.tensor(owner, device="cuda")
        tok = ops.sample(logits, temp[rows], seeds=seeds[rows], positions=pos)[0]
        return tok, tree, where

    # ordinary decoding: trees of one node
    k1, v1 = fresh_cache()
    plain = [list(t) for t in texts]
    for n in range(14):
        tok, _, _ = step(k1, v1, plain, [c + n for c in ctx0], [1] * B, [-1] * B, [t[-1] for t in plain])
        for b, x in enumerate(tok.tolist()):
            plain[b].append(x)
    # two rounds: trees whose branches hold some right guesses and some wrong ones
    k2, v2 = fresh_cache()
    text, ctx = [list(t) for t in texts], list(ctx0)
    moved = 0
    for rnd in range(2):
        sizes, parents, drafted = [6, 9, 4], [], []
        for b in range(B):
            good = plain[b][len(text[b]) :]
            par = [-1, 0, 0, 2, 3, 1, 4, 2, 6][: sizes[b]] if rnd == 0 else [-1, 0, 1, 1, 3, 2, 4, 0, 6][: sizes[b]]
            right = [0, 2, 3, 4, 6, 8] if rnd == 0 else [0, 1, 3, 4, 6, 8]
            ids = [text[b][-1]] + [(good[0] + 17 + i) % V for i in range(1, sizes[b])]
            for d, i in enumerate(right[1:]):
                if i < sizes[b]:
                    ids[i] = good[d]
            parents += par
            drafted += ids
        tok, tree, where = step(k2, v2, text, ctx, sizes, parents, drafted)
        path, new, count = ops.accept_tree(tok, tree[0], tree[1], tree[2], 9, k_caches=k2, v_caches=v2, block_table=dev_table, context_lens=where,
                                           page_size=page)  # fmt: skip
        for b in range(B):
            n = int(count[b])
            assert n >= 2
            text[b] += new[b, :n].tolist()
            ctx[b] += n
            moved += sum(int(path[b, j]) != j for j in range(n))
            assert text[b] == plain[b][: len(text[b])]
    assert moved > 0
    for b in range(B):
        at = torch.tensor([oracle.slot(table, b, p, page) for p in range(ctx[b])], device="cuda")
        assert torch.equal(k2[0, at], k1[0, at]) and torch.equal(v2[0, at], v1[0, at])


# ------------------------------------------------------------------------------------------------------- in the engine
def test_captured_decode_steps_adjust_their_logits():
    """Requests with penalties and biases beside one without: eager and replayed steps draw the same tokens, a later request in a
    used slot is what it is alone, and biases of more tokens than any request had before are taken up."""
    from slime_b200.engine.engine import Engine
    from slime_b200.engine.server_args import ServerArgs
    from slime_b200.models.config import get_preset

    prompts = [[(5 * i + 3 * j) % 500 for j in range(6 + i)] for i in range(4)]
    many = {t: -1e9 for t in range(100, 500)}
    asks = [dict(repetition_penalty=1.3), dict(frequency_penalty=0.4, presence_penalty=0.2), dict(), dict(logit_bias={7: 3.0, 9: -100.0}, repetition_penalty=0.9)]
    got = []
    for graphs in (False, True):
        e = Engine(get_preset("tiny"), ServerArgs(page_size=16, max_running_requests=4, context_length=128, disable_cuda_graph=not graphs),
                   device="cuda", num_pages=64)  # fmt: skip
        e.weights.init_random(0, std=0.2)
        base = dict(max_new_tokens=20, temperature=0, ignore_eos=True)
        first = e.generate(prompts, [dict(base, **a) for a in asks])
        assert bool(e.runner.graphs) == graphs
        plain = e.generate(prompts, dict(base))
        assert first[2].output_ids == plain[2].output_ids and 9 not in first[3].output_ids
        again = e.generate(prompts, [dict(base, logit_bias=many if i == 1 else None, presence_penalty=1e4 if i == 0 else 0) for i in range(4)])
        assert len(set(again[0].output_ids)) == 20 and not set(again[1].output_ids) & set(many)
        assert [r.output_ids for r in again[2:]] == [r.output_ids for r in plain[2:]]
        got.append([[r.output_ids for r in x] + [r.output_logprobs for r in x] for x in (first, plain, again)])
        e.shutdown()
    assert got[0] == got[1]


@pytest.mark.parametrize("graphs", [False, True])
def test_steps_of_many_requests_with_a_wide_context_adjust_their_logits(graphs):
    """A context as wide as the engine's default, and more requests than the operator takes in one launch (a row of 512 tokens is one CTA's, 8 for each SM): a presence penalty lets no
    token come twice, a negative frequency penalty no other than the first, biases none but a few, whatever was asked beside it; a request has a text of 9000 tokens."""
    from slime_b200 import ops
    from slime_b200.engine.engine import Engine
    from slime_b200.engine.server_args import ServerArgs
    from slime_b200.models.config import get_preset

    n = 8 * torch.cuda.get_device_properties(0).multi_processor_count + 16
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (3 + i % 5,), generator=g).tolist() for i in range(n)]
    prompts[8] = torch.randint(0, 500, (9000,), generator=g).tolist()
    few = {t: -1e9 for t in range(512) if t % 50 != 7}
    asks = [dict(presence_penalty=1e6), dict(frequency_penalty=-1e6), dict(), dict(logit_bias=few)]
    e = Engine(get_preset("tiny"), ServerArgs(page_size=16, max_running_requests=n, context_length=32768, disable_cuda_graph=not graphs),
               device="cuda", num_pages=2 * n + 700)  # fmt: skip
    e.weights.init_random(0, std=0.2)
    reqs = e.generate(prompts, [dict(max_new_tokens=12 if i < n - 400 else 5, temperature=0, ignore_eos=True, **asks[i % 4]) for i in range(n)])
    a = e.runner.adjustments
    assert a.work.numel() == ops.adjust_logits_workspace(n, 512, "cuda", text=32769, biases=512) > 0
    assert a.work.numel() <= n * (512 * 12 + 16) + 64  # (not by the width of the context)
    for i, r in enumerate(reqs):
        out = r.output_ids
        assert len(out) == (12 if i < n - 400 else 5)
        if i % 4 == 0:
            assert len(set(out)) == len(out)
        elif i % 4 == 1:
            assert set(out) == {out[0]}
        elif i % 4 == 3:
            assert all(t % 50 == 7 for t in out)
    e.shutdown()


@pytest.mark.parametrize("vocab, requests", [(512, 3), (20011, 40)])  # one launch, two
def test_chains_of_guesses_are_adjusted_in_place(vocab, requests):
    """The form that a speculating engine calls: rows for the last token of a text and the guesses behind it, in place, among requests that ask for nothing and rows that belong to none."""
    from slime_b200.engine import penalties
    from slime_b200.engine.request import Request, SamplingParams

    g = torch.Generator().manual_seed(vocab)
    ints = lambda n, hi=vocab: torch.randint(0, hi, (n,), generator=g).tolist()  # noqa: E731
    asks = [dict(repetition_penalty=1.3, frequency_penalty=0.4), dict(), dict(presence_penalty=0.7, logit_bias={3: 2.0, 9: -1.5, 10**6: 4.0}),
            dict(frequency_penalty=-0.2, presence_penalty=0.1, repetition_penalty=0.8)]  # fmt: skip
    reqs, ids, sizes = [], [], []
    for i in range(requests):
        r = Request(rid=str(i), input_ids=ints(4 + 31 * i, 60), sampling=SamplingParams(**asks[i % 4]))
        r.output_ids = ints(1 + 7 * i, 60)
        reqs.append(r)
        sizes.append(1 + i % 5)
        ids += [r.output_ids[-1]] + ints(sizes[-1] - 1, 60)
    spare = 2
    cu = torch.tensor([0] + sizes).cumsum(0).int()
    ids += [5] * spare
    x = 3 * torch.randn(len(ids), vocab, generator=g)
    logits = x.cuda()
    assert penalties.adjust(logits, reqs, (torch.tensor(ids, dtype=torch.int32, device="cuda"), cu.cuda())) is logits
    got = logits.cpu().double()
    for i, r in enumerate(reqs):
        s, a = r.sampling, int(cu[i])
        for d in range(sizes[i]):
            text, n = r.all_ids() + ids[a + 1 : a + 1 + d], len(r.input_ids)
            f = lambda v: torch.tensor([v])  # noqa: E731
            bias = {t: v for t, v in (s.logit_bias or {}).items()}
            want, _ = oracle.adjusted(x[a + d : a + d + 1], torch.tensor([text]), torch.tensor([len(text)]), torch.tensor([n]), f(s.repetition_penalty),
                                      f(s.frequency_penalty), f(s.presence_penalty), torch.tensor([list(bias)]) if bias else None,
                                      torch.tensor([list(bias.values())]) if bias else None)  # fmt: skip
            # five roundings of fp32 of values below 40 + 0.4 times the text's length, and penalties that are themselves rounded
            torch.testing.assert_close(got[a + d : a + d + 1], want, rtol=9 * F32, atol=10 * F32 * (40 + len(text)))
            if not s.adjusts:
                assert torch.equal(logits[a + d].cpu(), x[a + d])
    assert torch.equal(logits[-spare:].cpu(), x[-spare:])


def test_speculating_requests_keep_their_penalties():
    from slime_b200.engine.engine import Engine
    from slime_b200.engine.server_args import ServerArgs
    from slime_b200.models.config import ModelConfig

    cfg = ModelConfig(num_layers=2, hidden_size=128, num_attention_heads=4, num_query_groups=2, kv_channels=64, ffn_hidden_size=256, vocab_size=512, rotary_base=1e4,
                      tie_word_embeddings=False, mtp_num_layers=1, qk_layernorm=True, model_arch="Qwen3ForCausalLM")  # fmt: skip
    e = Engine(cfg, ServerArgs(page_size=16, max_running_requests=8, context_length=512, speculative_algorithm="EAGLE", speculative_num_steps=3,
                               speculative_num_draft_tokens=4), device="cuda", num_pages=400)  # fmt: skip
    e.weights.init_random(0, std=0.2)
    few = {t: -1e9 for t in range(512) if t % 50 != 7}
    asks = [dict(presence_penalty=1e6), dict(frequency_penalty=-1e6), dict(), dict(logit_bias=few)]
    prompts = [[(5 * i + 3 * j) % 500 for j in range(6 + i)] for i in range(8)]
    for temperature in (0, 1.0):
        reqs = e.generate(prompts, [dict(max_new_tokens=30, temperature=temperature, ignore_eos=True, **asks[i % 4]) for i in range(8)])
        for i, r in enumerate(reqs):
            assert len(r.output_ids) == 30
            if i % 4 == 0:
                assert len(set(r.output_ids)) == 30
            elif i % 4 == 1:
                assert len(set(r.output_ids)) == 1
            elif i % 4 == 3:
                assert all(t % 50 == 7 for t in r.output_ids)
    e.shutdown()


@pytest.mark.parametrize("speculate", [False, True])
def test_the_largest_penalties_leave_a_distribution_on_the_gpu(speculate):
    from slime_b200.engine.engine import Engine
    from slime_b200.engine.server_args import ServerArgs
    from slime_b200.models.config import ModelConfig

    cfg = ModelConfig(num_layers=2, hidden_size=128, num_attention_heads=4, num_query_groups=2, kv_channels=64, ffn_hidden_size=256, vocab_size=512, rotary_base=1e4,
                      tie_word_embeddings=False, mtp_num_layers=1, qk_layernorm=True, model_arch="Qwen3ForCausalLM")  # fmt: skip
    kw = dict(speculative_algorithm="EAGLE", speculative_num_steps=3, speculative_num_draft_tokens=4) if speculate else {}
    e = Engine(cfg, ServerArgs(page_size=16, max_running_requests=8, context_length=512, **kw), device="cuda", num_pages=400)
    e.weights.init_random(0, std=0.2)
    inf = math.inf
    asks = [dict(frequency_penalty=s * 1e9, presence_penalty=s * 1e9, repetition_penalty=r, logit_bias={5: s * 1e9, 6: -s * 1e9, 7: -inf})
            for s in (-1, 1) for r in (1e-9, 1e9)] + [dict(logit_bias={t: -inf for t in range(520) if t != 9}), {}]  # fmt: skip
    for sampling in (dict(temperature=0), dict(temperature=1.0), dict(temperature=0.01), dict(temperature=1.0, top_p=0.9, top_k=20)):
        reqs = e.generate([[1, 2, 3]] * len(asks), [dict(max_new_tokens=8, ignore_eos=True, **sampling, **a) for a in asks])
        for r, a in zip(reqs, asks):
            assert len(r.output_ids) == 8 and all(0 <= t < 512 for t in r.output_ids) and all(math.isfinite(x) for x in r.output_logprobs), (sampling, a, r.output_ids)
        assert reqs[4].output_ids == [9] * 8 and not any(7 in r.output_ids for r in reqs[:4])
    e.shutdown()
