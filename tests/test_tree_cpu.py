"""Operators of drafted-token trees and of logits before sampling on the CPU: definitions against 64-bit loops, and refusals."""

import math

import pytest
import torch
import tree_oracle as oracle

from slime_b200 import ops
from slime_b200.ops import _checks

F32 = 2.0**-24


def attention_case(sizes, ctx, heads=(4, 2, 8), page=4, seed=0, holes=0.0, shape="random", dtype=torch.float32):
    Hq, Hkv, D = heads
    g = torch.Generator().manual_seed(seed)
    cu, parents = oracle.make_trees(sizes, seed, holes, shape)
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, sizes)], page, seed)
    k, v = (torch.full((slots, Hkv, D), math.nan) for _ in range(2))
    for b, (c, n) in enumerate(zip(ctx, sizes)):
        for p in range(c + n):
            s = oracle.slot(table, b, p, page)
            k[s], v[s] = torch.randn(Hkv, D, generator=g), torch.randn(Hkv, D, generator=g)
    q = 2 * torch.randn(int(cu[-1]), Hq, D, generator=g)
    return q.to(dtype), k.to(dtype), v.to(dtype), table, torch.tensor(ctx, dtype=torch.int32), cu, parents


@pytest.mark.parametrize("sizes, ctx, kw", [
    ([1], [0], {}),
    ([1, 5, 3], [7, 0, 13], {}),
    ([6, 0, 4], [3, 9, 8], dict(shape="chain")),
    ([9, 33], [5, 16], dict(holes=0.2, seed=3)),
    ([40], [1], dict(shape="star", heads=(3, 3, 5), page=16)),
])  # fmt: skip
@pytest.mark.parametrize("sink", [False, True])
def test_attention_definition_is_the_formula(sizes, ctx, kw, sink):
    q, k, v, table, ctx, cu, parents = attention_case(sizes, ctx, **kw)
    page = kw.get("page", 4)
    sinks = torch.randn(q.shape[1], generator=torch.Generator().manual_seed(1)) if sink else None
    table = table.clamp(max=k.shape[0] // page - 1)
    got = ops.tree_attention(q, k, v, table, ctx, cu, parents, page, max(sizes), sinks=sinks)
    want, mass = oracle.attention(q, k, v, table, ctx, cu, parents, page, q.shape[2] ** -0.5, sinks)
    # products of D terms and sums over the keys: a few dozen roundings of fp32 each, on the scale of the values that are averaged
    assert ((got.double() - want).abs() <= 64 * F32 * (mass + 1)).all()


def test_a_chain_is_causal_attention():
    q, k, v, table, ctx, cu, parents = attention_case([7], [10], shape="chain")
    got = ops.tree_attention(q, k, v, table, ctx, cu, parents, 4, 7)
    for i in range(7):
        one = ops.paged_decode_attention(q[i : i + 1], k, v, table, torch.tensor([11 + i], dtype=torch.int32), 4)
        torch.testing.assert_close(got[i : i + 1], one, rtol=1e-5, atol=1e-5)


def test_attention_leaves_rows_behind_the_last_tree():
    q, k, v, table, ctx, cu, parents = attention_case([3, 2], [4, 4])
    q = torch.cat([q, q[:2]])
    out = torch.full_like(q, 7.0)
    pad = torch.cat([parents, torch.tensor([0, 0], dtype=torch.int32)])
    assert ops.tree_attention(q, k, v, table, ctx, cu, pad, 4, 3, out=out) is out
    assert (out[5:] == 7).all() and (out[:5] != 7).all()


@pytest.mark.parametrize("name, change, match", [
    ("nodes", dict(max_nodes=129), "129 nodes"),
    ("none", dict(max_nodes=0), "0 nodes"),
    ("parents", dict(parents=torch.zeros(4, dtype=torch.int32)), "parents"),
    ("long parents", dict(parents=torch.zeros(5, dtype=torch.int64)), "int32"),
    ("context", dict(context_lens=torch.zeros(3, dtype=torch.int32)), "context_lens"),
    ("table", dict(block_table=torch.zeros(1, 3, dtype=torch.int32)), "block_table"),
    ("width", dict(v_cache=torch.zeros(40, 2, 16)), "v_cache"),
    ("types", dict(k_cache=torch.zeros(40, 2, 8, dtype=torch.bfloat16)), "alike"),
    ("heads", dict(q=torch.zeros(5, 3, 8)), "3 query heads"),
    ("half", dict(q=torch.zeros(5, 4, 8, dtype=torch.float16)), "bf16 or fp32"),
    ("out", dict(out=torch.zeros(5, 4, 4)), "out"),
    ("sinks", dict(sinks=torch.zeros(3)), "sinks"),
    ("page", dict(page_size=0), "pages"),
])  # fmt: skip
def test_attention_refuses(name, change, match):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    args = dict(q=torch.zeros(5, 4, 8), k_cache=torch.zeros(40, 2, 8), v_cache=torch.zeros(40, 2, 8), block_table=z(2, 3), context_lens=z(2),
                cu_nodes=torch.tensor([0, 3, 5], dtype=torch.int32), parents=z(5), page_size=4, max_nodes=3)  # fmt: skip
    with pytest.raises(ValueError, match=match):
        ops.tree_attention(**{**args, **change})


def test_bad_pages_and_sizes_are_named_before_the_launch(monkeypatch):
    monkeypatch.setenv("SLIME_B200_CHECKS", "1")
    q, k, v, table, ctx, cu, parents = attention_case([3, 2], [4, 4])
    bad = table.clone()
    bad[1, 0] = 99
    with pytest.raises(_checks.IndexCheckError, match="block_table"):
        ops.tree_attention(q, k, v, bad, ctx, cu, parents, 4, 3)
    with pytest.raises(_checks.IndexCheckError, match="seq_lens"):
        ops.tree_attention(q, k, v, table, ctx + 20, cu, parents, 4, 3)
    with pytest.raises(_checks.IndexCheckError, match="tree sizes"):
        ops.tree_attention(q, k, v, table, ctx, cu, parents, 4, 2)
    with pytest.raises(_checks.IndexCheckError, match="cu_nodes"):
        ops.tree_attention(q, k, v, table, ctx, cu + 1, parents, 4, 3)


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
        kw["allowed"][R // 2] = 0  # a row that may go nowhere
    if sizes is not None:
        cu, parents = oracle.make_trees(sizes, seed, holes=0.1)
        kw["tree"] = (ints(0, V, R), parents, cu)
    x = 3 * torch.randn(R, V, generator=g)
    x[0, 0], x[-1, V // 2], x[R // 2, -1] = 0.0, -math.inf, math.nan
    return x.to(dtype), kw


ALL = ("repetition", "frequency", "presence", "bias", "allowed")


@pytest.mark.parametrize("parts", [ALL, (), ("repetition",), ("frequency",), ("presence",), ("bias",), ("allowed",)])
@pytest.mark.parametrize("sizes", [None, [3, 0, 9, 1]])
def test_logits_definition_is_the_formula(parts, sizes):
    x, kw = logits_case(4, 77, sizes, parts=parts)
    got = ops.adjust_logits(x, **kw)
    want, _ = oracle.adjusted(x, **kw)
    # five roundings of fp32, each of a value no larger than the sum of what is added
    torch.testing.assert_close(got.double(), want, rtol=8 * F32, atol=8 * F32 * 40, equal_nan=True)


def test_logits_in_place_and_rows_behind_the_last_tree():
    x, kw = logits_case(3, 50, [2, 3, 1])
    drafted, parents, cu = kw["tree"]
    more = torch.cat([x, x[:2]])
    pad = lambda t: torch.cat([t, t[:2]])  # noqa: E731
    kw["allowed"] = pad(kw["allowed"])
    kw["tree"] = (pad(drafted), pad(parents), cu)
    before = more.clone()
    assert ops.adjust_logits(more, **kw, out=more) is more
    assert torch.equal(more[6:].nan_to_num(1e9), before[6:].nan_to_num(1e9)) and not torch.equal(more[:6], before[:6])


@pytest.mark.parametrize("change, match", [
    (dict(logits=torch.zeros(3, 40, dtype=torch.float16)), "bf16 or fp32"),
    (dict(logits=torch.zeros(120)), "rows, vocabulary"),
    (dict(tokens=None), "tokens of the requests"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int64)), "int32"),
    (dict(tokens=torch.zeros(2, 5, dtype=torch.int32)), "tokens"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths"),
    (dict(prompt_lens=torch.zeros(2, dtype=torch.int32)), "prompt_lens"),
    (dict(repetition=torch.ones(2)), "repetition"),
    (dict(frequency=torch.ones(3, dtype=torch.float64)), "frequency"),
    (dict(bias_ids=torch.zeros(3, 2, dtype=torch.int32)), "ids and values"),
    (dict(bias_ids=torch.zeros(3, 2, dtype=torch.int32), bias_values=torch.zeros(3, 3)), "bias_values"),
    (dict(allowed=torch.zeros(3, 1, dtype=torch.int32)), "allowed"),
    (dict(out=torch.zeros(3, 41)), "out"),
    (dict(tree=(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.tensor([0, 1, 2, 3], dtype=torch.int32))), "parents"),
])  # fmt: skip
def test_logits_refuse(change, match):
    args = dict(logits=torch.zeros(3, 40), tokens=torch.zeros(3, 5, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32), repetition=torch.ones(3))
    with pytest.raises(ValueError, match=match):
        ops.adjust_logits(**{**args, **change})


def accept_case(sizes, seed=0, share=0.8, holes=0.0):
    """Trees whose rows sample one of their children's tokens most of the time; some siblings share a token."""
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


@pytest.mark.parametrize("sizes", [[1], [8], [0, 5, 1, 0], [31, 32, 33], [128, 2]])
@pytest.mark.parametrize("holes", [0.0, 0.2])
def test_acceptance_follows_the_sampled_tokens(sizes, holes):
    for seed in range(4):
        sampled, drafted, parents, cu = accept_case(sizes, seed, holes=holes)
        path, tokens, count = ops.accept_tree(sampled, drafted, parents, cu, max(sizes))
        want = oracle.accepted(sampled, drafted, parents, cu, max(sizes))
        assert path.tolist() == [w[0] for w in want] and tokens.tolist() == [w[1] for w in want] and count.tolist() == [w[2] for w in want]


@pytest.mark.parametrize("stacked", [True, False])
def test_accepted_rows_move_behind_each_other(stacked):
    sizes, ctx = [9, 1, 33], [6, 3, 0]
    sampled, drafted, parents, cu = accept_case(sizes, 2, share=1.0)
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, sizes)], 4, 1)
    ctx = torch.tensor(ctx, dtype=torch.int32)
    caches = [torch.randn(3, slots, 2, 4), torch.randn(3, slots, 2, 6)]
    path, _, count = ops.accept_tree(sampled, drafted, parents, cu, 33)
    want = oracle.moved(caches, table, ctx, path, count, 4)
    assert any(not torch.equal(a, b) for a, b in zip(caches, want))
    k, v = (caches if stacked else [list(c) for c in caches])
    ops.accept_tree(sampled, drafted, parents, cu, 33, k_caches=k, v_caches=v, block_table=table, context_lens=ctx, page_size=4)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


LATENT = torch.zeros(2, 8, 1, 4)


@pytest.mark.parametrize("change, match", [
    (dict(max_nodes=200), "200 nodes"),
    (dict(drafted=torch.zeros(4, dtype=torch.int32)), "drafted"),
    (dict(sampled=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(k_caches=torch.zeros(1, 8, 2, 4)), "come with"),
    (dict(k_caches=torch.zeros(1, 8, 4, 2).transpose(2, 3), block_table=torch.zeros(1, 2, dtype=torch.int32),
          context_lens=torch.zeros(1, dtype=torch.int32), page_size=4), "one piece"),
    (dict(k_caches=torch.zeros(1, 8, 2, 4), block_table=torch.zeros(2, 2, dtype=torch.int32), context_lens=torch.zeros(1, dtype=torch.int32),
          page_size=4), "block_table"),
    (dict(k_caches=LATENT, v_caches=LATENT, block_table=torch.zeros(1, 2, dtype=torch.int32), context_lens=torch.zeros(1, dtype=torch.int32), page_size=4),
     "share memory"),
    (dict(k_caches=list(LATENT), v_caches=[x[..., :2] for x in LATENT], block_table=torch.zeros(1, 2, dtype=torch.int32),
          context_lens=torch.zeros(1, dtype=torch.int32), page_size=4), "share memory"),
])  # fmt: skip
def test_acceptance_refuses(change, match):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    args = dict(sampled=z(3), drafted=z(3), parents=z(3), cu_nodes=torch.tensor([0, 3], dtype=torch.int32), max_nodes=3)
    with pytest.raises(ValueError, match=match):
        ops.accept_tree(**{**args, **change})


def test_the_entry_of_acceptance_moves_rows_in_pieces_that_fit():
    """Pieces are 1, 2, 4, 8 or 16 bytes, and addresses and pitches are multiples of them; the entry refuses any other call before it launches anything."""
    from slime_b200.ops import _lib, tree

    if not _lib.available():
        pytest.skip("the kernel library is not built")
    fn, invalid = _lib.lib().sb_tree_accept, 1  # cudaErrorInvalidValue
    # (unit, bytes from slot to slot, bytes from slab to slab, address)
    for unit, pitch, step, base in ((3, 3, 0, 48), (0, 16, 0, 48), (-1, 16, 0, 48), (32, 32, 0, 64), (2, 3, 0, 48), (2, 4, 5, 48), (2, 4, 0, 49)):
        call = tree._ACCEPT(*[0] * 9, 4, 1, 4, 1, 1, 1, 148, 1, step, 8, 3, unit, pitch, 1) + base.to_bytes(8, "little")
        assert fn(call, None) == invalid


@pytest.mark.parametrize("width", [1, 3, 6])
def test_accepted_rows_of_one_byte_elements(width):
    sampled, drafted, parents, cu = accept_case([9, 4], 3)
    ctx = [5, 11]
    table, slots = oracle.make_pages([c + n for c, n in zip(ctx, [9, 4])], 4, 0)
    caches = [torch.randint(0, 256, (2, slots, 1, width), dtype=torch.uint8)]
    want = oracle.accepted(sampled, drafted, parents, cu, 9)
    after = oracle.moved(caches, table, ctx, [w[0] for w in want], [w[2] for w in want], 4)
    ops.accept_tree(sampled, drafted, parents, cu, 9, k_caches=caches[0], block_table=table, context_lens=torch.tensor(ctx, dtype=torch.int32), page_size=4)
    assert torch.equal(caches[0], after[0])


def test_workspace_of_adjusted_logits():
    x, ids = torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.int32)
    assert ops.adjust_logits_workspace(2, 5, "cpu", text=3) == 0
    kw = dict(tokens=ids, lengths=ids[:, 0].contiguous(), frequency=torch.zeros(2))
    assert torch.equal(ops.adjust_logits(x, **kw, workspace=torch.empty(0, dtype=torch.uint8)), x)
    for bad in (torch.empty(64), torch.empty(64, dtype=torch.uint8)[::2], torch.empty(64, dtype=torch.uint8)[1:]):
        with pytest.raises(ValueError, match="workspace"):
            ops.adjust_logits(x, **kw, workspace=bad)


@pytest.mark.parametrize("requests, lists", [(16, 8), (32, 8), (64, 4), (148, 2), (149, 1), (256, 1)])
@pytest.mark.parametrize("biases", [0, 300])
def test_workspace_is_no_larger_than_what_lists_of_distinct_tokens_can_hold(requests, lists, biases):
    """With several lists of a request each has every second, fourth or eighth token of the vocabulary at most, however long the text may be."""
    from slime_b200.ops import _lib, logits

    if not _lib.available():
        pytest.skip("the kernel library is not built")
    vocab, text, sms = 151936, 32769, 148
    size = logits._workspace(requests, requests, vocab, text, biases, True, False, sms)
    most = min(text + biases, -(-vocab // lists))
    starts = -(-vocab // 256) + 1
    assert size <= requests * lists * (most * (12 if biases else 8) + starts * 4) + 64


def test_texts_that_could_not_be_counted_are_refused():
    wide = torch.zeros(2, 1, dtype=torch.int32).expand(2, 1 << 26)
    with pytest.raises(ValueError, match="texts of at most"):
        ops.adjust_logits(torch.zeros(2, 5), tokens=wide, lengths=torch.zeros(2, dtype=torch.int32), presence=torch.ones(2))


def test_page_tables_whose_last_nodes_would_pass_32_bits_are_refused():
    """A context that fills a table of 2^31 tokens has no place for nodes that an int can count; both entries of tree attention refuse the table before a launch."""
    import ctypes

    from slime_b200.ops import _lib

    if not _lib.available():
        pytest.skip("the kernel library is not built")
    lib, size = _lib.lib(), ctypes.c_long()
    for tokens, fits in (((1 << 31) - 256, True), ((1 << 31) - 128, False), ((1 << 31) - 1, False), (1 << 31, False)):
        assert (lib.sb_tree_attn_plan(1, 2, 2, 64, 4, tokens, 0, 148, ctypes.byref(size)) == 0) == fits
        if not fits:
            assert lib.sb_tree_attn(*[None] * 9, 4, 1, 2, 2, 64, 1, min(tokens, (1 << 31) - 1), 100, 4, *[0] * 7, 1.0, 0, None) == 1
