"""Trees of drafted tokens: attention over the paged cache, and acceptance.

The nodes of the trees of all requests lie packed: tree ``b`` holds rows ``cu_nodes[b] .. cu_nodes[b + 1]``. Node 0 of a tree is its root,
the request's last token, which the model has not been fed yet; ``parents[row]`` of every other node is the number (within its tree) of an
earlier node, and -1 for the root. A chain of guesses is the tree whose node i continues node i - 1. A node whose parent is anything else
belongs to no tree, and neither do the nodes below it (rows that pad a tree to a fixed size get -1): it sees nothing and is never
accepted. A tree has at most ``MAX_NODES`` nodes.

Node i's keys and values stand in the request's pages at position ``context_lens[b] + i``, behind the ``context_lens[b]`` cached tokens
(``ops.kv_write`` / ``ops.rope_kv_write`` put them there; the rotary position of a node is ``context_lens[b]`` plus its depth). One round:

    ctx = ops.tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, max_nodes)   # every layer
    logits = ops.adjust_logits(logits, ..., tree=(drafted, parents, cu_nodes))                                          # where asked for
    sampled = ops.sample(logits, ...)[0]
    path, tokens, count = ops.accept_tree(sampled, drafted, parents, cu_nodes, max_nodes, k_caches=..., v_caches=...,
                                          block_table=block_table, context_lens=context_lens, page_size=page_size)

Every row is sampled as an ordinary step at its position would, so the accepted tokens are draws of the model given the true prefix,
whatever was drafted. CPU tensors run the definitions in ``reference``.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from slime_b200 import ops
from slime_b200.ops import _checks, _lib, reference

P = _lib.ptr
MAX_NODES = 128  # of a tree


def _ints(op: str, device, **tensors):
    for name, t in tensors.items():
        if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{op}: {name} must be a contiguous int32 tensor on {device}, not {t.dtype} on {t.device}")


def _shape(op: str, name: str, t, *want):
    if t.dim() != len(want) or any(w is not None and s != w for s, w in zip(t.shape, want)):
        raise ValueError(f"{op}: {name} has shape {tuple(t.shape)}, not {tuple('any' if w is None else w for w in want)}")


def check_trees(op: str, rows: int, cu_nodes, max_nodes: int, **per_node):
    """Trees of at most ``max_nodes`` nodes in ``rows`` packed rows; raises on what does not fit."""
    if not 0 < max_nodes <= MAX_NODES:
        raise ValueError(f"{op}: trees of {max_nodes} nodes (1 to {MAX_NODES} are possible)")
    if cu_nodes.dim() != 1 or cu_nodes.shape[0] < 1:
        raise ValueError(f"{op}: cu_nodes has shape {tuple(cu_nodes.shape)}, not (trees + 1,)")
    for name, t in per_node.items():
        if t.dim() != 1 or t.shape[0] != rows:
            raise ValueError(f"{op}: {name} has shape {tuple(t.shape)}, not ({rows},)")
    _ints(op, cu_nodes.device, cu_nodes=cu_nodes, **per_node)
    if _checks.enabled():
        _checks.index_range(op, "cu_nodes", cu_nodes, upper=rows + 1)
        _checks.index_range(op, "tree sizes", cu_nodes[1:] - cu_nodes[:-1], upper=max_nodes + 1)


@functools.lru_cache(maxsize=4096)
def _workspace(B: int, Hq: int, Hkv: int, D: int, max_nodes: int, tokens: int, whole: int, sms: int) -> int:
    """Bytes of workspace of the tensor-core kernel; -1 where it does not cover the call."""
    size = ctypes.c_long()
    rc = _lib.lib().sb_tree_attn_plan(B, Hq, Hkv, D, max_nodes, tokens, whole, sms, ctypes.byref(size))
    return size.value if rc == 0 else -1


def tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size: int, max_nodes: int, scale=None,
                   sinks=None, out=None):  # fmt: skip
    """Attention of the nodes of drafted-token trees over a paged KV cache, which holds their own keys and values already.

    ``q`` [T, Hq, D] (rows and heads may be strided: a column range of a fused projection), caches [slots, Hkv, D], ``block_table`` [B, pages],
    ``context_lens`` [B], ``cu_nodes`` [B + 1], ``parents`` [T], all int32. A node sees the ``context_lens[b]`` cached tokens,
    the nodes above it and itself; a node that belongs to no tree gets zeros. ``sinks`` [Hq] fp32: score of an extra softmax column without
    a value. ``max_nodes``: no tree has more nodes. Rows of ``out`` behind ``cu_nodes[B]`` are left as they are (a new ``out``: undefined).

    Keys and values of hidden rows have weight zero and have to be finite where they belong to a tree; what stands in a page behind the
    last node may be anything. bf16, and fp32 throughout; heads up to 256 wide."""
    op = "tree_attention"
    T, Hq, D = q.shape
    Hkv = k_cache.shape[1]
    _shape(op, "k_cache", k_cache, None, None, D)
    _shape(op, "v_cache", v_cache, k_cache.shape[0], Hkv, D)
    B = cu_nodes.shape[0] - 1
    check_trees(op, T, cu_nodes, max_nodes, parents=parents)
    _shape(op, "block_table", block_table, B, None)
    _shape(op, "context_lens", context_lens, B)
    _ints(op, q.device, cu_nodes=cu_nodes, block_table=block_table, context_lens=context_lens)
    if Hkv == 0 or Hq % Hkv or page_size <= 0:
        raise ValueError(f"{op}: {Hq} query heads over {Hkv} key heads, pages of {page_size} tokens")
    if q.dtype not in (torch.bfloat16, torch.float32) or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{op}: queries and caches are bf16 or fp32 alike, not {q.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    if k_cache.device != q.device or v_cache.device != q.device:
        raise ValueError(f"{op}: queries on {q.device}, caches on {k_cache.device} and {v_cache.device}")
    if sinks is not None:
        _shape(op, "sinks", sinks, Hq)
        sinks = sinks.to(q.device, torch.float32).contiguous()
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError(f"{op}: out must be like q, with heads side by side")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if _checks.enabled() and B:
        _checks.paged(op, block_table, context_lens + (cu_nodes[1:] - cu_nodes[:-1]), page_size, k_cache.shape[0])
    if not q.is_cuda:
        return reference.tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, scale, sinks, out)
    if T == 0 or B == 0:
        return out
    if q.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(q.device):
            return tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, max_nodes, scale, sinks, out)
    q, k_cache, v_cache = (x if x.stride(-1) == 1 else x.contiguous() for x in (q, k_cache, v_cache))
    lib = _lib.lib()
    if q.dtype == torch.bfloat16 and scale > 0:
        whole, sms = int(ops.BATCH_INVARIANT), _lib.sm_count(q.device)
        size = _workspace(B, Hq, Hkv, D, max_nodes, block_table.shape[1] * page_size, whole, sms)
        if size >= 0:
            work = torch.empty(size, dtype=torch.uint8, device=q.device)
            rc = lib.sb_tree_attn_tc(
                P(q), P(k_cache), P(v_cache), P(block_table), P(context_lens), P(cu_nodes), P(parents), P(sinks), P(out), T, B, Hq, Hkv, D,
                page_size, block_table.shape[1], k_cache.shape[0], max_nodes, q.stride(0), q.stride(1), k_cache.stride(0), k_cache.stride(1),
                v_cache.stride(0), v_cache.stride(1), out.stride(0), scale, whole, P(work), size, sms, P(_lib.status_word(q.device)),
                _lib.stream())  # fmt: skip
            if rc != -1:
                _lib.check(rc, "sb_tree_attn_tc", 2 - whole)
                return out
    rc = lib.sb_tree_attn(
        P(q), P(k_cache), P(v_cache), P(block_table), P(context_lens), P(cu_nodes), P(parents), P(sinks), P(out), T, B, Hq, Hkv, D,
        page_size, block_table.shape[1], k_cache.shape[0], max_nodes, q.stride(0), q.stride(1), k_cache.stride(0), k_cache.stride(1),
        v_cache.stride(0), v_cache.stride(1), out.stride(0), scale, int(q.dtype == torch.float32), _lib.stream())  # fmt: skip
    if rc == -1:
        raise ValueError(f"{op}: heads {D} wide (at most 256)")
    _lib.check(rc, "sb_tree_attn")
    return out


def _slabs(op: str, caches):
    """The caches as (addresses, slabs behind each address, bytes between them) for every geometry of a slot's row: a stacked tensor
    [layers, slots, heads, width] is one address, a list of tensors [slots, heads, width] one each."""
    groups = {}
    for c in caches:
        layers, step = 1, 0
        if c.dim() == 4:
            layers, step = c.shape[0], c.stride(0) * c.element_size()
        if c.dim() not in (3, 4) or c.stride(-1) != 1 or (c.shape[-2] > 1 and c.stride(-2) != c.shape[-1]):
            raise ValueError(f"{op}: a cache is [layers, slots, heads, width], or a list of [slots, heads, width], each slot's row in one piece")
        width, pitch = c.shape[-1] * c.shape[-2] * c.element_size(), c.stride(-3) * c.element_size()
        if width and layers:  # (a cache of latents has no values)
            groups.setdefault((layers, step, c.shape[-3], width, pitch), []).append(c.data_ptr())
    return groups


def accept_tree(sampled, drafted, parents, cu_nodes, max_nodes: int, *, k_caches=None, v_caches=None, block_table=None, context_lens=None,
                page_size: int | None = None):  # fmt: skip
    """Follow the sampled tokens as far as they were drafted: ``(path [B, max_nodes], tokens [B, max_nodes], count [B])``, all int32.

    ``sampled`` [T]: the token drawn from each node's row; ``drafted`` [T]: the token that each node stands for. From the root, the walk goes to the child
    (of several, the lowest-numbered) whose token was sampled where it stands. ``path[b, :count[b]]`` are the nodes it stood on, the root
    first, ``tokens`` what was sampled there: the request's next ``count[b]`` tokens. -1 behind them; a request without nodes has count 0.

    With caches (a stacked tensor [layers, slots, heads, width] or a sequence of [slots, heads, width] each) the keys and values of the nodes on
    the path move, in place, to positions ``context_lens[b] + 0, 1, 2, ...``, so that the cache holds the accepted tokens in order. No page
    that holds nodes of one request may belong to another."""
    op = "accept_tree"
    T, B = sampled.shape[0], cu_nodes.shape[0] - 1
    check_trees(op, T, cu_nodes, max_nodes, sampled=sampled, drafted=drafted, parents=parents)
    groups = {}
    if k_caches is not None or v_caches is not None:
        if block_table is None or context_lens is None or not page_size or page_size <= 0:
            raise ValueError(f"{op}: caches come with block_table, context_lens and page_size")
        _shape(op, "block_table", block_table, B, None)
        _shape(op, "context_lens", context_lens, B)
        _ints(op, cu_nodes.device, block_table=block_table, context_lens=context_lens)
        caches = [c for kind in (k_caches, v_caches) if kind is not None for c in ((kind,) if isinstance(kind, torch.Tensor) else kind)]
        if any(c.device != cu_nodes.device for c in caches):
            raise ValueError(f"{op}: caches and trees are on one device")
        groups = _slabs(op, caches)
        if _checks.enabled() and B:
            for _, _, slots, _, _ in groups:
                _checks.paged(op, block_table, context_lens + (cu_nodes[1:] - cu_nodes[:-1]), page_size, slots)
    if not sampled.is_cuda:
        return reference.accept_tree(sampled, drafted, parents, cu_nodes, max_nodes, caches if groups else (), block_table, context_lens, page_size)
    if sampled.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(sampled.device):
            return accept_tree(sampled, drafted, parents, cu_nodes, max_nodes, k_caches=k_caches, v_caches=v_caches, block_table=block_table,
                               context_lens=context_lens, page_size=page_size)  # fmt: skip
    path = torch.empty(B, max_nodes, dtype=torch.int32, device=sampled.device)
    tokens, count = torch.empty_like(path), torch.empty(B, dtype=torch.int32, device=sampled.device)
    sms, stream, first = _lib.sm_count(sampled.device), _lib.stream(), True
    for (layers, step, slots, width, pitch), bases in groups.items() or [((1, 0, 0, 0, 0), [])]:
        unit = math.gcd(16, width, pitch, step, *bases)
        for i in range(0, max(1, len(bases)), 128):
            part = bases[i : i + 128]
            rc = _lib.lib().sb_tree_accept(
                P(sampled), P(drafted), P(parents), P(cu_nodes), P(path), P(tokens), P(count), T, B, max_nodes,
                (ctypes.c_ulonglong * len(part))(*part), len(part), layers, step, slots, width // unit, unit, pitch, P(block_table),
                P(context_lens), page_size or 1, 0 if block_table is None else block_table.shape[1], int(first), sms, stream)  # fmt: skip
            _lib.check(rc, "sb_tree_accept")
            first = False
    return path, tokens, count
