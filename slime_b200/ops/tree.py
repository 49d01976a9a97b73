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

import functools
import math
import struct

import torch

from slime_b200 import ops
from slime_b200.ops import _checks, _lib, reference

P = _lib.ptr
MAX_NODES = 128  # of a tree


_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
# Arguments of the C entries, as one array: a call costs some 0.1 us for every argument of its own.
_ATTENTION = struct.Struct("30q").pack
_ACCEPT = struct.Struct("23q").pack
_device_facts = {}  # by number: SMs, address of the status word


def _facts(device) -> tuple[int, int]:
    facts = _device_facts.get(device.index)
    if facts is None:
        facts = _device_facts[device.index] = _lib.sm_count(device), _lib.status_word(device).data_ptr()
    return facts


def _ints(op: str, device, **tensors):
    for name, t in tensors.items():
        if t.dtype != _I32 or t.device != device or not t.is_contiguous():
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


def check_tree_indices(op: str, rows: int, cu_nodes, max_nodes: int):
    """Debug mode: the trees lie within the rows, and none is larger than promised."""
    _checks.index_range(op, "cu_nodes", cu_nodes, upper=rows + 1)
    _checks.index_range(op, "tree sizes", cu_nodes[1:] - cu_nodes[:-1], upper=max_nodes + 1)


def _check_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, max_nodes, sinks, out):
    """Raises on what ``tree_attention`` does not take."""
    op = "tree_attention"
    _shape(op, "q", q, None, None, None)
    T, Hq, D = q.shape
    _shape(op, "k_cache", k_cache, None, None, D)
    Hkv = k_cache.shape[1]
    _shape(op, "v_cache", v_cache, k_cache.shape[0], Hkv, D)
    check_trees(op, T, cu_nodes, max_nodes, parents=parents)
    B = cu_nodes.shape[0] - 1
    _shape(op, "block_table", block_table, B, None)
    _shape(op, "context_lens", context_lens, B)
    _ints(op, q.device, cu_nodes=cu_nodes, block_table=block_table, context_lens=context_lens)
    if Hkv == 0 or Hq % Hkv or page_size <= 0:
        raise ValueError(f"{op}: {Hq} query heads over {Hkv} key heads, pages of {page_size} tokens")
    if q.dtype not in (_BF16, _F32) or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{op}: queries and caches are bf16 or fp32 alike, not {q.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    if k_cache.device != q.device or v_cache.device != q.device:
        raise ValueError(f"{op}: queries on {q.device}, caches on {k_cache.device} and {v_cache.device}")
    if D > 256:
        raise ValueError(f"{op}: heads {D} wide (at most 256)")
    if sinks is not None:
        _shape(op, "sinks", sinks, Hq)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or (out.numel() and (out.stride(2), out.stride(1)) != (1, D))):
        raise ValueError(f"{op}: out must be like q, with heads side by side")


@functools.lru_cache(maxsize=4096)
def _workspace(B: int, Hq: int, Hkv: int, D: int, max_nodes: int, tokens: int, whole: int, sms: int) -> int:
    """Bytes of workspace of the tensor-core kernel; -1 where it does not cover the call."""
    import ctypes

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

    What a row does not see may be anything, NaN too: other branches, nodes of no tree, the rest of a page. A row that sees a value that
    is not finite, with a weight above zero, has no finite output (of a node: its head is NaN as a whole). bf16, and fp32 throughout;
    heads up to 256 wide. In batch-invariant mode a row's bits depend on its own tree and ``max_nodes``, not on the requests beside it."""
    kv, dev, dtype, B = k_cache.shape, q.device, q.dtype, context_lens.shape[0]
    # (one expression for calls that are in order, which is most of what a call costs on the host; the check proper says what is wrong with others)
    if not (q.dim() == 3 and len(kv) == 3 and v_cache.shape == kv and kv[2] == q.shape[2] <= 256 and kv[1] > 0 and q.shape[1] % kv[1] == 0 and page_size > 0
            and (dtype is _BF16 or dtype is _F32) and k_cache.dtype is dtype and v_cache.dtype is dtype and k_cache.device == dev and v_cache.device == dev
            and cu_nodes.dtype is _I32 and parents.dtype is _I32 and block_table.dtype is _I32 and context_lens.dtype is _I32 and cu_nodes.device == dev
            and parents.device == dev and block_table.device == dev and context_lens.device == dev and cu_nodes.is_contiguous() and parents.is_contiguous()
            and block_table.is_contiguous() and context_lens.is_contiguous() and cu_nodes.shape == (B + 1,) and parents.shape == q.shape[:1]
            and block_table.dim() == 2 and block_table.shape[0] == B and context_lens.dim() == 1 and 0 < max_nodes <= MAX_NODES
            and sinks is None and out is None):  # fmt: skip
        _check_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, max_nodes, sinks, out)
    T, Hq, D = q.shape
    if out is None:
        out = q.new_empty(T, Hq, D)
    if sinks is not None:
        sinks = sinks.to(dev, _F32).contiguous()
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if _checks.enabled() and B:
        check_tree_indices("tree_attention", T, cu_nodes, max_nodes)
        _checks.paged("tree_attention", block_table, context_lens + (cu_nodes[1:] - cu_nodes[:-1]), page_size, kv[0])
    if not q.is_cuda:
        return reference.tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, scale, sinks, out)
    if T == 0 or B == 0:
        return out
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return tree_attention(q, k_cache, v_cache, block_table, context_lens, cu_nodes, parents, page_size, max_nodes, scale, sinks, out)
    if q.stride(2) != 1 or k_cache.stride(2) != 1 or v_cache.stride(2) != 1:
        q, k_cache, v_cache = (x if x.stride(2) == 1 else x.contiguous() for x in (q, k_cache, v_cache))
    pages = block_table.shape[1]
    strides = *q.stride()[:2], *k_cache.stride()[:2], *v_cache.stride()[:2], out.stride(0)
    lib = _lib.lib()
    if dtype is _BF16 and scale > 0:
        whole = 1 if ops.BATCH_INVARIANT else 0
        sms, status = _facts(dev)
        size = _workspace(B, Hq, kv[1], D, max_nodes, pages * page_size, whole, sms)
        if size >= 0:
            work = torch.empty(size, dtype=torch.uint8, device=dev)
            rc = lib.sb_tree_attn_tc(_ATTENTION(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(), cu_nodes.data_ptr(), parents.data_ptr(),
                0 if sinks is None else sinks.data_ptr(), out.data_ptr(), work.data_ptr(), status, T, B, Hq, kv[1], D, page_size, pages, kv[0], max_nodes,
                *strides, whole, size, sms), scale, _lib.stream())  # fmt: skip
            if rc != -1:
                _lib.check(rc, "sb_tree_attn_tc", 2 - whole)
                return out
    rc = lib.sb_tree_attn(
        P(q), P(k_cache), P(v_cache), P(block_table), P(context_lens), P(cu_nodes), P(parents), P(sinks), P(out), T, B, Hq, kv[1], D,
        page_size, pages, kv[0], max_nodes, *strides, scale, int(dtype is _F32), _lib.stream())  # fmt: skip
    _lib.check(rc, "sb_tree_attn")
    return out


def _check_caches(op: str, caches, block_table, context_lens, page_size, B: int, device):
    """Raises on caches that cannot be moved in; returns them as (slabs behind an address, bytes between them, slots, bytes of a slot's row, bytes from row to
    row) -> addresses. A stacked tensor [layers, slots, heads, width] is one address, a tensor [slots, heads, width] one of its own."""
    if block_table is None or context_lens is None or not page_size or page_size <= 0:
        raise ValueError(f"{op}: caches come with block_table, context_lens and page_size")
    _shape(op, "block_table", block_table, B, None)
    _shape(op, "context_lens", context_lens, B)
    _ints(op, device, block_table=block_table, context_lens=context_lens)
    groups, starts = {}, set()
    for c in caches:
        if c.device != device:
            raise ValueError(f"{op}: caches and trees are on one device")
        n, strides, shape = c.element_size(), c.stride(), c.shape
        if len(shape) not in (3, 4) or strides[-1] != 1 or (shape[-2] > 1 and strides[-2] != shape[-1]):
            raise ValueError(f"{op}: a cache is [layers, slots, heads, width], or a list of [slots, heads, width], each slot's row in one piece")
        layers, step = (shape[0], strides[0] * n) if len(shape) == 4 else (1, 0)
        width = shape[-1] * shape[-2] * n
        if width and layers:  # (a cache of latents has no values)
            if c.data_ptr() in starts:
                raise ValueError(f"{op}: two caches share memory (values that are a view of the keys move with them)")
            starts.add(c.data_ptr())
            groups.setdefault((layers, step, shape[-3], width, strides[-3] * n), []).append(c.data_ptr())
    return groups


def _two_stacks(k, v, block_table, context_lens, page_size, B: int, device):
    """What ``_check_caches`` returns, for two stacked tensors of one shape that are in order; None for anything else. (3 us on the host instead of 6.)"""
    if not (type(k) is torch.Tensor and type(v) is torch.Tensor and type(block_table) is torch.Tensor and type(context_lens) is torch.Tensor and page_size):
        return None
    shape, strides = k.shape, k.stride()
    if not (len(shape) == 4 and v.shape == shape and v.stride() == strides and k.dtype is v.dtype and k.device == device and v.device == device
            and strides[3] == 1 and strides[2] == shape[3] and shape[0] and page_size > 0 and block_table.dtype is _I32 and context_lens.dtype is _I32
            and block_table.device == device and context_lens.device == device and block_table.dim() == 2 and block_table.shape[0] == B
            and context_lens.shape == (B,) and block_table.is_contiguous() and context_lens.is_contiguous()):  # fmt: skip
        return None
    if k.data_ptr() == v.data_ptr():
        return None
    n = k.itemsize
    width = shape[2] * shape[3] * n
    return {(shape[0], strides[0] * n, shape[1], width, strides[1] * n): [k.data_ptr(), v.data_ptr()]} if width else {}


def accept_tree(sampled, drafted, parents, cu_nodes, max_nodes: int, *, k_caches=None, v_caches=None, block_table=None, context_lens=None,
                page_size: int | None = None):  # fmt: skip
    """Follow the sampled tokens as far as they were drafted: ``(path [B, max_nodes], tokens [B, max_nodes], count [B])``, all int32.

    ``sampled`` [T]: the token drawn from each node's row; ``drafted`` [T]: the token that each node stands for. From the root, the walk goes to the child
    (of several, the lowest-numbered) whose token was sampled where it stands. ``path[b, :count[b]]`` are the nodes it stood on, the root
    first, ``tokens`` what was sampled there: the request's next ``count[b]`` tokens. -1 behind them; a request without nodes has count 0.

    With caches (a stacked tensor [layers, slots, heads, width] or a sequence of [slots, heads, width] each) the keys and values of the nodes on
    the path move, in place, to positions ``context_lens[b] + 0, 1, 2, ...``, so that the cache holds the accepted tokens in order. No page
    that holds nodes of one request may belong to another, and no two caches share memory (values that are a
    view of the keys move with them and are left out)."""
    op, dev, rows = "accept_tree", cu_nodes.device, sampled.shape
    if not (0 < max_nodes <= MAX_NODES and len(rows) == 1 and cu_nodes.dim() == 1 and cu_nodes.shape[0] > 0 and drafted.shape == rows and parents.shape == rows
            and cu_nodes.dtype is _I32 and sampled.dtype is _I32 and drafted.dtype is _I32 and parents.dtype is _I32 and sampled.device == dev
            and drafted.device == dev and parents.device == dev and sampled.is_contiguous() and drafted.is_contiguous() and parents.is_contiguous()
            and cu_nodes.is_contiguous()):  # fmt: skip
        check_trees(op, rows[0], cu_nodes, max_nodes, sampled=sampled, drafted=drafted, parents=parents)
    T, B, groups, caches, checks = rows[0], cu_nodes.shape[0] - 1, None, (), _checks.enabled()
    if k_caches is not None or v_caches is not None:
        groups = _two_stacks(k_caches, v_caches, block_table, context_lens, page_size, B, dev)
        if groups is None or not sampled.is_cuda:
            caches = [c for kind in (k_caches, v_caches) if kind is not None for c in ((kind,) if isinstance(kind, torch.Tensor) else kind)]
            groups = _check_caches(op, caches, block_table, context_lens, page_size, B, dev)
    if checks and B:
        check_tree_indices(op, T, cu_nodes, max_nodes)
        for _, _, slots, _, _ in groups or ():
            _checks.paged(op, block_table, context_lens + (cu_nodes[1:] - cu_nodes[:-1]), page_size, slots)
    if not sampled.is_cuda:
        return reference.accept_tree(sampled, drafted, parents, cu_nodes, max_nodes, caches, block_table, context_lens, page_size)
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return accept_tree(sampled, drafted, parents, cu_nodes, max_nodes, k_caches=k_caches, v_caches=v_caches, block_table=block_table,
                               context_lens=context_lens, page_size=page_size)  # fmt: skip
    path, tokens, count = sampled.new_empty(B, max_nodes), sampled.new_empty(B, max_nodes), sampled.new_empty(B)
    first = (sampled.data_ptr(), drafted.data_ptr(), parents.data_ptr(), cu_nodes.data_ptr(), path.data_ptr(), tokens.data_ptr(), count.data_ptr())
    sms, stream, fn = _facts(dev)[0], _lib.stream(), _lib.lib().sb_tree_accept
    if not groups:
        _lib.check(fn(_ACCEPT(*first, 0, 0, T, B, max_nodes, 1, 0, 1, sms, 1, 0, 0, 0, 1, 0, 0), stream), "sb_tree_accept")
        return path, tokens, count
    where, writes = (block_table.data_ptr(), context_lens.data_ptr(), T, B, max_nodes, page_size, block_table.shape[1]), 1
    for (layers, step, slots, width, pitch), bases in groups.items():
        unit = math.gcd(16, width, pitch, step, *bases)
        for i in range(0, len(bases), 128):
            part = bases[i : i + 128]
            call = _ACCEPT(*first, *where, writes, sms, layers, step, slots, width // unit, unit, pitch, len(part)) + struct.pack(f"{len(part)}q", *part)
            _lib.check(fn(call, stream), "sb_tree_accept")
            writes = 0
    return path, tokens, count
