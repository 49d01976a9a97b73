"""What a request asks of its logits before they are sampled: penalties for tokens that were used, biases, and the mask of a grammar."""

from __future__ import annotations

import ctypes
import functools
import struct

import torch

from slime_b200.ops import _checks, _lib, reference, tree as _tree

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
MAX_VOCAB = 1 << 25  # the kernels sort tokens into 1024 buckets, each of which is within a table of 32768 tokens
MAX_TEXT = (1 << 26) - 256  # a token is counted in 26 bits, drafted nodes included
_CALL = struct.Struct("28q").pack  # arguments of the C entry


@functools.lru_cache(maxsize=4096)
def _workspace(rows: int, requests: int, vocab: int, text: int, biases: int, penal: bool, tree: bool, sms: int) -> int:
    """Bytes of workspace of a call."""
    size = ctypes.c_long()
    _lib.check(_lib.lib().sb_adjust_logits_work(rows, requests, vocab, text, biases, penal, tree, sms, ctypes.byref(size)), "sb_adjust_logits_work", 0)
    return size.value


def adjust_logits_workspace(rows: int, vocab: int, device, *, requests: int | None = None, text: int = 0, biases: int = 0, penalties: bool = True,
                            tree: bool = False) -> int:  # fmt: skip
    """Bytes that ``adjust_logits`` works in for so many rows and tokens of a text (columns of ``tokens``) and biases of a request; 0: none."""
    if torch.device(device).type != "cuda" or not (penalties or biases):
        return 0
    return _workspace(rows, rows if requests is None else requests, vocab, text if penalties else 0, biases, penalties, tree, _lib.sm_count(device))


def _per_request(op: str, name: str, t, requests: int, device):
    if t is not None and (t.shape != (requests,) or t.dtype != torch.float32 or t.device != device or not t.is_contiguous()):
        raise ValueError(f"{op}: {name} must be {requests} contiguous fp32 values on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}")


def adjust_logits(logits, tokens=None, lengths=None, prompt_lens=None, *, repetition=None, frequency=None, presence=None, bias_ids=None,
                  bias_values=None, allowed=None, tree=None, out=None, workspace=None):  # fmt: skip
    """Logits [R, V] (bf16 or fp32, rows may be strided) as the requests want them sampled; ``out`` may be ``logits`` itself.

    ``tokens`` [S, L]: the text of each of S requests, of which the first ``lengths`` [S] count and the first ``prompt_lens`` [S] are prompt (None: none are).
    For a token that occurs c times behind the prompt, in this order:

    * ``repetition`` [S]: a logit above zero is divided by it, any other multiplied, if the token stands anywhere in the text;
    * ``frequency`` [S] times c, and ``presence`` [S] if c > 0, are subtracted;
    * ``bias_values`` [S, K] of the tokens ``bias_ids`` [S, K] are added (a token that is listed twice gets both, a negative id none);
    * ``allowed`` [R, ceil(V / 32)]: where bit t % 32 of word t // 32 is 0 the logit becomes -inf, whatever it was.

    None: no such step; 1, 0 and 0 leave a request's logits as they are. ``tree`` = (drafted [R], parents [R], cu_nodes [S + 1]): row r belongs to a node of
    a tree of drafted tokens (``slime_b200.ops.tree``), and the drafted tokens of the node and those above it count as answered with. The root is the
    last token of the text already. Rows behind the last tree are left as they are. Without it row r is request r.

    ``workspace``: bytes (uint8) for calls that run one after the other to share, at least as many as ``adjust_logits_workspace`` names. A captured call keeps the
    memory that it works in for good, so a program that captures many gives them one. None: the call's own.

    Token ids, lengths and mask words are int32. Everything is worked out in fp32 and rounded once."""
    if logits.dim() != 2 or not (logits.dtype is _BF16 or logits.dtype is _F32):
        raise ValueError(f"adjust_logits: logits are [rows, vocabulary] in bf16 or fp32, not {tuple(logits.shape)} in {logits.dtype}")
    R, V = logits.shape
    dev, dtype = logits.device, logits.dtype
    drafted, parents, cu_nodes = tree if tree is not None else (None, None, None)
    S = R if cu_nodes is None else cu_nodes.shape[0] - 1
    penal = repetition is not None or frequency is not None or presence is not None
    # (as in ``tree.tree_attention``: one expression for what is in order)
    fine = V <= MAX_VOCAB and (out is None or (out.shape == logits.shape and out.dtype is dtype and out.device == dev and (V <= 1 or out.stride(1) == 1)))
    if fine and penal:
        fine = (tokens is not None and lengths is not None and tokens.dim() == 2 and tokens.shape[0] == S and tokens.shape[1] <= MAX_TEXT and tokens.dtype is _I32 and tokens.device == dev
                and (tokens.shape[1] <= 1 or tokens.stride(1) == 1) and lengths.shape == (S,) and lengths.dtype is _I32 and lengths.device == dev
                and lengths.is_contiguous())  # fmt: skip
        if prompt_lens is not None:
            fine = fine and prompt_lens.shape == (S,) and prompt_lens.dtype is _I32 and prompt_lens.device == dev and prompt_lens.is_contiguous()
        for t in (repetition, frequency, presence):
            fine = fine and (t is None or (t.shape == (S,) and t.dtype is _F32 and t.device == dev and t.is_contiguous()))
    if fine and (bias_ids is not None or bias_values is not None):
        fine = (bias_ids is not None and bias_values is not None and bias_ids.dim() == 2 and bias_ids.shape[0] == S and bias_values.shape == bias_ids.shape
                and bias_ids.dtype is _I32 and bias_values.dtype is _F32 and bias_ids.device == dev and bias_values.device == dev
                and bias_ids.is_contiguous() and bias_values.is_contiguous())  # fmt: skip
    if fine and allowed is not None:
        fine = (allowed.shape == (R, -(-V // 32)) and allowed.dtype is _I32 and allowed.device == dev and (allowed.shape[1] <= 1 or allowed.stride(1) == 1))
    if not fine or tree is not None:
        _check(logits, tokens, lengths, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, tree, out, S, penal)
    if workspace is not None and not (workspace.dtype is torch.uint8 and workspace.device == dev and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0):
        raise ValueError(f"adjust_logits: a workspace is uint8 on {dev}, in one piece from a boundary of 16 bytes, not {workspace.dtype} on {workspace.device}")
    if out is None:
        out = logits.new_empty(R, V)
    if _checks.enabled():
        if tree is not None:
            _tree.check_tree_indices("adjust_logits", R, cu_nodes, _tree.MAX_NODES)
        if penal:
            _checks.index_range("adjust_logits", "lengths", lengths, upper=tokens.shape[1] + 1)
    if not logits.is_cuda:
        return out.copy_(reference.adjust_logits(logits, tokens, lengths, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, tree, out))
    if R == 0 or V == 0 or S == 0:
        return out
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return adjust_logits(logits, tokens, lengths, prompt_lens, repetition=repetition, frequency=frequency, presence=presence, bias_ids=bias_ids,
                                 bias_values=bias_values, allowed=allowed, tree=tree, out=out, workspace=workspace)  # fmt: skip
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    K = 0 if bias_ids is None else bias_ids.shape[1]
    text, pitch = (tokens.shape[1], tokens.stride(0)) if penal else (0, 0)
    sms = _tree._facts(dev)[0]
    size = _workspace(R, S, V, text, K, penal, tree is not None, sms) if penal or K else 0
    if workspace is None:
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    elif workspace.numel() < size:
        raise ValueError(f"adjust_logits: a workspace of {workspace.numel()} bytes for a call that needs {size}")
    else:
        work = workspace
    rc = _lib.lib().sb_adjust_logits(
        _CALL(logits.data_ptr(), out.data_ptr(), at(tokens), at(lengths), at(prompt_lens), at(repetition), at(frequency), at(presence), at(bias_ids),
              at(bias_values), at(allowed), at(drafted), at(parents), at(cu_nodes), logits.stride(0), out.stride(0), pitch, K,
              0 if allowed is None else allowed.stride(0), R, S, V, text, K, dtype is _F32, sms, at(work), size), _lib.stream())  # fmt: skip
    _lib.check(rc, "sb_adjust_logits")
    return out


def _check(logits, tokens, lengths, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, tree, out, S: int, penal: bool):
    """Raises on what ``adjust_logits`` does not take."""
    op, dev, (R, V) = "adjust_logits", logits.device, logits.shape
    if V > MAX_VOCAB:
        raise ValueError(f"{op}: a vocabulary of at most {MAX_VOCAB} tokens, not {V}")
    if tree is not None:
        drafted, parents, cu_nodes = tree
        _tree.check_trees(op, R, cu_nodes, _tree.MAX_NODES, drafted=drafted, parents=parents)
        if cu_nodes.device != dev:
            raise ValueError(f"{op}: logits on {dev}, trees on {cu_nodes.device}")
    if penal:
        if tokens is None or lengths is None:
            raise ValueError(f"{op}: penalties need the tokens of the requests and their lengths")
        _tree._shape(op, "tokens", tokens, S, None)
        _tree._shape(op, "lengths", lengths, S)
        if tokens.shape[1] > MAX_TEXT:
            raise ValueError(f"{op}: texts of at most {MAX_TEXT} tokens, not {tokens.shape[1]}")
        if tokens.dtype != _I32 or tokens.device != dev or (tokens.shape[1] > 1 and tokens.stride(1) != 1):
            raise ValueError(f"{op}: tokens must be int32 rows on {dev}")
        _tree._ints(op, dev, lengths=lengths)
        if prompt_lens is not None:
            _tree._shape(op, "prompt_lens", prompt_lens, S)
            _tree._ints(op, dev, prompt_lens=prompt_lens)
        for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            _per_request(op, name, t, S, dev)
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None:
            raise ValueError(f"{op}: biases are ids and values")
        _tree._shape(op, "bias_ids", bias_ids, S, None)
        _tree._shape(op, "bias_values", bias_values, S, bias_ids.shape[1])
        _tree._ints(op, dev, bias_ids=bias_ids)
        if bias_values.dtype != _F32 or bias_values.device != dev or not bias_values.is_contiguous():
            raise ValueError(f"{op}: bias_values must be contiguous fp32 on {dev}")
    if allowed is not None:
        _tree._shape(op, "allowed", allowed, R, -(-V // 32))
        if allowed.dtype != _I32 or allowed.device != dev or (allowed.shape[1] > 1 and allowed.stride(1) != 1):
            raise ValueError(f"{op}: allowed must be int32 words on {dev}")
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or (V > 1 and out.stride(1) != 1)):
        raise ValueError(f"{op}: out must be like logits, its rows in one piece")
