"""What a request asks of its logits before they are sampled: penalties for tokens that were used, biases, and the mask of a grammar."""

from __future__ import annotations

import torch

from slime_b200.ops import _checks, _lib, reference, tree as _tree

P = _lib.ptr


def _per_request(op: str, name: str, t, requests: int, device):
    if t is not None and (t.shape != (requests,) or t.dtype != torch.float32 or t.device != device or not t.is_contiguous()):
        raise ValueError(f"{op}: {name} must be {requests} contiguous fp32 values on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}")


def adjust_logits(logits, tokens=None, lengths=None, prompt_lens=None, *, repetition=None, frequency=None, presence=None, bias_ids=None,
                  bias_values=None, allowed=None, tree=None, out=None):  # fmt: skip
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
    Token ids, lengths and mask words are int32. Everything is worked out in fp32 and rounded once."""
    op = "adjust_logits"
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{op}: logits are [rows, vocabulary] in bf16 or fp32, not {tuple(logits.shape)} in {logits.dtype}")
    R, V = logits.shape
    dev = logits.device
    if tree is not None:
        drafted, parents, cu_nodes = tree
        _tree.check_trees(op, R, cu_nodes, _tree.MAX_NODES, drafted=drafted, parents=parents)
        S = cu_nodes.shape[0] - 1
    else:
        drafted = parents = cu_nodes = None
        S = R
    L = 0
    if repetition is not None or frequency is not None or presence is not None:
        if tokens is None or lengths is None:
            raise ValueError(f"{op}: penalties need the tokens of the requests and their lengths")
        _tree._shape(op, "tokens", tokens, S, None)
        _tree._shape(op, "lengths", lengths, S)
        L = tokens.shape[1]
        if tokens.dtype != torch.int32 or tokens.device != dev or (L > 1 and tokens.stride(1) != 1):
            raise ValueError(f"{op}: tokens must be int32 rows on {dev}")
        _tree._ints(op, dev, lengths=lengths)
        if prompt_lens is not None:
            _tree._shape(op, "prompt_lens", prompt_lens, S)
            _tree._ints(op, dev, prompt_lens=prompt_lens)
        for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            _per_request(op, name, t, S, dev)
        if _checks.enabled():
            _checks.index_range(op, "lengths", lengths, upper=L + 1)
    K = 0
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None:
            raise ValueError(f"{op}: biases are ids and values")
        _tree._shape(op, "bias_ids", bias_ids, S, None)
        K = bias_ids.shape[1]
        _tree._shape(op, "bias_values", bias_values, S, K)
        _tree._ints(op, dev, bias_ids=bias_ids)
        if bias_values.dtype != torch.float32 or bias_values.device != dev or not bias_values.is_contiguous():
            raise ValueError(f"{op}: bias_values must be contiguous fp32 on {dev}")
    if allowed is not None:
        _tree._shape(op, "allowed", allowed, R, -(-V // 32))
        if allowed.dtype != torch.int32 or allowed.device != dev or (allowed.shape[1] > 1 and allowed.stride(1) != 1):
            raise ValueError(f"{op}: allowed must be int32 words on {dev}")
    if out is None:
        out = torch.empty(R, V, dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or (V > 1 and out.stride(1) != 1):
        raise ValueError(f"{op}: out must be like logits, its rows in one piece")
    if not logits.is_cuda:
        return out.copy_(reference.adjust_logits(logits, tokens, lengths, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, tree, out))
    if R == 0 or V == 0 or (tree is not None and S == 0):
        return out
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return adjust_logits(logits, tokens, lengths, prompt_lens, repetition=repetition, frequency=frequency, presence=presence, bias_ids=bias_ids,
                                 bias_values=bias_values, allowed=allowed, tree=tree, out=out)  # fmt: skip
    logits = logits if V == 1 or logits.stride(1) == 1 else logits.contiguous()
    rc = _lib.lib().sb_adjust_logits(
        P(logits), P(out), P(tokens), P(lengths), P(prompt_lens), P(repetition), P(frequency), P(presence), P(bias_ids), P(bias_values), P(allowed),
        P(drafted), P(parents), P(cu_nodes), logits.stride(0), out.stride(0), tokens.stride(0) if L else 0, K,
        allowed.stride(0) if allowed is not None else 0, R, S, V, L, K, int(logits.dtype == torch.float32), _lib.stream())  # fmt: skip
    _lib.check(rc, "sb_adjust_logits")
    return out
