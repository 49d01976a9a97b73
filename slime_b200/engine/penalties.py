"""What requests ask of their logits before a token is drawn: repetition, frequency and presence penalties and biases of tokens
(``ops.adjust_logits``). Same fields as the ``sampling_params`` of the ``/generate`` payload that the reference's rollouts send
(slime/rollout/sglang_rollout.py:152-221); returned log-probabilities are those of the adjusted distribution.

Requests that ask for nothing pass through untouched, and a batch in which nobody asks launches nothing."""

from __future__ import annotations

import math

import torch

from slime_b200 import ops
from slime_b200.ops import tree as tree_ops


# Penalties and biases are worked out in fp32: up to this size (a repetition penalty: and down to its inverse) a count of 2^24 tokens times a penalty, a bias
# behind it and a temperature of 1e-10 stay within its range, and a logit is never zero times or divided by zero.
LARGEST = 1e9


def check(sampling, vocab: int, rows: int = 1):
    """Raises ValueError on penalties that have no meaning or none in fp32, on biases that leave no token of the ``vocab``, and where a pass has more ``rows`` for a
    request than a tree of the operator has nodes."""
    if sampling.adjusts and rows > tree_ops.MAX_NODES:
        raise ValueError(f"penalties take chains of at most {tree_ops.MAX_NODES - 1} guesses, not {rows - 1}")
    if not 1 / LARGEST <= sampling.repetition_penalty <= LARGEST:
        raise ValueError(f"repetition_penalty must be from {1 / LARGEST:g} to {LARGEST:g}, not {sampling.repetition_penalty}")
    for name in ("frequency_penalty", "presence_penalty"):
        if not abs(getattr(sampling, name)) <= LARGEST:
            raise ValueError(f"{name} must be a number of at most {LARGEST:g} either way, not {getattr(sampling, name)}")
    hidden = 0
    for token, value in (sampling.logit_bias or {}).items():
        if not isinstance(token, int) or not 0 <= token < 1 << 31 or not (abs(value) <= LARGEST or value == -math.inf):
            raise ValueError(f"logit_bias: {value} for token {token!r} (a number of at most {LARGEST:g} either way, or minus infinity)")
        hidden += token < vocab and value == -math.inf
    if hidden >= vocab:
        raise ValueError("logit_bias: no token of the vocabulary is left")


def adjust(logits, reqs, chains=None):
    """Logits of ``reqs`` adjusted in place, a row for each; nothing happens if no request asks. ``chains`` = (ids, cu), device tensors: request b
    has the rows cu[b] .. cu[b + 1], for the last token of its text and the guesses behind it, which ``ids`` names."""
    if not any(r.sampling.adjusts for r in reqs):
        return logits
    dev, B = logits.device, len(reqs)
    texts = [r.all_ids() if r.sampling.adjusts else [] for r in reqs]
    lens = torch.tensor([len(t) for t in texts], dtype=torch.int32)
    tokens = torch.zeros(B, max(int(lens.max()), 1), dtype=torch.int32)
    for row, text in zip(tokens, texts):
        row[: len(text)] = torch.tensor(text, dtype=torch.int32)
    numbers = torch.tensor([_numbers(r.sampling) for r in reqs], dtype=torch.float32).t().contiguous().to(dev)
    ids, values = _biases([r.sampling for r in reqs], logits.shape[1])
    tree = None
    if chains is not None:
        drafted, cu = chains
        at = torch.arange(drafted.shape[0], device=dev, dtype=torch.int32)
        owner = torch.searchsorted(cu, at, right=True) - 1
        tree = (drafted, at - cu[owner] - 1, cu)  # a guess hangs on the one before it, the first row on nothing (-1)
    return ops.adjust_logits(
        logits, tokens.to(dev), lens.to(dev), torch.tensor([len(r.input_ids) for r in reqs], dtype=torch.int32).to(dev), repetition=numbers[0],
        frequency=numbers[1], presence=numbers[2], bias_ids=None if ids is None else ids.to(dev), bias_values=None if ids is None else values.to(dev),
        tree=tree, out=logits)  # fmt: skip


def _numbers(s):
    return s.repetition_penalty, s.frequency_penalty, s.presence_penalty


def _biases(samplings, vocab: int):
    """([B, K] token ids, -1 behind the last; [B, K] values), or (None, None). Tokens outside the vocabulary count for nothing and are left out."""
    lists = [[(t, v) for t, v in (s.logit_bias or {}).items() if t < vocab] for s in samplings]
    K = max(len(x) for x in lists)
    if K == 0:
        return None, None
    ids, values = torch.full((len(lists), K), -1, dtype=torch.int32), torch.zeros(len(lists), K)
    for b, x in enumerate(lists):
        if x:
            ids[b, : len(x)] = torch.tensor([t for t, _ in x], dtype=torch.int32)
            values[b, : len(x)] = torch.tensor([v for _, v in x], dtype=torch.float32)
    return ids, values


class SlotAdjustments:
    """The same for decode slots, whose texts the host does not know up to the last token: the device keeps them, a step adds the token that it is fed."""

    def __init__(self, slots: int, max_context: int, vocab: int, device):
        self.vocab = vocab
        self.text = torch.zeros(slots, max_context + 1, dtype=torch.int32, device=device)
        self.prompt_lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.numbers = torch.zeros(3, slots, device=device)
        self.numbers[0] = 1.0
        self.bias_ids = self.bias_values = None
        self.asked = [False] * slots
        self._make_room()

    def _make_room(self):
        """The memory that every step works in, whatever the number of slots: captured steps, which run one after the other, would each keep their own."""
        slots, width = self.text.shape
        biases = 0 if self.bias_ids is None else self.bias_ids.shape[1]
        size = max(ops.adjust_logits_workspace(n, self.vocab, self.text.device, text=width, biases=biases) for n in range(1, slots + 1))
        self.work = torch.empty(size, dtype=torch.uint8, device=self.text.device) if size else None

    def set(self, slot: int, req) -> bool:
        """The slot's next steps are of this request. True: the buffers of biases and workspace are others now, and a captured step is stale."""
        s = req.sampling
        if not (s.adjusts or self.asked[slot]):
            return False
        self.asked[slot] = s.adjusts
        dev = self.text.device
        self.numbers[:, slot] = torch.tensor(_numbers(s), dtype=torch.float32).to(dev)
        if s.adjusts:
            ids = torch.tensor(req.all_ids(), dtype=torch.int32)
            self.text[slot, : len(ids)] = ids.to(dev)
            self.prompt_lens[slot] = len(req.input_ids)
        ids, values = _biases([s], self.vocab)
        need, have = 0 if ids is None else ids.shape[1], 0 if self.bias_ids is None else self.bias_ids.shape[1]
        if need > have:
            room = min(max(16, 1 << (need - 1).bit_length()), self.vocab)
            grown = (torch.full((self.text.shape[0], room), -1, dtype=torch.int32, device=dev), torch.zeros(self.text.shape[0], room, device=dev))
            if have:
                grown[0][:, :have], grown[1][:, :have] = self.bias_ids, self.bias_values
            self.bias_ids, self.bias_values = grown
            self._make_room()
        if self.bias_ids is not None:
            self.bias_ids[slot] = -1
            if need:
                self.bias_ids[slot, :need], self.bias_values[slot, :need] = ids[0].to(dev), values[0].to(dev)
        return need > have

    def step(self, logits, ids, pos, seq_lens, active):
        """Logits of the first slots adjusted in place. The token that a slot was fed, ``ids`` at ``pos``, joins its text; idle slots keep theirs."""
        n = logits.shape[0]
        text, at = self.text[:n], pos.long()[:, None]
        text.scatter_(1, at, torch.where(active[:, None] != 0, ids[:, None], text.gather(1, at)))
        some = self.bias_ids is not None
        return ops.adjust_logits(
            logits, text, seq_lens, self.prompt_lens[:n], repetition=self.numbers[0, :n], frequency=self.numbers[1, :n], presence=self.numbers[2, :n],
            bias_ids=self.bias_ids[:n] if some else None, bias_values=self.bias_values[:n] if some else None, out=logits,
            workspace=self.work)  # fmt: skip
