"""The work that is measured: what a rollout engine does around the model's products when it answers with drafted tokens.

A step of speculative decoding verifies, for every running request, a tree of drafted tokens: node 0 is the last token of the request,
which the model has not been fed yet, and every other node continues an earlier one. Three operators carry such a step:

* ``attention``: ``ops.tree_attention``. Queries of all nodes of all trees over the paged cache: a node sees the request's cached
  context, its ancestors and itself. Once a layer.
* ``logits``: ``ops.adjust_logits``. Penalties for tokens that were used before, biases and masks of a grammar on the logits of every
  row that is sampled; a row of a tree counts the drafted tokens on its path as used. Once a step, in ordinary decoding too.
* ``accept``: ``ops.accept_tree``. Follows the sampled tokens from the root as far as they were drafted, and moves the keys and values
  of the accepted nodes of all layers behind each other in the cache. Once a step.

Heads, head widths, layers and vocabularies are those of Qwen2.5-0.5B, Qwen3-4B and Qwen3-30B-A3B, which the launch recipes and the
benchmark name. Lengths are spread evenly from a shortest to a longest and then shuffled.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
#: query heads, key heads, head width, layers
HEADS = {"qwen2.5-0.5b": (14, 2, 64, 24), "qwen3-4b": (32, 8, 128, 36), "qwen3-30b-a3b": (32, 4, 128, 48)}


def _attention(name, model, requests, fewest, most, shortest, longest):
    c = dict(op="attention", model=model, requests=requests, fewest=fewest, most=most, shortest=shortest, longest=longest)
    return dict(c, name=name) if name else c


def _logits(name, requests, fewest, most, vocab, shortest, longest, bf16, penalties, biases, mask):
    c = dict(op="logits", requests=requests, fewest=fewest, most=most, vocab=vocab, shortest=shortest, longest=longest, bf16=bf16,
             penalties=penalties, biases=biases, mask=mask)  # fmt: skip
    return dict(c, name=name) if name else c


def _accept(name, model, requests, fewest, most, shortest, longest):
    c = dict(op="accept", model=model, requests=requests, fewest=fewest, most=most, shortest=shortest, longest=longest)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one conversation, a small tree: latency
        _attention("attend-one", "qwen3-4b", 1, 8, 8, 1023, 1023),
        # the benchmark's rollout: many requests, chains and small trees, heads of 64
        _attention("attend-many", "qwen2.5-0.5b", 256, 3, 9, 257, 1279),
        # long reasoning rollouts of the Qwen3-4B recipe, trees of 16 nodes: the cache is what there is to read
        _attention("attend-long", "qwen3-4b", 64, 16, 16, 1025, 5111),
        # the end of a rollout: few requests with very long answers, wide trees (8 x 64 rows on a key head)
        _attention("attend-few", "qwen3-30b-a3b", 4, 64, 64, 24001, 31999),
        # mixed traffic: requests that have just begun beside others, trees of any size
        _attention("attend-ragged", "qwen2.5-0.5b", 33, 1, 61, 0, 4097),
        # one request samples its next token, fp32 logits: latency
        _logits("logits-one", 1, 1, 1, 151936, 700, 700, False, True, 4, False),
        # a decode step of the benchmark's rollout with penalties and biases
        _logits("logits-many", 256, 1, 1, 151936, 257, 2047, False, True, 16, False),
        # the rows of drafted trees under grammars, with penalties: each row has its own mask
        _logits("logits-trees", 61, 9, 16, 151936, 129, 4095, False, True, 0, True),
        # bf16 logits of an odd vocabulary, grammars and long lists of biases, no penalties
        _logits("logits-bf16", 512, 1, 1, 32003, 33, 511, True, False, 300, True),
        # one conversation's tree: latency
        _accept("accept-one", "qwen3-4b", 1, 8, 8, 1023, 1023),
        # the rollout of the Qwen3-4B recipe
        _accept("accept-many", "qwen3-4b", 64, 16, 16, 65, 255),
        # many small heads, wide trees of all sizes
        _accept("accept-wide", "qwen2.5-0.5b", 256, 1, 64, 1, 127),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    """Any of the three operators, over the range from the smallest to the largest listed case of it."""
    op = rng.choice(["attention", "attention", "logits", "accept"])
    model = rng.choice(sorted(HEADS))
    fewest = _between(rng, 1, 64)
    most = _between(rng, fewest, 64)
    if op == "attention":
        requests = _between(rng, 1, 256)
        # cached tokens over all requests, and rows times cached tokens: no more than the largest listed cases have
        hq, hkv, d, _ = HEADS[model]
        room = min(190_000 * 8 * 128 // (hkv * d), 64 * 110_000 * 32 * 128 // (most * hq * d)) // requests
        longest = _between(rng, 1, max(1, min(32_000, room)))
        return _attention(None, model, requests, fewest, most, rng.randint(0, longest), longest)
    if op == "logits":
        vocab = rng.choice([32003, 50257, 151936, 152064, 248320])
        trees = rng.random() < 0.5
        rows = max(1, 120_000_000 // vocab)
        most = min(most, 32) if trees else 1
        fewest = min(fewest, most)
        requests = _between(rng, 1, min(512, rows // most))
        longest = _between(rng, 1, 8191)
        penalties, mask = rng.random() < 0.7, rng.random() < 0.5
        biases = rng.choice([0, 1, 7, 64, 300])
        return _logits(None, requests, fewest, most, vocab, rng.randint(0, longest), longest, rng.random() < 0.5, penalties or not (biases or mask),
                       biases, mask)  # fmt: skip
    longest = _between(rng, 1, 200)
    room = 64 * 300 * 36 * 8 * 128 // (math.prod(HEADS[model][1:]) * (longest + most))
    return _accept(None, model, _between(rng, 1, max(1, min(256, room))), fewest, most, rng.randint(0, longest), longest)


# ------------------------------------------------------------------------------------------------------------ inputs
def _spread(rng, lo, hi, n):
    """n whole numbers evenly from lo to hi, shuffled."""
    x = np.full(n, (lo + hi) // 2) if n == 1 else lo + (hi - lo) * np.arange(n) // (n - 1)
    return rng.permutation(x)


def _trees(case, rng):
    """Boundaries of the trees, and for every node its parent (an earlier node of its tree; -1: the root)."""
    n = _spread(rng, case["fewest"], case["most"], case["requests"])
    cu = np.concatenate([[0], np.cumsum(n)])
    i = np.arange(cu[-1]) - np.repeat(cu[:-1], n)
    return cu, i, np.where(i == 0, -1, (rng.random_sample(len(i)) * i).astype(np.int64))


def _pages(case, rng, tokens):
    """Page table of requests with so many tokens, over a cache in which their pages lie in no order; page 0 is nobody's."""
    need = -(-tokens // PAGE)
    first = np.concatenate([[0], np.cumsum(need)])
    order = 1 + rng.permutation(first[-1])
    table = np.zeros((len(tokens), need.max()), dtype=np.int64)
    for b in range(len(tokens)):
        table[b, : need[b]] = order[first[b] : first[b + 1]]
    return table, int(tokens.sum()) // PAGE + len(tokens) + 1  # as many for every seed


def _guesses(case, rng, cu, i, parents):
    """Drafted tokens (siblings differ), and the token that each node's row sampled: three times in four one of its children."""
    drafted = (1000 * i + rng.randint(0, 1000, len(i))).astype(np.int64)
    sampled = 100_000 + rng.randint(0, 1000, len(i))
    start = np.repeat(cu[:-1], np.diff(cu))
    at = np.flatnonzero(i > 0)
    at = at[rng.random_sample(len(at)) < 0.75]
    for t in rng.permutation(at):
        sampled[start[t] + parents[t]] = drafted[t]
    return drafted, sampled


def _int(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", torch.int32)


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *shape, dtype=torch.bfloat16: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    cu, i, parents = _trees(case, rng)
    lengths = _spread(rng, case["shortest"], case["longest"], case["requests"])
    s = dict(op=case["op"], most=case["most"], cu=_int(cu), parents=_int(parents))
    if case["op"] == "logits":
        V, S, R = case["vocab"], case["requests"], int(cu[-1])
        uniform = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
        # few tokens make up most of a text
        words = lambda *shape: (V * uniform(*shape) ** 4).long().clamp_(max=V - 1).to(torch.int32)  # noqa: E731
        s["logits"] = (3 * normal(R, V, dtype=torch.float32)).to(torch.bfloat16 if case["bf16"] else torch.float32)
        s["tokens"] = words(S, max(1, case["longest"]))
        s["lengths"], s["prompts"] = _int(lengths), _int((lengths * rng.random_sample(S)).astype(np.int64))
        s["repetition"] = s["frequency"] = s["presence"] = s["bias_ids"] = s["biases"] = s["allowed"] = None
        if case["penalties"]:  # some requests ask for none
            asked = (uniform(3, S) < 0.75).float()
            s["repetition"] = 1 + 0.3 * asked[0] * uniform(S)
            s["frequency"], s["presence"] = 0.5 * asked[1] * uniform(S), asked[2] * uniform(S)
        if case["biases"]:  # lists of different lengths: what is not used is -1
            K = case["biases"]
            ids = torch.argsort(uniform(S, min(V, 8 * K)), dim=1)[:, :K] * (V // min(V, 8 * K))
            used = torch.arange(K, device="cuda") < (K * uniform(S, 1)).long() + 1
            s["bias_ids"] = torch.where(used, ids, -1).to(torch.int32)
            s["biases"] = 5 * normal(S, K, dtype=torch.float32)
        if case["mask"]:  # one row in four is free, the others may go on with one token in sixteen
            bits = [torch.randint(-(1 << 31), 1 << 31, (R, -(-V // 32)), generator=g, device="cuda") for _ in range(4)]
            s["allowed"] = torch.where(uniform(R, 1) < 0.25, -1, bits[0] & bits[1] & bits[2] & bits[3]).to(torch.int32)
        s["drafted"] = words(R)
        return s
    hq, hkv, d, layers = HEADS[case["model"]]
    n = np.diff(cu)
    table, pages = _pages(case, rng, lengths + n)
    s["table"], s["context"] = _int(table), _int(lengths)
    if case["op"] == "attention":
        s["q"] = 2 * normal(int(cu[-1]), hq, d)
        s["k"], s["v"] = normal(pages * PAGE, hkv, d), normal(pages * PAGE, hkv, d)
        return s
    drafted, sampled = _guesses(case, rng, cu, i, parents)
    s["drafted"], s["sampled"] = _int(drafted), _int(sampled)
    s["k"], s["v"] = normal(layers, pages * PAGE, hkv, d), normal(layers, pages * PAGE, hkv, d)
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        from slime_b200 import ops

        if s["op"] == "attention":
            return ops.tree_attention(s["q"], s["k"], s["v"], s["table"], s["context"], s["cu"], s["parents"], PAGE, s["most"])
        if s["op"] == "logits":
            return ops.adjust_logits(s["logits"], s["tokens"], s["lengths"], s["prompts"], repetition=s["repetition"], frequency=s["frequency"],
                                     presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["biases"], allowed=s["allowed"],
                                     tree=(s["drafted"], s["parents"], s["cu"]) if s["most"] > 1 else None)  # fmt: skip
        path, tokens, count = ops.accept_tree(s["sampled"], s["drafted"], s["parents"], s["cu"], s["most"], k_caches=s["k"], v_caches=s["v"],
                                              block_table=s["table"], context_lens=s["context"], page_size=PAGE)  # fmt: skip
        return {"path": path, "tokens": tokens, "count": count, "k": s["k"], "v": s["v"]}
    return {"attention": _plain_attention, "logits": _plain_logits, "accept": _plain_accept}[s["op"]](s)


def _rows(cu, rows):
    """Tree of each packed row, and its number in the tree."""
    t = torch.arange(rows, device=cu.device)
    tree = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return tree, t - cu.long()[tree]


def _padded(cu, x, most, fill):
    """[rows] -> [trees, most]."""
    at = cu[:-1, None].long() + torch.arange(most, device=cu.device)
    return torch.where(at < cu[1:, None], x[at.clamp(max=x.shape[0] - 1)].long(), fill)


def _ancestors(parents, most):
    """[trees, most] parents -> [trees, most, most]: 1 where the second node is the first one or above it."""
    up = (parents[:, :, None] == torch.arange(most, device=parents.device)).float()
    up = up + torch.eye(most, device=parents.device)
    for _ in range(max(1, (most - 1).bit_length())):
        up = (up @ up).clamp(max=1.0)
    return up


def _slots(table, at):
    return table.long().gather(1, (at // PAGE).clamp(max=table.shape[1] - 1)) * PAGE + at % PAGE


def _plain_attention(s):
    q, cu, most = s["q"], s["cu"], s["most"]
    (T, hq, d), hkv = q.shape, s["k"].shape[1]
    B, L = s["table"].shape[0], s["table"].shape[1] * PAGE
    tree, node = _rows(cu, T)
    qp = torch.zeros(B, most, hkv, hq // hkv, d, device=q.device)
    qp[tree, node] = q.view(T, hkv, hq // hkv, d).float()
    at = torch.arange(L, device=q.device).expand(B, L)
    slots = _slots(s["table"], at)
    k, v = s["k"][slots].float(), s["v"][slots].float()
    behind = at - s["context"][:, None]
    above = _ancestors(_padded(cu, s["parents"], most, -1), most)
    sees = above.gather(2, behind.clamp(0, most - 1)[:, None, :].expand(B, most, L)) > 0
    sees = torch.where(behind[:, None, :] < 0, True, sees & (behind < (cu[1:] - cu[:-1])[:, None])[:, None, :])
    x = (qp.permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d) @ k.permute(0, 2, 3, 1)).view(B, hkv, hq // hkv, most, L) / math.sqrt(d)
    x = torch.where(sees[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (x.view(B, hkv, -1, L) @ v.permute(0, 2, 1, 3)).view(B, hkv, hq // hkv, most, d).permute(0, 3, 1, 2, 4)
    return o[tree, node].reshape(T, hq, d).to(q.dtype)


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    most = s["most"]
    row = _rows(s["cu"], R)[0]
    if s["repetition"] is not None:
        S, L = s["tokens"].shape
        at = torch.arange(L, device=x.device)
        known, output = at < s["lengths"][:, None], (at < s["lengths"][:, None]) & (at >= s["prompts"][:, None])
        text = s["tokens"].long()
        seen = torch.zeros(S, V, device=x.device).scatter_add_(1, text, known.float())
        used = torch.zeros(S, V, device=x.device).scatter_add_(1, text, output.float())
        seen, used = seen[row], used[row]
        if most > 1:  # the drafted tokens on the way from the root, which is the text's last token itself
            above = _ancestors(_padded(s["cu"], s["parents"], most, -1), most)
            above = above * (torch.arange(most, device=x.device) > 0)
            tree, node = _rows(s["cu"], R)
            path = _padded(s["cu"], s["drafted"], most, 0)[tree]
            seen.scatter_add_(1, path, above[tree, node])
            used.scatter_add_(1, path, above[tree, node])
        r = s["repetition"][row, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][row, None] * used - s["presence"][row, None] * (used > 0)
    if s["bias_ids"] is not None:
        ids, values = s["bias_ids"][row].long(), s["biases"][row]
        x = x.scatter_add(1, ids.clamp(min=0), torch.where(ids >= 0, values, 0.0))
    if s["allowed"] is not None:
        word = torch.arange(V, device=x.device)
        x = torch.where((s["allowed"][:, word // 32] >> (word % 32)) & 1 > 0, x, -math.inf)
    return x.to(s["logits"].dtype)


def _plain_accept(s):
    most, cu = s["most"], s["cu"]
    parents, drafted, sampled = _padded(cu, s["parents"], most, -1), _padded(cu, s["drafted"], most, -1), _padded(cu, s["sampled"], most, -1)
    B = parents.shape[0]
    nodes = torch.arange(most, device=cu.device)
    here = torch.where(cu[1:] > cu[:-1], 0, -1).long()[:, None]
    path = [here]
    for _ in range(most - 1):
        said = sampled.gather(1, here.clamp(min=0))
        child = (parents == here) & (drafted == said) & (here >= 0) & (nodes > 0)
        here = torch.where(child, nodes, most).amin(1, keepdim=True)
        here = torch.where(here < most, here, -1)
        path.append(here)
    path = torch.cat(path, 1)
    count = (path >= 0).sum(1)
    tokens = torch.where(path >= 0, sampled.gather(1, path.clamp(min=0)), -1)
    # a request's rows behind the accepted ones are copied onto themselves
    context = s["context"][:, None].long()
    src = _slots(s["table"], context + torch.where(path >= 0, path, 0)).view(-1)
    dst = _slots(s["table"], context + torch.where(path >= 0, nodes, 0).view(B, most)).view(-1)
    for cache in (s["k"], s["v"]):
        cache[:, dst] = cache[:, src]
    return {"path": path.int(), "tokens": tokens.int(), "count": count.int(), "k": s["k"], "v": s["v"]}


# --------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    cu, parents = s["cu"].tolist(), s["parents"].tolist()
    if case["op"] == "attention":
        return _exact_attention(s, cu, parents)
    if case["op"] == "logits":
        return _exact_logits(s, cu, parents)
    path, tokens, count = [], [], []
    drafted, sampled = s["drafted"].tolist(), s["sampled"].tolist()
    for a, b in zip(cu[:-1], cu[1:]):
        walk = [0] if b > a else []
        while walk:
            nxt = [j for j in range(1, b - a) if parents[a + j] == walk[-1] and drafted[a + j] == sampled[a + walk[-1]]]
            if not nxt:
                break
            walk.append(nxt[0])
        rest = [-1] * (case["most"] - len(walk))
        path.append(walk + rest)
        tokens.append([sampled[a + w] for w in walk] + rest)
        count.append(len(walk))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return {"path": i32(path), "tokens": i32(tokens), "count": i32(count), "k": None, "v": None}  # what is moved is not computed


def _way_up(parents, i):
    """A node and those above it, without the root."""
    way = []
    while i > 0:
        way.append(i)
        i = parents[i]
    return way


def _exact_attention(s, cu, parents):
    T, hq, d = s["q"].shape
    group = hq // s["k"].shape[1]
    out = torch.zeros(T, hq, d, dtype=torch.float64, device="cuda")
    table, context = s["table"].tolist(), s["context"].tolist()
    for b, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        c, n = context[b], hi - lo
        slots = torch.tensor([table[b][p // PAGE] * PAGE + p % PAGE for p in range(c + n)], device="cuda")
        hidden = torch.ones(n, c + n, dtype=torch.bool)
        hidden[:, :c] = False
        for i in range(n):
            hidden[i, [c] + [c + j for j in _way_up(parents[lo:hi], i)]] = False
        k = s["k"][slots].double().permute(1, 2, 0).repeat_interleave(group, 0)
        v = s["v"][slots].double().transpose(0, 1).repeat_interleave(group, 0)
        x = torch.matmul(s["q"][lo:hi].double().transpose(0, 1), k) * d**-0.5
        out[lo:hi] = torch.matmul(x.masked_fill(hidden.cuda(), -math.inf).softmax(-1), v).transpose(0, 1)
    return out


def _exact_logits(s, cu, parents):
    R, V = s["logits"].shape
    out = torch.empty(R, V, dtype=torch.float64, device="cuda")
    lengths, prompts, drafted = s["lengths"].tolist(), s["prompts"].tolist(), s["drafted"].tolist()
    param = lambda name: None if s[name] is None else s[name].double().tolist()  # noqa: E731
    repetition, frequency, presence = param("repetition"), param("frequency"), param("presence")
    for b, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        text = s["tokens"][b, : lengths[b]].long()
        for t in range(lo, hi):
            x = s["logits"][t].double()
            if repetition is not None:
                extra = torch.tensor([drafted[lo + j] for j in _way_up(parents[lo:hi], t - lo)], dtype=torch.long, device="cuda")
                kinds = torch.cat([text, extra]).unique()
                x[kinds] = torch.where(x[kinds] > 0, x[kinds] / repetition[b], x[kinds] * repetition[b])
                kinds, times = torch.cat([text[prompts[b] :], extra]).unique(return_counts=True)
                x[kinds] -= frequency[b] * times.double() + presence[b]
            if s["bias_ids"] is not None:
                mine = s["bias_ids"][b] >= 0
                x.index_add_(0, s["bias_ids"][b][mine].long(), s["biases"][b][mine].double())
            if s["allowed"] is not None:
                bits = s["allowed"][t][:, None] >> torch.arange(32, device="cuda") & 1
                x[bits.view(-1)[:V] == 0] = -math.inf
            out[t] = x
    return out


# ------------------------------------------------------------------------------------------------------------ floor
def work(case):
    """Each input read once, each output written once. ``flops`` of the attention: its two products."""
    rng = np.random.RandomState(0)
    cu, i, parents = _trees(case, rng)
    lengths = _spread(rng, case["shortest"], case["longest"], case["requests"])
    T, n = int(cu[-1]), np.diff(cu)
    if case["op"] == "logits":
        V, S = case["vocab"], case["requests"]
        moved = T * V * (4 if case["bf16"] else 8) + 8 * S * case["biases"]
        moved += 4 * int(lengths.sum()) + 20 * S if case["penalties"] else 0
        moved += T * 4 * -(-V // 32) if case["mask"] else 0
        return {"bytes": moved, "flops": 4 * T * V}
    hq, hkv, d, layers = HEADS[case["model"]]
    pages = int((-(-(lengths + n) // PAGE)).sum())
    if case["op"] == "attention":
        keys = int((lengths + n).sum())
        depth = np.zeros(T, dtype=np.int64)
        for t in range(T):
            depth[t] = 0 if i[t] == 0 else 1 + depth[t - i[t] + parents[t]]
        pairs = int((np.repeat(lengths, n) + depth + 1).sum())  # of a node and a key that it sees
        return {"bytes": 2 * keys * hkv * d * 2 + 2 * T * hq * d * 2 + 4 * (pages + 2 * T), "flops": 4 * pairs * hq * d}
    drafted, sampled = _guesses(case, rng, cu, i, parents)
    rows = 0
    for a, b in zip(cu[:-1], cu[1:]):
        at, j = 0, 0
        while True:
            nxt = [c for c in range(at + 1, b - a) if parents[a + c] == at and drafted[a + c] == sampled[a + at]]
            if not nxt:
                break
            at, j = nxt[0], j + 1
            rows += at != j
    return {"bytes": 12 * T + 4 * len(n) * (2 * case["most"] + 3) + 2 * rows * layers * 2 * hkv * d * 2, "flops": 0}
