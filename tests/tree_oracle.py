"""Trees of drafted tokens, written node by node in 64 bits."""

from collections import Counter

import numpy as np
import torch


def way_up(parents, i):
    """Node i and those above it, [] where the way does not end at node 0."""
    way = [i]
    while i > 0:
        up = int(parents[i])
        if not 0 <= up < i:
            return []
        i = up
        way.append(i)
    return way


def make_trees(sizes, seed, holes=0.0, shape="random"):
    """(cu, parents) int32 of trees with so many nodes; a share of the nodes belongs to no tree."""
    rng = np.random.RandomState(seed)
    parents = []
    for n in sizes:
        for i in range(n):
            up = -1 if i == 0 else i - 1 if shape == "chain" else 0 if shape == "star" else int(rng.randint(0, i))
            if i > 0 and rng.random_sample() < holes:
                up = int(rng.choice([-1, -7, i, i + 1, 500]))
            parents.append(up)
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32), torch.tensor(parents, dtype=torch.int32)


def make_pages(lengths, page, seed, extra=2):
    """A page table whose pages lie in no order, entries behind the last page point far away; (table, slots of the cache)."""
    rng = np.random.RandomState(seed)
    need = [-(-n // page) for n in lengths]
    order = list(rng.permutation(sum(need) + extra))
    table = np.full((len(lengths), max(1, max(need, default=1))), 1 << 20, dtype=np.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return torch.from_numpy(table), (sum(need) + extra) * page


def slot(table, b, pos, page):
    return int(table[b, pos // page]) * page + pos % page


def attention(q, k, v, table, ctx, cu, parents, page, scale, sinks=None):
    """(outputs, sum of weight times |value|) of every row, float64; rows of no tree are zero."""
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, mass = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    q, k, v, par, cu = q.double().cpu(), k.cpu(), v.cpu(), parents.tolist(), cu.tolist()
    for b in range(len(cu) - 1):
        for i in range(cu[b + 1] - cu[b]):
            way = way_up(par[cu[b] : cu[b + 1]], i)
            if not way:
                continue
            c = int(ctx[b])
            at = torch.tensor([slot(table, b, p, page) for p in list(range(c)) + [c + j for j in sorted(way)]])
            for h in range(Hq):
                kk, vv = k[at, h // G].double(), v[at, h // G].double()
                x = scale * (kk @ q[cu[b] + i, h])
                top = x.max() if sinks is None else torch.maximum(x.max(), sinks[h].double().cpu())
                p = torch.exp(x - top)
                den = p.sum() + (0 if sinks is None else torch.exp(sinks[h].double().cpu() - top))
                out[cu[b] + i, h] = p @ vv / den
                mass[cu[b] + i, h] = p @ vv.abs() / den
    return out, mass


def adjusted(logits, tokens=None, lengths=None, prompt_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None,
             allowed=None, tree=None):  # fmt: skip
    """(logits float64, rows that are written)."""
    R, V = logits.shape
    x = logits.double().cpu().clone().numpy()
    num = lambda t, b, d: d if t is None else float(t[b])  # noqa: E731
    written = []
    for r in range(R):
        b, extra = r, []
        if tree is not None:
            drafted, parents, cu = tree[0].tolist(), tree[1].tolist(), tree[2].tolist()
            mine = [j for j in range(len(cu) - 1) if cu[j] <= r < cu[j + 1]]
            if not mine:
                continue
            b = mine[0]
            extra = [drafted[cu[b] + j] for j in way_up(parents[cu[b] : cu[b + 1]], r - cu[b]) if j > 0]
        written.append(r)
        if repetition is not None or frequency is not None or presence is not None:
            text = tokens[b, : int(lengths[b])].tolist()
            answer = text[int(prompt_lens[b]) if prompt_lens is not None else 0 :] + extra
            for t in set(text + extra):
                if 0 <= t < V:
                    f = num(repetition, b, 1.0)
                    x[r, t] = x[r, t] / f if x[r, t] > 0 else x[r, t] * f
            for t, times in Counter(answer).items():
                if 0 <= t < V:
                    x[r, t] -= num(frequency, b, 0.0) * times + num(presence, b, 0.0)
        if bias_ids is not None:
            for t, add in zip(bias_ids[b].tolist(), bias_values[b].tolist()):
                if 0 <= t < V:
                    x[r, t] += add
        if allowed is not None:
            words = allowed[r].cpu().numpy().view(np.uint32)
            for t in range(V):
                if not int(words[t // 32]) >> (t % 32) & 1:
                    x[r, t] = -np.inf
    return torch.from_numpy(x), written


def accepted(sampled, drafted, parents, cu, max_nodes):
    """Path, tokens and count of every tree, as lists."""
    said, guess, par, cu = sampled.tolist(), drafted.tolist(), parents.tolist(), cu.tolist()
    out = []
    for a, b in zip(cu[:-1], cu[1:]):
        walk = [0] if b > a else []
        while walk:
            here = walk[-1]
            nxt = [j for j in range(here + 1, b - a) if par[a + j] == here and guess[a + j] == said[a + here]]
            if not nxt:
                break
            walk.append(nxt[0])
        rest = [-1] * (max_nodes - len(walk))
        out.append((walk + rest, [said[a + i] for i in walk] + rest, len(walk)))
    return out


def moved(caches, table, ctx, path, count, page):
    """What the caches [layers, slots, ...] hold when the rows of the paths stand behind each other."""
    new = [c.clone() for c in caches]
    for b in range(len(count)):
        for j in range(int(count[b])):
            s, d = slot(table, b, int(ctx[b]) + int(path[b][j]), page), slot(table, b, int(ctx[b]) + j, page)
            for old, c in zip(caches, new):
                c[:, d] = old[:, s]
    return new
