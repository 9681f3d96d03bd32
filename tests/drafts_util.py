"""Definitions of the operators for steps of drafted tokens, for their tests: trees, attention with a mask among the new rows, verification in 64 bits."""
import math

import numpy as np
import torch

from tests.paged_util import D, F64


def random_parents(rng, new, padded=True):
    """Trees of `new` rows each: parents among the six rows ahead; now and then a row that is padding."""
    out = []
    for n in new:
        p = [-1] * n
        for i in range(1, n):
            p[i] = int(rng.integers(max(0, i - 6), i))
            if padded and rng.random() < 0.08:
                p[i] = [-1, i, n + 3, -2 ** 31][int(rng.integers(4))]
        out += p
    return out


def tree64(parents, new, first):
    """Ancestors of every row as Python's whole numbers, and positions."""
    seen, positions, at = [], [], 0
    for n, f in zip(new, first):
        for i in range(n):
            bits, depth, row = 0, 0, i
            while row > 0 and 0 <= parents[at + row] < row:
                bits |= 1 << row
                row = parents[at + row]
                depth += 1
            seen.append(bits | (row == 0))
            positions.append(f + depth)
        at += n
    return seen, positions


def words_of(seen, words, dev):
    flat = np.array([[(x >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for x in seen], dtype=np.uint64).reshape(len(seen), words)
    return torch.from_numpy(flat.view(np.int64)).to(dev)


def attention_seen64(q, k, v, seen, scale):
    """attention64 of paged_util with a mask seen [n, L] in place of limits."""
    n, hq, _ = q.shape
    if k.shape[0] == 0:
        zero = torch.zeros(n, hq, D, dtype=F64, device=q.device)
        return zero, zero, zero, zero[..., 0]
    k, v = (x.repeat_interleave(hq // x.shape[1], 1) for x in (k, v))
    s = (torch.einsum("nhd,lhd->nhl", q.to(F64), k) * scale).masked_fill(~seen[:, None], -math.inf)
    w = torch.where(seen.any(1)[:, None, None], torch.softmax(s, -1), 0.0)
    mass = torch.einsum("nhd,lhd->nhl", q.to(F64).abs(), k.abs()).masked_fill(~seen[:, None], 0.0).amax(-1)
    return torch.einsum("nhl,lhd->nhd", w, v), torch.einsum("nhl,lhd->nhd", w, v.abs()), torch.einsum("nhl,lhd->nhd", w * w, v * v).sqrt(), mass


def weights64(x, t):
    """exp((x - largest) / t) of a row; numbers that are none weigh nothing, infinite ones take all."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return None
    if top == np.inf:
        return (x == np.inf).astype(np.float64)
    with np.errstate(under="ignore"):
        return np.exp((x - top) / t)


def drawn(w, r):
    sums = np.cumsum(w)
    return min(int(np.searchsorted(sums, r * sums[-1], side="right")), int(np.flatnonzero(w)[-1]))


def verify64(logits, tokens, new, coins, draws, parents=None, probs=None, heats=None, top=None):
    """tokens, rows, counts of the definition; logits [T, V] and probs as 64-bit arrays.  Also the least distance of a decision from its border."""
    V, B = logits.shape[1], len(new)
    top = max(new) if top is None else top
    out, rows, counts, start, near = np.full((B, top), -1, np.int64), np.full((B, top), -1, np.int32), np.zeros(B, np.int32), 0, 1.0
    for b, whole in enumerate(new):
        n = min(whole, top)
        t = 1.0 if heats is None else heats[b]
        if n == 0:
            start += whole
            continue
        path, node, taken, last = [0], 0, [], -1
        while True:
            x = logits[start + node]
            above = (lambda i: i - 1) if parents is None else (lambda i: parents[start + i])
            kids = [i for i in range(node + 1, n) if above(i) == node]
            follow = None
            if not t > 0:
                x = np.where(np.isnan(x), -np.inf, x)
                last = int(np.argmax(x)) if x.max() > -np.inf else -1
                follow = next((i for i in kids if last >= 0 and tokens[start + i] == last), None)
            else:
                w = weights64(x, t)
                if w is None:
                    last = -1
                else:
                    p = w / math.fsum(w)
                    u, rest = coins[start + node], p.copy()
                    valid = [i for i in kids if 0 <= tokens[start + i] < V]
                    if probs is not None:
                        q = probs[start + node]
                        for i in valid:
                            near = min(near, abs(u * q[tokens[start + i]] - p[tokens[start + i]]))
                            if u * q[tokens[start + i]] < p[tokens[start + i]]:
                                follow = i
                        if kids:
                            rest = np.where(p > 0, np.maximum(p - q, 0.0), 0.0)
                    else:
                        mass = 0.0
                        for i in valid:
                            mass += rest[tokens[start + i]]
                            near = min(near, abs(u - mass))
                            if follow is None and rest[tokens[start + i]] > 0 and u < mass:
                                follow = i
                            rest[tokens[start + i]] = 0.0
                    last = drawn(rest if rest.any() else p, draws[b])
            if follow is None:
                break
            taken.append(int(tokens[start + follow]))
            path.append(follow)
            node = follow
        counts[b] = len(path)
        rows[b, :len(path)] = path
        out[b, :len(path)] = taken + [last]
        start += whole
    return out, rows, counts, near
