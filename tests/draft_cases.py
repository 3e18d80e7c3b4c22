"""Trees of drafted tokens and what their operators have to give, on the host and in 64 bits, shared by their tests."""

from __future__ import annotations

import math
import random

import torch

from attention_cases import EPS, HALF_STEP


def random_tree(n, rng, width=3):
    """Parents of n nodes: node 0 the root, every other behind one of the few nodes before it."""
    return [-1 if i == 0 else rng.randrange(max(0, i - width), i) for i in range(n)]


def chain(n):
    return [i - 1 for i in range(n)]


def ancestors_of(parents):
    """For every node the set of itself and its ancestors, as an int64 word; parents that are none begin a tree."""
    bits = []
    for i, p in enumerate(parents[:64]):
        bits.append((bits[p] if 0 <= p < i else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits] + [0] * (len(parents) - 64)


def positions_of(parents, context):
    depth = []
    for i, p in enumerate(parents[:64]):
        depth.append(depth[p] + 1 if 0 <= p < i else 0)
    return [context + d for d in depth] + [-1] * (len(parents) - 64)


def tree64(q, k, v, bits, there=None, scale=None):
    """(reference, bound) float64 [n, heads, d]: attention of n new tokens, the last of the keys, of which token t sees all keys
    before the new ones and new token j where bit j of bits[t] is set (j < 64).  The bound is that of attend64: the sums have the
    same terms in other number, and rows that see no key have to be zeros."""
    n, heads, d = q.shape
    keys, kv_heads, _ = k.shape
    rep, first = heads // kv_heads, keys - n
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = HALF_STEP[q.dtype]
    seen = torch.zeros(n, keys, dtype=torch.bool)
    seen[:, :max(first, 0)] = True
    for t, word in enumerate(bits):
        for j in range(min(n, 64)):
            seen[t, first + j] = bool(word >> j & 1)
    seen = seen.to(q.device)
    if there is not None:
        seen = seen & there[None, :]
    ref = torch.zeros(n, heads, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(ref)
    for h in range(heads):
        q64 = q[:, h].double()
        used = seen.any(0)[:, None]  # a key that no row sees adds nothing, whatever it holds
        k64, v64 = (torch.where(used, x[:, h // rep].double(), 0.0) for x in (k, v))
        s = torch.where(seen, (q64 @ k64.T) * scale, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        ref[:, h] = p @ v64
        mag = torch.where(seen, (q64.abs() @ k64.abs().T) * scale, 0.0).amax(-1, keepdim=True)
        rel = u + 2 * (d + 8) * EPS * mag + (keys + 64) * EPS
        sub = 2.0 ** -25 * (seen.double() @ v64.abs()) if q.dtype == torch.float16 else 0.0
        bound[:, h] = rel * (p @ v64.abs()) + sub + u * ref[:, h].abs() + 2.0 ** -25
    return ref, bound


def first_largest(row):
    """The first index of the largest value, NaN above all numbers."""
    nan = row.isnan()
    return int(nan.nonzero()[0]) if nan.any() else int((row == row.max()).nonzero()[0])


def mass(row):
    row = row.double()
    return torch.where(row > 0, row, 0.0)


def drawn_index(f, u):
    """The first index at which the running sum of f is above u times all of it, else the last with any."""
    total = torch.cumsum(f, 0)
    above = (total > u * total[-1]).nonzero()
    return int(above[0]) if len(above) else int((f > 0).nonzero()[-1])


def verify_on_host(tokens, parents, lens, target, accept=None, sample=None, draft=None, width=64):
    """counts, path, emitted as lists, request by request along the tree (tensors on the host)."""
    counts, paths, emitted, at, vocab = [], [], [], 0, target.shape[1]
    for r, n in enumerate(lens):
        tree, words = parents[at:at + n][:width], tokens[at:at + n][:width]
        path, node = ([0] if n else []), 0
        while n:
            children = [c for c in range(1, len(tree)) if tree[c] == node]
            step = None
            if accept is None:
                best = first_largest(target[at + node].float())
                step = next((c for c in children if words[c] == best), None)
            else:
                p = mass(target[at + node])
                f, m = p.clone(), 1.0
                for c in children:
                    x, u = words[c], float(accept[at + c])
                    inside = 0 <= x < vocab
                    if draft is None:
                        if inside and u * m < float(f[x]):
                            step = c
                            break
                        if inside:
                            m -= float(f[x])
                            f[x] = 0.0
                    else:
                        q = draft[at + node].double()
                        if inside and u * m * float(q[x]) < float(f[x]):
                            step = c
                            break
                        f = mass(f - m * q)
                        m = float(f.sum())
                if step is None:
                    f = f if float(f.sum()) > 0 else p
                    best = drawn_index(f, float(sample[r])) if float(f.sum()) > 0 else 0
            if step is None:
                break
            path.append(step)
            node = step
        out = [words[c] for c in path[1:]] + ([best] if n else [])
        counts.append(len(path))
        paths.append(path + [-1] * (width - len(path)))
        emitted.append(out + [-1] * (width - len(out)))
        at += n
    return counts, paths, emitted


def random_trees(lens, seed, width=3):
    rng = random.Random(seed)
    return [random_tree(n, rng, width) for n in lens]
