"""Operators for decoding with drafted tokens over the paged cache, as cases that can be timed and compared.

Four operators, in the order in which a step that verifies drafts calls them.  The new tokens of a request are its pending token
(node 0) and drafted ones behind it, packed; parents name each node's parent by its number in the request.

  trees   ops.draft_trees           ancestor bits and positions of every node, from the parents.
  attend  ops.paged_tree_attention  each node over the request's cached tokens and its own ancestors.
  verify  ops.verify_drafts         which drafts stay, and the token behind them: by the largest score, or from the target's
                                    probabilities and given random numbers, with or without those the drafts were drawn from.
  keep    ops.keep_drafts           the kept nodes' keys and values moved together in all layers, spare pages given back.

Head layouts are those of the package's two benchmark models (32 query heads on 4 of 64; 12 on 2 of 128) and generic ones; the
vocabulary of 32000 is its first model's.  ``own`` False: the same results from elementary torch operations, in 32 bits,
sums over a vocabulary in 64.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
NODES = 64  # of a request's tree, at most
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

SMALL_HEADS = {"heads": 32, "kv_heads": 4, "d": 64}    # the benchmark's first model
MEDIUM_HEADS = {"heads": 12, "kv_heads": 2, "d": 128}  # the second: six query heads share a KV head
LARGE_HEADS = {"heads": 32, "kv_heads": 8, "d": 128}   # a generic larger model
LAYOUTS = [SMALL_HEADS, MEDIUM_HEADS, LARGE_HEADS, {"heads": 8, "kv_heads": 8, "d": 96},
           {"heads": 16, "kv_heads": 1, "d": 80}]

# No drawn case costs more than the largest listed ones.
_MAX_FLOPS = 1.1e11
_MAX_BYTES = 1.0e9
# Scores of the plain form (requests x heads x nodes x keys of the longest), probabilities, values in the caches.
_MAX_SIZE = {"attend": 5.1e8, "verify": 1.0e8, "keep": 6.0e8, "trees": 1}


def listed() -> list[dict]:
    return [
        # One stream, a small tree behind the pending token, at the package's own cache length: latency.
        {"name": "attend_single", "op": "attend", **SMALL_HEADS, "dtype": "fp16", "seqs": 1, "ctx_lo": 120, "ctx_hi": 120,
         "new_lo": 16, "new_hi": 16, "shape": "levels", "block": 16, "mix": 1, "pad": 0},
        # A server's batch: short trees behind requests of very different lengths.
        {"name": "attend_batch", "op": "attend", **MEDIUM_HEADS, "dtype": "bf16", "seqs": 16, "ctx_lo": 100, "ctx_hi": 8191,
         "new_lo": 5, "new_hi": 31, "shape": "levels", "block": 16, "mix": 4, "pad": 3},
        # Wide trees: many rows per request, where the products count.
        {"name": "attend_wide", "op": "attend", **LARGE_HEADS, "dtype": "bf16", "seqs": 8, "ctx_lo": 500, "ctx_hi": 4000,
         "new_lo": 64, "new_hi": 64, "shape": "branches", "block": 32, "mix": 9, "pad": 0},
        # Two requests with very long contexts.
        {"name": "attend_long", "op": "attend", **LARGE_HEADS, "dtype": "bf16", "seqs": 2, "ctx_lo": 60001, "ctx_hi": 131071,
         "new_lo": 25, "new_hi": 61, "shape": "levels", "block": 64, "mix": 2, "pad": 0},
        # Greedy verification of one stream's tree by the first model's logits: latency.
        {"name": "verify_greedy", "op": "verify", "mode": "greedy", "dtype": "fp16", "vocab": 32000, "seqs": 1, "new_lo": 16,
         "new_hi": 16, "shape": "levels", "mix": 1, "pad": 0},
        # The same for a batch, with a large, odd vocabulary.
        {"name": "verify_greedy_batch", "op": "verify", "mode": "greedy", "dtype": "bf16", "vocab": 100003, "seqs": 16,
         "new_lo": 12, "new_hi": 64, "shape": "levels", "mix": 3, "pad": 2},
        # Drafts without probabilities (looked up in the text, or the draft's best): trees of a large batch.
        {"name": "verify_tokens", "op": "verify", "mode": "tokens", "dtype": "fp32", "vocab": 32000, "seqs": 64, "new_lo": 2,
         "new_hi": 24, "shape": "levels", "mix": 5, "pad": 0},
        # Drafts drawn from a smaller model's probabilities, several for a place.
        {"name": "verify_drawn", "op": "verify", "mode": "drawn", "dtype": "fp32", "vocab": 150001, "seqs": 16, "new_lo": 5,
         "new_hi": 19, "shape": "branches", "mix": 6, "pad": 1},
        # What is kept of one stream's tree, in all layers of the first model.
        {"name": "keep_single", "op": "keep", **SMALL_HEADS, "dtype": "fp16", "layers": 22, "seqs": 1, "ctx_lo": 120,
         "ctx_hi": 120, "new_lo": 16, "new_hi": 16, "block": 16, "mix": 5, "pad": 0},
        # Of a batch's, in all layers of the second.
        {"name": "keep_batch", "op": "keep", **MEDIUM_HEADS, "dtype": "bf16", "layers": 28, "seqs": 64, "ctx_lo": 30,
         "ctx_hi": 1500, "new_lo": 8, "new_hi": 64, "block": 16, "mix": 4, "pad": 0},
        # The tables of one stream's tree, and of a large batch of trees.
        {"name": "trees_single", "op": "trees", "seqs": 1, "ctx_lo": 120, "ctx_hi": 120, "new_lo": 16, "new_hi": 16,
         "shape": "levels", "mix": 1, "pad": 0},
        {"name": "trees_many", "op": "trees", "seqs": 500, "ctx_lo": 0, "ctx_hi": 8191, "new_lo": 1, "new_hi": 64,
         "shape": "levels", "mix": 7, "pad": 33},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, count: int, lo: int, hi: int) -> list[int]:
    """Lengths spread over the logarithm of [lo, hi]; lo = 0 leaves about every sixth empty."""
    return [0 if lo == 0 and rng.random() < 0.17 else _log_int(rng, max(lo, 1), max(hi, 1)) for _ in range(count)]


def _case_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens in the cache, nodes) of a case's requests."""
    rng = random.Random(case["mix"])
    ctx = _lengths(rng, case["seqs"], case["ctx_lo"], case["ctx_hi"]) if "ctx_lo" in case else [0] * case["seqs"]
    return ctx, _lengths(rng, case["seqs"], case["new_lo"], case["new_hi"])


def _tree(rng, n: int, shape: str) -> list[int]:
    """Parents of a tree of n nodes, node 0 its root."""
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "branches":  # a main chain of the drafter's first choices, then shorter alternatives from places on it
        main = max(1, (n + 1) // 2) if n > 1 else 0
        parents = [i - 1 for i in range(min(n, main + 1))]
        while len(parents) < n:
            start = rng.randrange(0, main)
            at = start
            for _ in range(min(rng.randrange(1, 4), main - start, n - len(parents))):
                parents.append(at)
                at = len(parents) - 1
        return parents
    # Levels: every level's nodes hang from random ones of the level before, three to one place at most or so.
    parents, level = [-1][:n], [0]
    while len(parents) < n:
        width = min(n - len(parents), max(1, min(3 * len(level), rng.randrange(1, 10))))
        parents += sorted(rng.choice(level) for _ in range(width))
        level = list(range(len(parents) - width, len(parents)))
    return parents


def _case_parents(case: dict) -> list[list[int]]:
    rng = random.Random(1000 + case["mix"])
    return [_tree(rng, n, case.get("shape", "branches")) for n in _case_lengths(case)[1]]


def _case_paths(case: dict) -> list[list[int]]:
    """Of each request's tree the nodes that are kept: the root's path to some node.  Nodes that move lie behind every place that
    is written, so the call can be made again on the same caches."""
    rng = random.Random(2000 + case["mix"])
    paths = []
    for parents in _case_parents(case):
        path, at = [], rng.randrange(len(parents)) if parents else -1
        while at >= 0:
            path.append(at)
            at = parents[at]
        paths.append(path[::-1])
    return paths


def _pairs(case: dict) -> int:
    """(node, key) pairs of an attention case: the cached tokens and the node's ancestors."""
    total = 0
    for ctx, parents in zip(_case_lengths(case)[0], _case_parents(case)):
        depth = []
        for p in parents:
            depth.append(1 if p < 0 else depth[p] + 1)
        total += ctx * len(parents) + sum(depth)
    return total


def work(case: dict) -> dict:
    ctx, new = _case_lengths(case)
    total = sum(new)
    if case["op"] == "trees":  # parents, offsets and lengths in; bits and positions out
        return {"bytes": 4 * total + 8 * len(ctx) + 4 + 16 * (total + case["pad"]), "flops": 12 * total}
    if case["op"] == "attend":
        h, hk, d = case["heads"], case["kv_heads"], case["d"]
        keys = sum(c + n for c, n in zip(ctx, new) if n)
        return {"bytes": 2 * d * (h * total + h * (total + case["pad"]) + 2 * hk * keys) + 8 * total,
                "flops": 4 * d * h * _pairs(case)}
    if case["op"] == "verify":
        small = total * (8 + 4 + 8) + len(ctx) * (4 + 8 + 16 * NODES)
        if case["mode"] == "greedy":
            size = 4 if case["dtype"] == "fp32" else 2
            return {"bytes": total * case["vocab"] * size + small, "flops": total * case["vocab"]}
        live = sum(n > 0 for n in new)  # the last node's row of each request, and the row that its drafts were drawn from
        rows = 2 if case["mode"] == "drawn" else 1
        return {"bytes": 4 * live * case["vocab"] * rows + small, "flops": 2 * rows * live * case["vocab"]}
    moved = sum(i != p for path in _case_paths(case) for i, p in enumerate(path))
    entry = 2 * case["kv_heads"] * case["d"]  # bytes of one token in one array
    return {"bytes": 2 * moved * entry * 2 * case["layers"] + 4 * len(ctx) * (4 + NODES), "flops": total}


def draw(rng) -> dict:
    """One more case of the listed ones' ranges."""
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "verify", "keep", "trees"])
    mix, pad = rng.randrange(1, 1000), rng.choice([0, 0, 1, 5, 33])
    while True:
        new_hi = _log_int(rng, 1, NODES)
        case = {"op": op, "new_lo": rng.choice([0, 1, max(1, new_hi // 3), new_hi]), "new_hi": new_hi, "mix": mix, "pad": pad,
                "shape": rng.choice(["levels", "levels", "branches", "chain"])}
        if op == "verify":
            mode = rng.choice(["greedy", "tokens", "drawn"])
            case.update(mode=mode, dtype=rng.choice(["fp16", "bf16", "fp32"]) if mode == "greedy" else "fp32",
                        vocab=_log_int(rng, 500, 150001), seqs=_log_int(rng, 1, 64))
        else:
            ctx_hi = _log_int(rng, 30, {"attend": 131071, "keep": 1500, "trees": 131071}[op])
            case.update(ctx_lo=rng.choice([0, max(1, ctx_hi // 60)]), ctx_hi=ctx_hi,
                        seqs=_log_int(rng, 1, 500 if op == "trees" else 64))
        if op in ("attend", "keep"):
            case.update(rng.choice(LAYOUTS), dtype=rng.choice(["fp16", "bf16"]), block=rng.choice([16, 32, 64, 128]))
        if op == "keep":
            case.update(layers=_log_int(rng, 1, 32), shape="branches", new_lo=max(1, case["new_lo"]), pad=0)
        ctx, new = _case_lengths(case)
        if sum(new) == 0 or (op == "keep" and not any(i != p for path in _case_paths(case) for i, p in enumerate(path))):
            mix += 1
            continue
        w = work(case)
        size = 0
        if op == "attend":
            size = len(ctx) * case["heads"] * max(new) * (max(ctx) + max(new))
        elif op == "verify":
            size = 2 * (sum(new) + pad) * case["vocab"]
        elif op == "keep":
            size = 2 * case["layers"] * case["kv_heads"] * case["d"] * sum(c + n + case["block"] for c, n in zip(ctx, new))
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES and size <= _MAX_SIZE[op]:
            return case


# ---- inputs -------------------------------------------------------------------------------------------


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(lens: list[int]) -> list[int]:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _ops():
    root = str(Path(__file__).resolve().parent.parent / "kernel-forge_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kernelforge import ops

    return ops


def _pages(ctx, new, block: int, width: int, g) -> tuple[torch.Tensor, int]:
    """(table [seqs, width] with the pages of the first ctx + new tokens, pages in all), in random order."""
    need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(ctx), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    return table, total


def _normal(shape, dtype, g) -> torch.Tensor:
    """Normal values drawn in pieces: the 32-bit draws need not fit twice."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 28):
        piece = flat[a:a + (1 << 28)]
        piece.copy_(torch.randn(piece.numel(), generator=g, device=DEV))
    return out


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    ctx, new = _case_lengths(case)
    parents = _case_parents(case)
    offsets = _offsets(new)
    tokens = offsets[-1] + case["pad"]
    flat = [p for tree in parents for p in tree] + [-1] * case["pad"]
    state = {"case": case, "ctx": ctx, "new": new, "cu": _int32(offsets), "parents": _int32(flat), "max_new": max(new),
             "seq_lens": _int32([c + n for c, n in zip(ctx, new)])}
    if own:
        state["ops"] = _ops()
    if case["op"] == "trees":
        # Another seed, other lengths in the caches: the trees are the drafter's.
        shift = torch.randint(0, 50, (len(ctx),), generator=g, device=DEV).int()
        state["seq_lens"] += shift
        return state
    if case["op"] == "verify":
        _prepare_verify(state, flat, offsets, tokens, g)
        return state
    dtype, hk, d, block = _DTYPES[case["dtype"]], case["kv_heads"], case["d"], case["block"]
    width = max(-(-(c + n) // block) for c, n in zip(ctx, new)) + 1
    table, pages = _pages(ctx, new, block, width, g)
    state["table"] = table
    if case["op"] == "keep":
        state["caches"] = _normal((2 * case["layers"], pages, hk, block, d), dtype, g)
        paths = _case_paths(case)
        state["counts"] = _int32([len(p) for p in paths])
        state["path"] = _int32([p + [-1] * (NODES - len(p)) for p in paths])
        # The stack after the step's pages were taken: three are left, the places above are free to take pages back.
        state["free_pages"] = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
        held = set(table.flatten().tolist())
        state["free_pages"][:3] = _int32([p for p in range(pages) if p not in held])
        state["free_count"] = _int32([3])
        state["context_lens"] = _int32(ctx)
        return state
    qk = torch.randn(tokens, case["heads"] + hk, d, generator=g, device=DEV).to(dtype)
    bits = []  # as ops.draft_trees gives them
    for tree in parents:
        mine = []
        for i, p in enumerate(tree):
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
        bits += mine
    bits = [b - (1 << 64) if b >> 63 else b for b in bits] + [0] * case["pad"]
    state.update(q=qk[:, :case["heads"]], cache_k=_normal((pages, hk, block, d), dtype, g),
                 cache_v=_normal((pages, hk, block, d), dtype, g),
                 ancestors=torch.tensor(bits, dtype=torch.int64, device=DEV))
    return state


def _prepare_verify(state: dict, flat: list[int], offsets: list[int], tokens: int, g) -> None:
    """Scores or probabilities of a model that is fairly sure of some tokens, and drafts that it often agrees with."""
    case = state["case"]
    vocab = case["vocab"]
    first = [o for o, n in zip(offsets, state["new"]) for _ in range(n)] + [0] * case["pad"]
    above = torch.tensor([f + max(p, 0) for f, p in zip(first, flat)], dtype=torch.int64, device=DEV)
    logits = torch.randn(tokens, vocab, generator=g, device=DEV)
    chance = torch.rand(tokens, generator=g, device=DEV)
    if case["mode"] == "greedy":
        state["target"] = logits.to(_DTYPES[case["dtype"]])
        best = state["target"].float().argmax(-1)[above]
        other = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
        state["tokens"] = torch.where(chance < 0.6, best, other)
        return
    logits.mul_(5.0)
    rough = logits + 0.7 * torch.randn(tokens, vocab, generator=g, device=DEV)
    state["target"] = torch.softmax(logits, -1)
    draft = torch.softmax(rough, -1)
    u = torch.rand(tokens, generator=g, device=DEV, dtype=torch.float64)
    drawn = torch.empty(tokens, dtype=torch.int64, device=DEV)
    for a in range(0, tokens, 64):  # each node's token from its parent's row
        rows = draft[above[a:a + 64]].double().cumsum(-1)
        drawn[a:a + 64] = torch.searchsorted(rows, (u[a:a + 64] * rows[:, -1])[:, None], right=True)[:, 0]
    state["tokens"] = drawn.clamp(max=vocab - 1)
    if case["mode"] == "drawn":
        state["draft"] = draft
    state["accept_u"] = chance
    state["sample_u"] = torch.rand(len(state["new"]), generator=g, device=DEV)


# ---- one pass -----------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return _run_own(state)
    return {"trees": _plain_trees, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[
        state["case"]["op"]](state)


def _run_own(s: dict):
    ops, op = s["ops"], s["case"]["op"]
    if op == "trees":
        return tuple(ops.draft_trees(s["parents"], s["cu"], s["seq_lens"]))
    if op == "attend":
        return ops.paged_tree_attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["cu"], s["seq_lens"], s["ancestors"],
                                        max_new=s["max_new"])
    if op == "verify":
        return tuple(ops.verify_drafts(s["tokens"], s["parents"], s["cu"], s["target"], s.get("accept_u"), s.get("sample_u"),
                                       draft=s.get("draft")))
    kept = ops.keep_drafts(s["caches"], s["table"], s["context_lens"], s["seq_lens"], s["counts"], s["path"], s["free_pages"],
                           s["free_count"])
    return s["caches"], s["free_pages"], kept.context_lens, kept.free_count


def _rows_of(s: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(row, there, parent) [seqs, NODES]: every node's row of the packed tokens, whether it is one, its parent's number."""
    cu = s["cu"].long()
    node = torch.arange(NODES, device=cu.device)[None]
    there = node < (cu[1:] - cu[:-1])[:, None]
    row = torch.where(there, cu[:-1, None] + node, 0)
    parent = torch.where(there, s["parents"].long()[row], -1)
    return row, there, parent


def _plain_bits(parent: torch.Tensor, there: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(ancestors [seqs, NODES, NODES] of truth values, a node its own; depth): pointers doubled six times."""
    node = torch.arange(NODES, device=parent.device)
    anc = torch.eye(NODES, dtype=torch.bool, device=parent.device).expand(parent.shape[0], -1, -1) & there[:, :, None]
    jump = torch.where(parent >= 0, parent, node)
    for _ in range(6):
        anc = anc | anc.gather(1, jump[:, :, None].expand(-1, -1, NODES))
        jump = jump.gather(1, jump)
    return anc, anc.sum(-1) - 1


def _plain_trees(s: dict):
    row, there, parent = _rows_of(s)
    anc, depth = _plain_bits(parent, there)
    bits = (anc.long() << torch.arange(NODES, device=row.device)).sum(-1)
    total = s["parents"].numel()
    ancestors = torch.zeros(total, dtype=torch.int64, device=row.device)
    positions = torch.full((total,), -1, dtype=torch.int64, device=row.device)
    cu = s["cu"].long()
    context = s["seq_lens"].long() - (cu[1:] - cu[:-1])
    ancestors[row[there]] = bits[there]
    positions[row[there]] = (context[:, None] + depth)[there]
    return ancestors, positions


def _plain_attend(s: dict):
    case = s["case"]
    h, hk, d, block = case["heads"], case["kv_heads"], case["d"], case["block"]
    b, n, keys = len(s["new"]), s["max_new"], max(c + m for c, m in zip(s["ctx"], s["new"]))
    dev, rep = s["q"].device, h // hk
    row, there, _ = _rows_of(s)
    row, there = row[:, :n], there[:, :n]
    at = torch.arange(keys, device=dev)
    page = s["table"].long()[:, at // block].clamp(min=0)  # [b, keys]
    k, v = (s[name][page, :, at % block].float().permute(0, 2, 1, 3).contiguous() for name in ("cache_k", "cache_v"))
    q = s["q"][row].float().view(b, n, hk, rep, d).permute(0, 2, 3, 1, 4).reshape(b, hk, rep * n, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d)).view(b, hk, rep, n, keys)
    context = (s["seq_lens"] - (s["cu"][1:] - s["cu"][:-1])).long()[:, None]
    node = at - context  # [b, keys]: of a new token, its number
    bits = s["ancestors"][row]
    seen = (node < 0)[:, None] | ((node < n)[:, None] & ((bits[:, :, None] >> node.clamp(0, 63)[:, None]) & 1).bool()
                                  & (node >= 0)[:, None])
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    score = (score - score.amax(-1, keepdim=True)).exp_()
    score /= score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(b, hk, rep * n, keys), v).view(b, hk, rep, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)
    out = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=dev)
    out[row[there]] = o[there].to(out.dtype)
    return out


def _plain_verify(s: dict):
    case = s["case"]
    vocab, mode, target = case["vocab"], case["mode"], s["target"]
    row, there, parent = _rows_of(s)
    dev = row.device
    node = torch.arange(NODES, device=dev)
    token = s["tokens"][row]
    child = there & (parent >= 0)
    up = parent.clamp(min=0)
    up_row = row.gather(1, up)
    # elder[b, c, e]: e is a child of c's parent and comes before c.
    elder = child[:, :, None] & child[:, None] & (parent[:, :, None] == parent[:, None]) & (node[None] < node[:, None])
    if mode == "greedy":
        top = target.amax(-1, keepdim=True)
        best = torch.where(target == top, torch.arange(vocab, device=dev), vocab).amin(-1)
        accept = child & (token == best[up_row])
    elif mode == "tokens":
        p = target[up_row, token].double()
        again = elder & (token[:, :, None] == token[:, None])
        fresh = ~again.any(-1)  # of several children with one token the first counts
        left = 1.0 - ((elder & fresh[:, None]).double() * p[:, None]).sum(-1)
        accept = child & fresh & (s["accept_u"][row].double() * left < p)
    else:
        draft, rank = s["draft"], elder.sum(-1)
        taken = torch.zeros(row.shape, dtype=torch.float64, device=dev)  # of the draft's probabilities, for this node's test
        left = torch.ones_like(taken)
        p, q = target[up_row, token].double(), draft[up_row, token].double()
        per_row = torch.zeros(target.shape[0], 2, dtype=torch.float64, device=dev)
        per_row[:, 1] = 1.0
        for k in range(1, int(rank.amax()) + 2):  # what the tests of the k-th children, or the draw behind k, go by
            rows = up_row[child & (rank == k - 1)]
            a, z = per_row[rows, 0] + per_row[rows, 1], per_row[rows, 1]
            z = (target[rows].double() - a[:, None] * draft[rows].double()).clamp_(min=0).sum(-1)
            per_row[rows] = torch.stack([a, z], -1)
            here = child & (rank == k)
            taken = torch.where(here, per_row[up_row, 0], taken)
            left = torch.where(here, per_row[up_row, 1], left)
        accept = child & (s["accept_u"][row].double() * left * q < (p - taken * q).clamp(min=0))
    chosen = accept & ~(elder & accept[:, None]).any(-1)  # the first that is accepted
    chosen[:, 0] = there[:, 0]
    anc, _ = _plain_bits(parent, there)
    on = there & ~(anc & ~chosen[:, None]).any(-1)
    counts = on.sum(-1)
    path = torch.where(on, node, NODES).sort(-1).values
    path = torch.where(path < NODES, path, -1)
    last = path.gather(1, (counts - 1).clamp(min=0)[:, None])
    last_row = row.gather(1, last.clamp(min=0))[:, 0]
    if mode == "greedy":
        following = best[last_row]
    else:
        f = target[last_row].double()
        under = child & (parent == last)  # rejected children of the last node
        if mode == "tokens":
            gone = torch.zeros(f.shape[0], vocab + 1, dtype=torch.bool, device=dev)
            gone.scatter_(1, torch.where(under, token, vocab), True)
            f = f.masked_fill(gone[:, :vocab], 0.0)
        else:
            a = torch.where(under.any(-1), per_row[last_row, 0], 0.0)
            f = (f - a[:, None] * draft[last_row].double()).clamp_(min=0)
        total = f.cumsum(-1)
        following = (total <= (s["sample_u"].double() * total[:, -1])[:, None]).sum(-1).clamp(max=vocab - 1)
    step = torch.where(path[:, 1:] >= 0, token.gather(1, path[:, 1:].clamp(min=0)), -1)
    emitted = torch.cat([step, torch.full_like(step[:, :1], -1)], 1)
    live = counts > 0
    emitted.scatter_(1, (counts - 1).clamp(min=0)[:, None], torch.where(live, following, -1)[:, None])
    return counts.int(), path.int(), emitted


def _plain_keep(s: dict):
    block, caches, table = s["case"]["block"], s["caches"], s["table"].long()
    ctx, counts, path = s["context_lens"].long()[:, None], s["counts"].long()[:, None], s["path"].long()
    node = torch.arange(NODES, device=path.device)[None]
    moved = (node < counts) & (path != node)
    src, dst = ctx + path, (ctx + node).expand(path.shape)
    request = torch.arange(path.shape[0], device=path.device)[:, None].expand(path.shape)[moved]
    src, dst = src[moved], dst[moved]
    caches[:, table[request, dst // block], :, dst % block] = caches[:, table[request, src // block], :, src % block]
    context = (ctx + counts)[:, 0]
    held, need = (s["seq_lens"].long() + block - 1) // block, (context + block - 1) // block
    spare = (held - need).clamp(min=0)
    col = torch.arange(table.shape[1], device=path.device)[None]
    back = (col >= need[:, None]) & (col < held[:, None])
    at = s["free_count"].long() + (spare.cumsum(0) - spare)[:, None] + col - need[:, None]
    s["free_pages"][at[back]] = s["table"][back]
    return caches, s["free_pages"], context.int(), (s["free_count"] + spare.sum()).int()


# ---- from the definition, in 64 bits ------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"trees": _exact_trees, "attend": _exact_attend, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](s)


def _exact_trees(s: dict):
    """Node by node on the host."""
    bits, positions, seq = [], [], s["seq_lens"].tolist()
    for r, tree in enumerate(_case_parents(s["case"])):
        mine, depth = [], []
        for i, p in enumerate(tree):
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        bits += [b - (1 << 64) if b >> 63 else b for b in mine]
        positions += [seq[r] - len(tree) + x for x in depth]
    pad = s["case"]["pad"]
    return (torch.tensor(bits + [0] * pad, dtype=torch.int64, device=DEV),
            torch.tensor(positions + [-1] * pad, dtype=torch.int64, device=DEV))


def _exact_attend(s: dict):
    case = s["case"]
    hk, rep = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for r, tree in enumerate(_case_parents(case)):
        ctx = s["ctx"][r]
        n = len(tree)
        if n == 0:
            continue
        keep = torch.zeros(n, n, dtype=torch.bool)
        for i, p in enumerate(tree):
            if p >= 0:
                keep[i] = keep[p]
            keep[i, i] = True
        index = torch.arange(ctx + n, device=DEV)
        page = s["table"][r].long()[index // case["block"]]
        hidden = (~keep).to(DEV)
        for j in range(hk):
            keys, values = (s[name][page, j, index % case["block"]].double() for name in ("cache_k", "cache_v"))
            for h in range(j * rep, (j + 1) * rep):
                score = s["q"][row:row + n, h].double() @ keys.t() / math.sqrt(case["d"])
                score[:, ctx:].masked_fill_(hidden, -math.inf)
                prob = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
                out[row:row + n, h] = prob @ values
        row += n
    return out


def _exact_verify(s: dict):
    """Request by request, walking the tree from its root."""
    case, mode, vocab = s["case"], s["case"]["mode"], s["case"]["vocab"]
    tokens = s["tokens"].tolist()
    accept_u = s["accept_u"].double().tolist() if mode != "greedy" else []
    sample_u = s["sample_u"].double().tolist() if mode != "greedy" else []
    counts, paths, emitted, first = [], [], [], 0
    for r, tree in enumerate(_case_parents(case)):
        if not tree:
            counts.append(0)
            paths.append([-1] * NODES)
            emitted.append([-1] * NODES)
            continue
        at, path = 0, [0]
        while True:
            children = [c for c, p in enumerate(tree) if c > 0 and p == at]
            p = s["target"][first + at].double()
            step = None
            if mode == "greedy":
                best = int((p == p.max()).nonzero()[0])
                step = next((c for c in children if tokens[first + c] == best), None)
            else:
                left = p.clone()  # mass that is left to draw from
                mass = torch.ones((), dtype=torch.float64, device=DEV)
                q = s["draft"][first + at].double() if mode == "drawn" else None
                for c in children:
                    x = tokens[first + c]
                    weight = 1.0 if q is None else q[x]
                    if accept_u[first + c] * mass * weight < left[x]:
                        step = c
                        break
                    if q is None:
                        mass = mass - left[x]
                        left[x] = 0.0
                    else:
                        left = torch.clamp(left - mass * q, min=0.0)
                        mass = left.sum()
            if step is None:
                break
            path.append(step)
            at = step
        if mode != "greedy":
            below = torch.cumsum(left, 0)
            best = min(int((below <= sample_u[r] * below[-1]).sum()), vocab - 1)
        counts.append(len(path))
        paths.append(path + [-1] * (NODES - len(path)))
        out = [tokens[first + c] for c in path[1:]] + [best]
        emitted.append(out + [-1] * (NODES - len(out)))
        first += len(tree)
    return _int32(counts), _int32(paths), torch.tensor(emitted, dtype=torch.int64, device=DEV)


def _exact_keep(s: dict):
    """Entry by entry; values are moved, not computed."""
    block, table, seq = s["case"]["block"], s["table"].tolist(), s["seq_lens"].tolist()
    free, lens = s["free_pages"].tolist(), []
    count = s["free_count"].item()
    caches = s["caches"]
    for r, path in enumerate(_case_paths(s["case"])):
        for i, p in enumerate(path):
            if i != p:
                a, b = s["ctx"][r] + p, s["ctx"][r] + i
                caches[:, table[r][b // block], :, b % block] = caches[:, table[r][a // block], :, a % block]
        lens.append(s["ctx"][r] + len(path))
        for j in range(-(-lens[-1] // block), -(-seq[r] // block)):
            free[count] = table[r][j]
            count += 1
    return caches, _int32(free), _int32(lens), _int32([count])
