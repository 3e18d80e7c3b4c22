"""Serving operators of the package as cases that can be timed and compared.

Four operators, in the order in which one step of a server that decodes many requests at once calls them:

  tables   ops.paged_tables      what the step's kernels need, from the requests' lengths: new pages of the
                                 KV cache entered into the block table, offsets of the packed tokens, every
                                 token's position and the cache slot it goes to.
  rope     ops.rope_paged_cache  RoPE on q and k of a fused q|k|v projection, k and v into their slots.
  paged    ops.paged_attention   causal attention of each request's new tokens over its pages of the cache:
                                 single tokens (decode), chunks of a prompt, or both in one batch.
  prompt   ops.prompt_attention  causal attention over whole prompts, packed, straight from the projection.

Head layouts are those of the package's two benchmark models (32 query heads on 4 of 64; 12 on 2 of 128)
and generic ones.  ``own`` False: the same results from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

SMALL_HEADS = {"heads": 32, "kv_heads": 4, "d": 64}    # the benchmark's first model
MEDIUM_HEADS = {"heads": 12, "kv_heads": 2, "d": 128}  # the second: six query heads share a KV head
LARGE_HEADS = {"heads": 32, "kv_heads": 8, "d": 128}   # a generic larger model
LAYOUTS = [SMALL_HEADS, MEDIUM_HEADS, LARGE_HEADS, {"heads": 8, "kv_heads": 8, "d": 96},
           {"heads": 16, "kv_heads": 1, "d": 80}]

# No drawn case costs more than the largest listed ones.
_MAX_FLOPS = 1.0e12
_MAX_BYTES = 2.0e9


def listed() -> list[dict]:
    return [
        # A handful of short prompts that arrive together, one of them empty, two rows of padding.
        {"name": "prompt_short", "op": "prompt", **SMALL_HEADS, "dtype": "fp16", "seqs": 5, "lo": 0, "hi": 60, "mix": 8,
         "pad": 2},
        # A batch of prompts of ordinary, uneven lengths.
        {"name": "prompt_ragged", "op": "prompt", **MEDIUM_HEADS, "dtype": "bf16", "seqs": 16, "lo": 17, "hi": 1900,
         "mix": 5, "pad": 0},
        # One long document.
        {"name": "prompt_long", "op": "prompt", **SMALL_HEADS, "dtype": "fp16", "seqs": 1, "lo": 16001, "hi": 16001,
         "mix": 1, "pad": 0},
        # Single-stream decode at the package's own cache length: latency.
        {"name": "decode_single", "op": "paged", **SMALL_HEADS, "dtype": "fp16", "seqs": 1, "ctx_lo": 120, "ctx_hi": 120,
         "new_lo": 1, "new_hi": 1, "block": 16, "mix": 1, "pad": 0},
        # A server's decode batch, requests of very different lengths.
        {"name": "decode_batch", "op": "paged", **MEDIUM_HEADS, "dtype": "bf16", "seqs": 64, "ctx_lo": 100,
         "ctx_hi": 8191, "new_lo": 1, "new_hi": 1, "block": 16, "mix": 4, "pad": 0},
        # A few requests with very long contexts.
        {"name": "decode_long", "op": "paged", **LARGE_HEADS, "dtype": "bf16", "seqs": 3, "ctx_lo": 60001,
         "ctx_hi": 131071, "new_lo": 1, "new_hi": 1, "block": 64, "mix": 2, "pad": 0},
        # A long prompt worked off in chunks: one chunk of it over what is cached.
        {"name": "chunk_long", "op": "paged", **SMALL_HEADS, "dtype": "fp16", "seqs": 1, "ctx_lo": 29999,
         "ctx_hi": 29999, "new_lo": 2047, "new_hi": 2047, "block": 32, "mix": 1, "pad": 1},
        # A mixed batch: chunks of some prompts beside the single tokens of other requests.
        {"name": "chunk_mixed", "op": "paged", **LARGE_HEADS, "dtype": "bf16", "seqs": 24, "ctx_lo": 30, "ctx_hi": 4000,
         "new_lo": 1, "new_hi": 700, "block": 16, "mix": 9, "pad": 5},
        # The decode batch's new keys and values.
        {"name": "rope_decode", "op": "rope", **MEDIUM_HEADS, "dtype": "bf16", "tokens": 64, "pages": 600, "block": 16,
         "max_pos": 8192, "pad": 0},
        # The keys and values of packed prompts.
        {"name": "rope_prompt", "op": "rope", **SMALL_HEADS, "dtype": "fp16", "tokens": 8191, "pages": 700, "block": 16,
         "max_pos": 32768, "pad": 7},
        # A decode step's tables, and a step that admits many prompts.
        {"name": "tables_decode", "op": "tables", "seqs": 64, "ctx_lo": 100, "ctx_hi": 8191, "new_lo": 1, "new_hi": 1,
         "block": 16, "mix": 4, "pad": 0, "width": 513},
        {"name": "tables_admit", "op": "tables", "seqs": 500, "ctx_lo": 0, "ctx_hi": 2000, "new_lo": 0, "new_hi": 1500,
         "block": 16, "mix": 7, "pad": 100, "width": 260},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, count: int, lo: int, hi: int) -> list[int]:
    """Lengths spread over the logarithm of [lo, hi]; lo = 0 leaves about every sixth empty."""
    return [0 if lo == 0 and rng.random() < 0.17 else _log_int(rng, max(lo, 1), max(hi, 1)) for _ in range(count)]


def _case_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(context lengths, new lengths) of a case's requests."""
    rng = random.Random(case["mix"])
    if case["op"] == "prompt":
        return [0] * case["seqs"], _lengths(rng, case["seqs"], case["lo"], case["hi"])
    ctx = _lengths(rng, case["seqs"], case["ctx_lo"], case["ctx_hi"])
    return ctx, _lengths(rng, case["seqs"], case["new_lo"], case["new_hi"])


def work(case: dict) -> dict:
    if case["op"] == "rope":
        h, hk, d, t = case["heads"], case["kv_heads"], case["d"], case["tokens"]
        # q, k, v in; q, k out; k, v into the cache; fp32 cos and sin rows, positions and slots.
        return {"bytes": 2 * t * d * ((h + 2 * hk) + (h + hk) + 2 * hk) + 8 * t * d + 16 * t,
                "flops": 3 * t * d * (h + hk)}
    ctx, new = _case_lengths(case)
    total = sum(new)
    if case["op"] == "tables":
        bs = case["block"]
        pages = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        return {"bytes": 4 * (4 * len(ctx) + 1) + 8 * pages + 16 * (total + case["pad"]) + 8,
                "flops": 2 * len(ctx) + 4 * total}
    h, hk, d = case["heads"], case["kv_heads"], case["d"]
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    keys = sum(c + n for c, n in zip(ctx, new) if n)
    return {"bytes": 2 * d * (h * total + h * (total + case["pad"]) + 2 * hk * keys), "flops": 4 * d * h * pairs}


def draw(rng) -> dict:
    """One more case of the listed ones' ranges."""
    op = rng.choice(["prompt", "paged", "paged", "paged", "rope", "tables"])
    layout = dict(rng.choice(LAYOUTS))
    dtype = rng.choice(["fp16", "bf16"])
    block = rng.choice([16, 32, 64, 128])
    mix, pad = rng.randrange(1, 1000), rng.choice([0, 0, 1, 5, 33])
    if op == "rope":
        tokens = _log_int(rng, 1, 8191)
        return {"op": op, **layout, "dtype": dtype, "tokens": tokens, "block": block, "pad": min(pad, tokens - 1),
                "pages": -(-tokens // block) + rng.randrange(1, 200), "max_pos": _log_int(rng, 512, 32768)}
    while True:
        if op == "prompt":
            hi = _log_int(rng, 1, 16001)
            case = {"op": op, **layout, "dtype": dtype, "seqs": _log_int(rng, 1, 64), "lo": rng.choice([0, max(1, hi // 50)]),
                    "hi": hi, "mix": mix, "pad": pad}
        else:
            kind = rng.choice(["decode", "chunk", "mixed"])
            ctx_hi = _log_int(rng, 30, 131071 if op == "paged" else 8000)
            new_hi = 1 if kind == "decode" else _log_int(rng, 2, 2047)
            case = {"op": op, "dtype": dtype, "seqs": _log_int(rng, 1, 128 if op == "paged" else 500),
                    "ctx_lo": rng.choice([0, max(1, ctx_hi // 60)]), "ctx_hi": ctx_hi,
                    "new_lo": new_hi if kind == "decode" else rng.choice([0, 1, max(1, new_hi // 4)]), "new_hi": new_hi,
                    "block": block, "mix": mix, "pad": pad}
            if op == "paged":
                case.update(layout)
            else:
                case["width"] = -(-(ctx_hi + new_hi) // block) + rng.randrange(0, 9)
        if sum(_case_lengths(case)[1]) == 0:
            mix += 1
            continue
        w = work(case)
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES:
            return case


# ---- inputs -------------------------------------------------------------------------------------------


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _offsets(lens: list[int]) -> list[int]:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _ops():
    root = str(Path(__file__).resolve().parent.parent / "kernel-forge_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kernelforge import ops

    return ops


def _rope_tables(max_pos: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 [max_pos, d] cos and sin, the sign of the rotation folded into sin's first half."""
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    ang = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * inv
    cos, sin = ang.cos().float(), ang.sin().float()
    return torch.cat([cos, cos], 1), torch.cat([-sin, sin], 1)


def _block_table(ctx, new, block: int, width: int, g) -> tuple[torch.Tensor, torch.Tensor, int]:
    """(table [seqs, width] with the pages of the first ctx + new tokens, the pages left, pages in all):
    pages in random order, as a cache that has run for a while hands them out."""
    need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(ctx), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    return table, perm[at:], total


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    state = {"case": case}
    if own:
        state["ops"] = _ops()
    if case["op"] == "tables":
        ctx, new = _case_lengths(case)
        block, width = case["block"], case["width"]
        table, _, pages = _block_table(ctx, [0] * len(ctx), block, width, g)
        extra = sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(ctx, new)) + 11
        free = pages + torch.randperm(extra, generator=g, device=DEV).int()
        state.update(table=table, context_lens=_int32(ctx), new_lens=_int32(new), free_pages=free,
                     free_count=_int32([extra]), max_tokens=sum(new) + case["pad"])
        return state
    h, hk, d, dtype = case["heads"], case["kv_heads"], case["d"], _DTYPES[case["dtype"]]
    if case["op"] == "rope":
        t, block, pages = case["tokens"], case["block"], case["pages"]
        qkv = torch.randn(t, (h + 2 * hk) * d, generator=g, device=DEV).to(dtype)
        cos, sin = _rope_tables(case["max_pos"], d)
        positions = torch.randint(0, case["max_pos"], (t,), generator=g, device=DEV)
        slots = torch.randperm(pages * block, generator=g, device=DEV)[:t].clone()
        if case["pad"]:
            positions[t - case["pad"]:] = -1
            slots[t - case["pad"]:] = -1
        caches = [torch.randn(pages, hk, block, d, generator=g, device=DEV).to(dtype) for _ in range(2)]
        state.update(qkv=qkv, cos=cos, sin=sin, positions=positions, slots=slots, cache_k=caches[0], cache_v=caches[1])
        return state
    ctx, new = _case_lengths(case)
    offsets = _offsets(new)
    tokens = offsets[-1] + case["pad"]
    state.update(ctx=ctx, new=new, cu=_int32(offsets))
    if case["op"] == "prompt":
        # Views as the projection and RoPE leave them: q and k side by side, v inside q|k|v.
        qk = torch.randn(tokens, h + hk, d, generator=g, device=DEV).to(dtype)
        qkv = torch.randn(tokens, h + 2 * hk, d, generator=g, device=DEV).to(dtype)
        state.update(q=qk[:, :h], k=qk[:, h:], v=qkv[:, h + hk:])
        return state
    block = case["block"]
    width = max(-(-(c + n) // block) for c, n in zip(ctx, new)) + 1
    table, _, pages = _block_table(ctx, new, block, width, g)
    qk = torch.randn(tokens, h + hk, d, generator=g, device=DEV).to(dtype)
    cache_k = torch.empty(pages, hk, block, d, device=DEV, dtype=dtype)
    cache_v = torch.empty(pages, hk, block, d, device=DEV, dtype=dtype)
    for cache in (cache_k, cache_v):
        for a in range(0, pages, 4096):  # in pieces: the 32-bit draws need not fit twice
            piece = cache[a:a + 4096]
            piece.copy_(torch.randn(piece.shape, generator=g, device=DEV))
    state.update(q=qk[:, :h], cache_k=cache_k, cache_v=cache_v, table=table, max_new=max(new),
                 seq_lens=_int32([c + n for c, n in zip(ctx, new)]))
    return state


# ---- one pass -----------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return _run_own(state)
    return {"prompt": _plain_prompt, "paged": _plain_paged, "rope": _plain_rope, "tables": _plain_tables}[
        state["case"]["op"]](state)


def _run_own(s: dict):
    ops, op = s["ops"], s["case"]["op"]
    if op == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"])
    if op == "paged":
        return ops.paged_attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["cu"], s["seq_lens"],
                                   max_new=s["max_new"])
    if op == "rope":
        q, k = ops.rope_paged_cache(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["cache_k"],
                                    s["cache_v"], heads=s["case"]["heads"])
        return q, k, s["cache_k"], s["cache_v"]
    step = ops.paged_tables(s["table"], s["context_lens"], s["new_lens"], s["free_pages"], s["free_count"],
                            block_size=s["case"]["block"], max_tokens=s["max_tokens"])
    return (s["table"], step.cu_new, step.seq_lens, step.positions, step.slots, step.free_count)


def _plain_attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ctx: int) -> torch.Tensor:
    """q [n, heads, d] at positions ctx ..; k, v [kv_heads, ctx + n, d] in 32 bits: [n, heads, d] in q's type."""
    n, h, d = q.shape
    hk = k.shape[0]
    rep = h // hk
    out = torch.empty_like(q)
    step = max(1, (1 << 27) // (h * (ctx + n)))
    for a in range(0, n, step):
        b = min(a + step, n)
        rows = q[a:b].float().reshape(b - a, hk, rep, d).permute(1, 2, 0, 3).reshape(hk, rep * (b - a), d)
        keys = ctx + b
        s = torch.matmul(rows, k[:, :keys].transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(d))
        s = s.view(hk, rep, b - a, keys)
        limit = torch.arange(ctx + a, ctx + b, device=q.device)[:, None]
        s.masked_fill_(torch.arange(keys, device=q.device)[None, :] > limit, float("-inf"))
        s = (s - s.amax(-1, keepdim=True)).exp_()
        s /= s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(hk, rep * (b - a), keys), v[:, :keys])
        out[a:b] = o.view(hk, rep, b - a, d).permute(2, 0, 1, 3).reshape(b - a, h, d).to(q.dtype)
    return out


def _plain_prompt(s: dict):
    out = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    at = 0
    for n in s["new"]:
        if n:
            k, v = (s[name][at:at + n].float().transpose(0, 1).contiguous() for name in ("k", "v"))
            out[at:at + n] = _plain_attend(s["q"][at:at + n], k, v, 0)
            at += n
    return out


def _plain_paged(s: dict):
    out = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    block, hk, d = s["case"]["block"], s["case"]["kv_heads"], s["case"]["d"]
    at = 0
    for r, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        if n:
            pages = s["table"][r, :-(-(c + n) // block)].long()
            k, v = (s[name][pages].float().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :c + n]
                    for name in ("cache_k", "cache_v"))
            out[at:at + n] = _plain_attend(s["q"][at:at + n], k, v, c)
            at += n
    return out


def _plain_rope(s: dict):
    case = s["case"]
    h, hk, d, block = case["heads"], case["kv_heads"], case["d"], case["block"]
    t = case["tokens"]
    x = s["qkv"].float().view(t, h + 2 * hk, d)
    pos = s["positions"].clamp(min=0)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = x[:, :h + hk]
    qk = (qk * cos + torch.cat([qk[..., d // 2:], qk[..., :d // 2]], -1) * sin).to(s["qkv"].dtype)
    live = t - case["pad"]  # padding comes last
    page, offset = s["slots"][:live] // block, s["slots"][:live] % block
    s["cache_k"][page, :, offset] = qk[:live, h:]
    s["cache_v"][page, :, offset] = s["qkv"].view(t, h + 2 * hk, d)[:live, h + hk:]
    return qk[:, :h], qk[:, h:], s["cache_k"], s["cache_v"]


def _plain_tables(s: dict):
    block, max_tokens, table = s["case"]["block"], s["max_tokens"], s["table"]
    ctx, new = s["context_lens"].long(), s["new_lens"].long()
    seq = ctx + new
    held, need = (ctx + block - 1) // block, (seq + block - 1) // block
    first = torch.cumsum(need - held, 0) - (need - held)  # pages taken by the requests before
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    order = first[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    taken = s["free_pages"][(s["free_count"].long() - 1 - order).clamp(0, s["free_pages"].numel() - 1)]
    table.copy_(torch.where(fresh, torch.where(order < s["free_count"], taken, -1), table))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=table.device), torch.cumsum(new, 0)])
    token = torch.arange(max_tokens, device=table.device)
    row = (torch.searchsorted(cu, token, right=True) - 1).clamp(max=ctx.numel() - 1)
    live = token < cu[-1]
    pos = torch.where(live, ctx[row] + token - cu[row], -1)
    page = table[row, (pos // block).clamp(min=0)].long()
    slots = torch.where(live & (page >= 0), page * block + pos % block, -1)
    left = (s["free_count"] - (need - held).sum()).clamp(min=0).int()
    return table, cu.int(), seq.int(), pos, slots, left


# ---- from the definition, in 64 bits ------------------------------------------------------------------


def _exact_rows(q, keys, values, first: int) -> torch.Tensor:
    """One KV head: q [n, rep, d] at positions first .., keys and values [first + n, d], all 64 bits."""
    n, rep, d = q.shape
    out = torch.empty_like(q)
    step = max(1, (1 << 26) // (rep * keys.shape[0]))
    for a in range(0, n, step):
        b = min(a + step, n)
        score = (q[a:b].reshape(-1, d) @ keys.t()) / math.sqrt(d)
        pos = (first + torch.arange(a, b, device=q.device)).repeat_interleave(rep)
        score = torch.where(torch.arange(keys.shape[0], device=q.device) <= pos[:, None], score, -math.inf)
        prob = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
        out[a:b] = (prob @ values).view(b - a, rep, d)
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(s)
    h, hk, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "rope":
        t, block = case["tokens"], case["block"]
        x = s["qkv"].double().view(t, h + 2 * hk, d)
        rows = torch.where(s["positions"] < 0, 0, s["positions"])
        c, sn = s["cos"].double()[rows, None, :d // 2], s["sin"].double()[rows, None, d // 2:]
        lo, hi = x[:, :h + hk, :d // 2], x[:, :h + hk, d // 2:]
        qk = torch.cat([lo * c - hi * sn, hi * c + lo * sn], dim=2)
        caches = []
        for cache, src in ((s["cache_k"], qk[:, h:]), (s["cache_v"], x[:, h + hk:])):
            flat = cache.double().permute(0, 2, 1, 3).reshape(-1, hk, d)
            flat[s["slots"][s["slots"] >= 0]] = src[s["slots"] >= 0]
            caches.append(flat.view(-1, block, hk, d).permute(0, 2, 1, 3).contiguous())
        return qk[:, :h], qk[:, h:], caches[0], caches[1]
    rep = h // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    offsets = _offsets(s["new"])
    for r, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        if n == 0:
            continue
        a, b = offsets[r], offsets[r + 1]
        if case["op"] == "paged":
            index = torch.arange(c + n, device=DEV)
            page = s["table"][r].long()[index // case["block"]]
        for j in range(hk):
            if case["op"] == "paged":
                keys, values = (s[name][page, j, index % case["block"]].double() for name in ("cache_k", "cache_v"))
            else:
                keys, values = s["k"][a:b, j].double(), s["v"][a:b, j].double()
            out[a:b, j * rep:(j + 1) * rep] = _exact_rows(s["q"][a:b, j * rep:(j + 1) * rep].double(), keys, values, c)
    return out


def _exact_tables(s: dict):
    """Request by request and token by token on the host."""
    block = s["case"]["block"]
    table, free = s["table"].tolist(), s["free_pages"].tolist()
    ctx, new = s["context_lens"].tolist(), s["new_lens"].tolist()
    count = s["free_count"].item()
    positions, slots, cu = [], [], [0]
    for r, (c, n) in enumerate(zip(ctx, new)):
        for j in range(-(-c // block), -(-(c + n) // block)):
            count -= 1
            table[r][j] = free[count] if count >= 0 else -1
        for p in range(c, c + n):
            page = table[r][p // block]
            positions.append(p)
            slots.append(page * block + p % block if page >= 0 else -1)
        cu.append(len(positions))
    tail = [-1] * (s["max_tokens"] - len(positions))

    def whole(values):
        return torch.tensor(values, dtype=torch.int64, device=DEV)

    return (whole(table).int(), whole(cu).int(), whole([c + n for c, n in zip(ctx, new)]).int(), whole(positions + tail),
            whole(slots + tail), whole([max(count, 0)]).int())
