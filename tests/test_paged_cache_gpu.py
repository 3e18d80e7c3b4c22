"""Tables and writer of the paged cache (needs a GPU): tables against a token-by-token construction on the host,
RoPE and the cache's update against float64, and the operators in a row as a server calls them."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from attention_cases import HALF_STEP, attend64, check

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def tables_on_host(table, ctx, new, free, count, block, max_tokens):
    table = [list(row) for row in table]
    width = len(table[0])
    pos, slots, cu = [], [], [0]
    for r, (c, n) in enumerate(zip(ctx, new)):
        n = max(n, 0)
        for j in range(-(-c // block), min(-(-(c + n) // block), width)):
            count -= 1
            table[r][j] = free[count] if count >= 0 else -1
        for p in range(c, c + n):
            page = table[r][p // block] if p // block < width else -1
            pos.append(p)
            slots.append(page * block + p % block if page >= 0 else -1)
        cu.append(len(pos))
    fill = [-1] * (max_tokens - len(pos))
    return (table, cu, [c + max(n, 0) for c, n in zip(ctx, new)], (pos + fill)[:max_tokens], (slots + fill)[:max_tokens],
            [max(count, 0)])


@pytest.mark.parametrize("ctx,new,block,width,free,slack", [
    ([0], [1], 16, 1, 5, 0), ([15, 16, 17, 0], [1, 1, 1, 1], 16, 3, 10, 4), ([0] * 3, [0] * 3, 32, 2, 0, 7),
    ([100, 0, 33, 64], [0, 50, 500, 64], 16, 40, 60, 100), ([10, 20], [100, 100], 16, 8, 3, 0),  # the stack runs dry
    ([60], [20], 16, 4, 9, 0),                                                             # past the table's width
    ([5, 0, 7], [-3, 2, 1], 64, 2, 4, 1), (list(range(300)), [1 + i % 40 for i in range(300)], 16, 25, 2000, 33),
    ([0], [9001], 128, 80, 100, 1), ([7], [30], 16, 6, 8, -9),                              # fewer rows than tokens
])
def test_tables(ctx, new, block, width, free, slack):
    g = torch.Generator().manual_seed(len(ctx) + block)
    perm = torch.randperm(width * len(ctx) + free, generator=g).tolist()
    table = [[-1] * width for _ in ctx]
    for r, c in enumerate(ctx):
        for j in range(-(-c // block)):
            table[r][j] = perm.pop()
    stack = [perm.pop() for _ in range(free)] + [-9] * 3  # what lies above the top is not taken
    max_tokens = max(sum(max(n, 0) for n in new) + slack, 0)
    want = tables_on_host(table, ctx, new, stack, free, block, max_tokens)
    dt = i32(table)
    for _ in range(2):  # again: the same pages, as the stack is not changed
        step = ops.paged_tables(dt, i32(ctx), i32(new), i32(stack), i32([free]), block_size=block, max_tokens=max_tokens)
        got = (dt, step.cu_new, step.seq_lens, step.positions, step.slots, step.free_count)
        for a, b in zip(got, want):
            assert a.tolist() == b


def test_tables_wrong_counts_stay_inside():
    table = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    big = 2 ** 31 - 1
    for ctx, new, count in (([0, 0], [big, big], 5), ([big, 3], [big, 5], 99), ([0, 1], [20, 1], -3)):
        step = ops.paged_tables(table, i32(ctx), i32(new), i32([1, 2, 3]), i32([count]), block_size=16, max_tokens=50)
        assert bool((table <= 3).all()) and bool((step.slots < 64).all()) and int(step.free_count) in (0, 1, 2, 3)


def rope64(qkv, cos, sin, pos, heads, kv_heads, d):
    x = qkv.double().view(-1, heads + 2 * kv_heads, d)[:, :heads + kv_heads]
    p = torch.where((pos >= 0) & (pos < cos.shape[0]), pos, 0)
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    swapped = torch.cat([x[..., d // 2:], x[..., :d // 2]], -1)
    return x * c + swapped * s, (x * c).abs() + (swapped * s).abs()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,block", [(32, 4, 64, 16), (12, 2, 128, 32), (8, 8, 96, 16), (3, 1, 8, 64),
                                                    (2, 2, 40, 16), (1, 1, 256, 128)])
@pytest.mark.parametrize("t", [1, 3, 130])
def test_rope_and_cache(dtype, heads, kv_heads, d, block, t):
    g = torch.Generator(device=DEV).manual_seed(t + d)
    qkv = torch.randn(t, (heads + 2 * kv_heads) * d, generator=g, device=DEV).to(dtype)
    cos, sin = (torch.rand(50, d, generator=g, device=DEV) * 2 - 1 for _ in range(2))
    pages = -(-t // block) + 3
    slots = torch.randperm(pages * block, generator=g, device=DEV)[:t].clone()
    pos = torch.randint(0, 50, (t,), generator=g, device=DEV)
    if t > 2:
        slots[1], pos[2] = -1, 50  # no slot; a position past the tables
    if t > 100:
        slots[100], pos[101] = pages * block, -1
    caches = [torch.randn(pages, kv_heads, block, d, generator=g, device=DEV).to(dtype) for _ in range(2)]
    before = [c.clone() for c in caches]
    q, k = ops.rope_paged_cache(qkv, cos, sin, pos, slots, *caches, heads=heads)
    ref, mag = rope64(qkv, cos, sin, pos, heads, kv_heads, d)
    got = torch.cat([q, k], 1).double()
    # Two products and a sum in 32 bits, then half a step of the type.
    assert bool(((got - ref).abs() <= 2 * 2.0 ** -24 * mag + HALF_STEP[dtype] * ref.abs() + 2.0 ** -25).all())
    live = (slots >= 0) & (slots < pages * block) & (pos >= 0) & (pos < 50)
    for cache, want, src in zip(caches, before, (k, qkv.view(t, -1, d)[:, heads + kv_heads:])):
        want[slots[live] // block, :, slots[live] % block] = src[live]
        assert torch.equal(cache, want)


def test_rope_strides_and_layouts():
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = torch.randn(20, 8 * 64 + 24, generator=g, device=DEV).half()
    cos, sin = (torch.rand(64, 64, generator=g, device=DEV) for _ in range(2))
    pos, slots = torch.arange(20, device=DEV), torch.arange(20, device=DEV) + 5
    want = [torch.zeros(3, 2, 16, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    q, k = ops.rope_paged_cache(wide[:, :512].contiguous(), cos, sin, pos, slots, *want, heads=4)
    got = [torch.zeros(3, 16, 2, 64, dtype=torch.float16, device=DEV).transpose(1, 2) for _ in range(2)]
    q2, k2 = ops.rope_paged_cache(wide[:, :512], cos, sin, pos, slots, *got, heads=4)
    assert torch.equal(q, q2) and torch.equal(k, k2) and all(torch.equal(a, b) for a, b in zip(got, want))
    got = [torch.zeros(3, 2, 16, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    odd = torch.zeros(20 * 512 + 5, dtype=torch.float16, device=DEV)[5:].view(20, 512)
    odd.copy_(wide[:, :512])
    q2, k2 = ops.rope_paged_cache(odd, cos, sin, pos, slots, *got, heads=4)
    assert torch.equal(q, q2) and torch.equal(k, k2) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_served_steps():
    """Prompts of different lengths, a chunk, then single tokens, with a request that pauses: each step's attention
    against the whole history of every request in 64 bits; a prompt step the same from both attentions."""
    heads, kv_heads, d, block, b, width = 8, 2, 64, 16, 4, 20
    g = torch.Generator(device=DEV).manual_seed(11)
    pages = 50
    caches = [torch.full((pages, kv_heads, block, d), float("nan"), device=DEV).half() for _ in range(2)]
    table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
    free, count = torch.randperm(pages, generator=g, device=DEV).int(), i32([pages])
    ang = torch.arange(512, device=DEV)[:, None] * 0.01 * torch.arange(1, d // 2 + 1, device=DEV)
    cos, sin = torch.cat([ang.cos()] * 2, 1), torch.cat([-ang.sin(), ang.sin()], 1)
    ctx = i32([0] * b)
    history = [[torch.empty(0, kv_heads, d, device=DEV).half()] * 2 for _ in range(b)]
    for new in ([37, 16, 5, 100], [1, 1, 60, 1], [1, 0, 1, 1], [1, 1, 1, 1], [2, 3, 1, 40]):
        max_tokens = sum(new) + 2
        step = ops.paged_tables(table, ctx, i32(new), free, count, block_size=block, max_tokens=max_tokens)
        qkv = torch.randn(max_tokens, (heads + 2 * kv_heads) * d, generator=g, device=DEV).half()
        q, k = ops.rope_paged_cache(qkv, cos, sin, step.positions, step.slots, *caches, heads=heads)
        v = qkv.view(max_tokens, -1, d)[:, heads + kv_heads:]
        out = ops.paged_attention(q, *caches, table, step.cu_new, step.seq_lens, max_new=max(new))
        at = 0
        for r, n in enumerate(new):
            history[r] = [torch.cat([history[r][0], k[at:at + n]]), torch.cat([history[r][1], v[at:at + n]])]
            if n:
                ref, bound = attend64(q[at:at + n], *history[r])
                check(out[at:at + n], ref, bound, f"request {r}, {n} new")
                if int(ctx[r]) == 0:
                    one = torch.zeros(max_tokens, heads, d, device=DEV).half()
                    ops.prompt_attention(q, k, v, step.cu_new, out=one)
                    check(one[at:at + n], ref, bound, "prompt")
            at += n
        assert bool((out[at:] == 0).all())
        ctx, count = step.seq_lens, step.free_count
    used = sum(-(-int(n) // block) for n in ctx.tolist())
    assert int(count) == pages - used
