"""Calls of the attention over a cache at the edges of what it takes (needs a GPU)."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from attention_cases import attend64, check, offsets
from test_paged_attention_gpu import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("requests,tokens", [(512, 8192), (4096, 4096)])
def test_offsets_whose_work_passes_31_bits(requests, tokens):
    """Offsets 0, T, 0, T, .. that add up to more work than is counted: no work, and calls after it are as before."""
    cache = [torch.randn(3, 4, 16, 64, device=DEV).half() for _ in range(2)]
    table = i32([0] * 8192).expand(requests, 8192)
    q = torch.randn(tokens, 32, 64, device=DEV).half()
    lens = i32([131072] * requests)
    right = dict(block_table=i32([[1, 2]]), cu_new=i32([0, 1]), seq_lens=i32([20]))
    want = ops.paged_attention(q[:1], *cache, **right)
    ops.paged_attention(q, *cache, table, i32([0, tokens] * (requests // 2) + [0]), lens, max_new=1)
    torch.cuda.synchronize()
    assert torch.equal(ops.paged_attention(q[:1], *cache, **right), want)


def test_long_chunks_over_wide_tables():
    """Two chunks of 2048 tokens in tables of 2^20 tokens: more rows x keys than the kernel of few rows takes, which
    gets none of them."""
    heads, kv_heads, d, n, block = 1024, 8, 8, 2048, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    pages = 2 * n // block
    k, v = (torch.randn(pages, kv_heads, block, d, generator=g, device=DEV).half() for _ in range(2))
    table = torch.full((2, (1 << 20) // block), -1, dtype=torch.int32, device=DEV)
    table[:, :n // block] = torch.arange(pages, device=DEV).view(2, -1)
    q = torch.randn(2 * n, heads, d, generator=g, device=DEV).half()
    out = ops.paged_attention(q, k, v, table, offsets([n, n], DEV), i32([n, n]), max_new=n)
    some = torch.arange(0, heads, heads // kv_heads, device=DEV)  # a query head of each KV head
    for r in range(2):
        rows = slice(r * n, (r + 1) * n)
        keys, values = (c[table[r, :n // block].long()].transpose(1, 2).reshape(n, kv_heads, d) for c in (k, v))
        ref, bound = attend64(q[rows][:, some], keys, values)
        check(out[rows][:, some], ref, bound, f"request {r}")


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (4, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("ctx,new,width", [([60, 64, 70, 3], [1, 1, 1, 1], 4), ([60, 0, 40, 10], [8, 90, 30, 1], 4),
                                           ([3, 300, 0, 100], [200, 5, 700, 300], 16), ([5000, 30], [300, 1], 320),
                                           ([300, 0, 20] * 8, [80, 300, 1] * 8, 20), ([2500], [100], 160)],
                         ids=["single", "short", "chunks", "long", "both", "cut"])
def test_tables_that_are_too_narrow(heads, kv_heads, d, ctx, new, width):
    """Requests that pass their table's width: new tokens keep their positions and attend to the keys that have a
    place, as single tokens, in chunks and in both kinds of cut items."""
    b = Batch(ctx, new, heads, kv_heads, d, torch.float16, 16, pad=2)
    b.table = b.table[:, :width]
    there = [torch.arange(c + n, device=DEV) < 16 * width for c, n in zip(ctx, new)]
    assert not all(bool(t.all()) for t in there)
    b.check(b(max_new=max(new)), there)
    b.check(b(), there)


@pytest.mark.parametrize("d", [64, 128])
def test_a_cut_prompt_far_past_its_table(d):
    """Row tiles whose keys end with the table while their number goes on: pieces without a key."""
    b = Batch([0], [9000], 1, 1, d, torch.bfloat16, 16)
    b.table = b.table[:, :250]
    b.check(b(max_new=9000), [torch.arange(9000, device=DEV) < 4000])


def test_a_step_that_passes_its_table():
    """paged_tables gives such tokens no slot, rope_paged_cache leaves the cache, and paged_attention attends to the rest."""
    heads, kv_heads, d, block = 4, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(9)
    caches = [torch.randn(9, kv_heads, block, d, generator=g, device=DEV).half() for _ in range(2)]
    table = i32([[5, 2, 7, -1], [1, -1, -1, -1]])
    step = ops.paged_tables(table, i32([45, 10]), i32([30, 2]), i32([0, 8, 3]), i32([3]), block_size=block, max_tokens=32)
    qkv = torch.randn(32, (heads + 2 * kv_heads) * d, generator=g, device=DEV).half()
    cos, sin = (torch.rand(128, d, generator=g, device=DEV) for _ in range(2))
    q, _ = ops.rope_paged_cache(qkv, cos, sin, step.positions, step.slots, *caches, heads=heads)
    out = ops.paged_attention(q, *caches, table, step.cu_new, step.seq_lens, max_new=30)
    assert table.tolist() == [[5, 2, 7, 3], [1, -1, -1, -1]]
    for r, (rows, n) in enumerate(((slice(0, 30), 75), (slice(30, 32), 12))):
        pages = table[r][table[r] >= 0].long()
        k, v = (torch.cat([c[pages].transpose(1, 2).reshape(-1, kv_heads, d), c.new_zeros(32, kv_heads, d)])[:n] for c in caches)
        ref, bound = attend64(q[rows], k, v, torch.arange(n, device=DEV) < 16 * pages.numel())
        check(out[rows], ref, bound, f"request {r}")


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 4, 64), (12, 2, 128), (8, 8, 96), (4, 1, 256), (16, 1, 80)])
@pytest.mark.parametrize("ctx,new", [([0, 17, 130, 400], [1, 1, 1, 1]), ([40] * 70, [1] * 70), ([0], [300]), ([900, 3], [33, 1]),
                                     ([0, 70, 500], [0, 260, 2]), ([100] * 12, [1, 200, 1, 9] * 3), ([5], [1])],
                         ids=["decode", "many", "prompt", "short", "chunk", "mixed", "one"])
def test_tables_much_wider_than_the_requests(heads, kv_heads, d, ctx, new):
    """A server's table is as wide as its longest request may get, and the plans go by its width."""
    b = Batch(ctx, new, heads, kv_heads, d, torch.bfloat16, 16, pad=1, extra_width=6000)
    b.check(b(max_new=max(new)))
    b.check(b())
