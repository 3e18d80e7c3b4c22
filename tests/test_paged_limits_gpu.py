"""Calls of the attention over a cache at the edges of what it takes (needs a GPU)."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from attention_cases import attend64, check, offsets

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
