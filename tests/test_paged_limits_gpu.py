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
