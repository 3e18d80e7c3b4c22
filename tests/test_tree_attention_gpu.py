"""Attention of drafted trees over a paged cache against float64 (needs a GPU): trees and any other words, at the edges of pages,
tiles and splits; keys that nobody sees; caches and queries of other layouts."""

from __future__ import annotations

import random

import pytest
import torch

from kernelforge import ops

from attention_cases import check
from draft_cases import ancestors_of, chain, random_trees, tree64
from test_paged_attention_gpu import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYOUTS = [(32, 4, 64), (12, 2, 128), (8, 8, 96), (16, 1, 80), (4, 2, 256), (3, 3, 8), (40, 1, 64), (24, 1, 200)]
DTYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])


class Trees(Batch):
    def __init__(self, ctx, new, *args, words=None, pad=0, **kw):
        super().__init__(ctx, new, *args, pad=pad, **kw)
        self.words = words or [ancestors_of(t) for t in random_trees(new, len(ctx) + sum(new))]
        self.ancestors = torch.tensor([w for tree in self.words for w in tree] + [-1] * pad, dtype=torch.int64, device=DEV)

    def __call__(self, **kw):
        return ops.paged_tree_attention(self.q, self.cache_k, self.cache_v, self.table, self.cu, self.seq_lens, self.ancestors,
                                        **kw)

    def check(self, out, there=None):
        at, worst = 0, 0.0
        for r, n in enumerate(self.new):
            if n:
                ref, bound = tree64(self.q[at:at + n], self.k[r], self.v[r], self.words[r], None if there is None else there[r])
                worst = max(worst, check(out[at:at + n], ref, bound, f"request {r}"))
            at += n
        assert bool((out[at:] == 0).all())
        return worst


@DTYPES
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("block", [16, 64])
def test_small_trees(dtype, heads, kv_heads, d, block):
    b = Trees([0, 1, 15, 16, 31, 127, 128, 500, 1025], [3, 1, 2, 7, 1, 4, 8, 5, 2], heads, kv_heads, d, dtype, block, pad=2)
    b.check(b(max_new=8))


@DTYPES
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("block", [16, 128])
def test_large_and_small_trees(dtype, heads, kv_heads, d, block):
    b = Trees([0, 70, 300, 5, 640, 33], [64, 1, 17, 0, 3, 63], heads, kv_heads, d, dtype, block, pad=3)
    b.check(b(max_new=64))
    assert torch.equal(b(), b())


@pytest.mark.parametrize("ctx,new", [([20000], [9]), ([20000], [64]), ([9000, 3], [20, 64]), ([0], [64]), ([5000] * 3, [2] * 3),
                                     ([40] * 300, [5] * 300), ([700] * 40, [64] * 40), ([3000, 0, 17], [1, 60, 2])],
                         ids=["long", "long_wide", "uneven", "new", "few", "many", "many_wide", "both"])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (16, 2, 128)])
def test_lengths(ctx, new, heads, kv_heads, d):
    b = Trees(ctx, new, heads, kv_heads, d, torch.float16, 16)
    b.check(b(max_new=max(new)))


@DTYPES
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
def test_wide_tables(dtype, heads, kv_heads, d):
    """Tables that long requests would fill: row tiles are cut into pieces, most of short requests' into one."""
    b = Trees([0, 70, 3000, 5, 640, 1], [64, 1, 17, 0, 30, 63], heads, kv_heads, d, dtype, 16, pad=3, extra_width=90)
    b.check(b(max_new=64))
    b.check(b())
    assert torch.equal(b(), b(max_new=64))


@pytest.mark.parametrize("requests,new", [(65, 8), (100, 20), (300, 3), (1000, 2)])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (16, 2, 128), (2, 1, 256)])
def test_more_requests_than_lanes(requests, new, heads, kv_heads, d):
    """With and without pieces; the requests' pieces are counted by one wavefront, a run of requests a lane."""
    rng = random.Random(requests)
    ctx = [rng.choice([0, 3, 40, 200, 1500 if requests < 300 else 90]) for _ in range(requests)]
    lens = [rng.randrange(0, new + 1) for _ in range(requests)]
    b = Trees(ctx, lens, heads, kv_heads, d, torch.float16, 16, pad=2, extra_width=70)
    out = b(max_new=max(lens))
    at = 0
    assert bool((out[sum(lens):] == 0).all())
    for r, n in enumerate(lens):
        if n and r % (1 + requests // 60) == 0:  # a sample of them against 64 bits
            ref, bound = tree64(b.q[at:at + n], b.k[r], b.v[r], b.words[r])
            check(out[at:at + n], ref, bound, f"request {r}")
        at += n


@DTYPES
@pytest.mark.parametrize("ctx", [[0, 1, 61, 300], [64, 128, 1000, 4000]])
def test_any_words(dtype, ctx):
    """Words that are no tree's: later tokens, none at all, bits past the new tokens."""
    rng = random.Random(sum(ctx))
    new = [64, 9, 40, 1]
    words = [[rng.getrandbits(64) & rng.getrandbits(64) for _ in range(n)] for n in new]
    words[0][3] = words[1][0] = words[2][39] = 0
    words[3][0] = (1 << 64) - 2  # all but its own
    words = [[w - (1 << 64) if w >> 63 else w for w in tree] for tree in words]
    for heads, kv_heads, d in ((8, 2, 64), (6, 2, 128), (2, 1, 256)):
        b = Trees(ctx, new, heads, kv_heads, d, dtype, 16, words=words)
        out = b(max_new=64)
        b.check(out)
        if ctx[0] == 0:
            assert bool((out[3] == 0).all())  # no token in the cache and no bit: zeros
        elif ctx[3] == 0:
            assert bool((out[-1] == 0).all())


@DTYPES
def test_more_new_tokens_than_words_have_bits(dtype):
    """Tokens past the 64th see the cached ones and what their words say; nobody sees them."""
    new = [70, 130]
    words = [ancestors_of(chain(n)) for n in new]
    words[0][66] = words[1][64] = 5
    b = Trees([100, 7], new, 8, 2, 64, dtype, 16, words=words)
    b.check(b(max_new=130))
    b.check(b(max_new=64))  # a hint that is too small costs time, never rows
    b.check(b())


@DTYPES
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (32, 2, 128), (2, 1, 200)])
def test_a_chain_is_paged_attention(dtype, heads, kv_heads, d):
    ctx, new = [0, 30, 500, 77], [5, 33, 64, 1]
    b = Trees(ctx, new, heads, kv_heads, d, dtype, 32, words=[ancestors_of(chain(n)) for n in new])
    Batch.check(b, b(max_new=64))


@DTYPES
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads,kv_heads,d,ctx,more", [(8, 2, 64, 40, 2), (32, 2, 128, 300, 2), (32, 2, 64, 20, 2), (4, 2, 256, 90, 2),
                                                       (2, 2, 128, 50, 2), (8, 2, 64, 900, 2), (32, 2, 128, 1400, 2),
                                                       (4, 2, 256, 800, 2), (32, 2, 64, 30, 80)])
def test_keys_and_values_that_are_not_finite(dtype, bad, heads, kv_heads, d, ctx, more):
    """In nodes beside a row's own branch they do not reach it; values in its branch do."""
    parents = [-1, 0, 0, 1, 2, 3, 4, 5]
    b = Trees([ctx, ctx + 7], [8, 8], heads, kv_heads, d, dtype, 16, words=[ancestors_of(parents)] * 2,
              extra_width=more)
    clean = b(max_new=8)
    b.check(clean)
    node = ctx + 3  # seen by nodes 3, 5 and 7
    page, at = int(b.table[0, node // 16]), node % 16
    b.cache_k[page, :, at] = bad
    b.cache_v[page, :, at, ::3] = bad
    out = b(max_new=8)
    others = [0, 1, 2, 4, 6, *range(8, 16)]
    assert torch.equal(out[others], clean[others])
    b.cache_k[page, :, at] = b.k[0][node]
    out = b(max_new=8)
    assert torch.equal(out[others], clean[others])
    for row in (3, 5, 7):
        hit = out[row, :, ::3]
        assert bool((hit.isnan() if bad != bad else hit == bad).all())
        rest = torch.ones(d, dtype=torch.bool, device=DEV)
        rest[::3] = False
        assert torch.equal(out[row][:, rest], clean[row][:, rest])


def test_pages_that_are_not_there():
    for ctx, new in (([200, 64, 10], [3, 2, 1]), ([200, 0, 10], [64, 50, 6])):
        b = Trees(ctx, new, 8, 2, 128, torch.bfloat16, 16)
        there = [torch.ones(c + n, dtype=torch.bool, device=DEV) for c, n in zip(ctx, new)]
        for r, page, value in ((0, 0, -1), (0, 5, 1 << 30), (0, 12, b.cache_k.shape[0]), (2, 0, -7)):
            b.table[r, page] = value
            there[r][16 * page:16 * page + 16] = False
        out = b(max_new=max(new))
        b.check(out, there)


def test_tables_that_are_too_narrow():
    """Tokens behind the table's last page are not attended to, drafted ones among them."""
    b = Trees([60, 20], [30, 5], 8, 2, 64, torch.float16, 16, extra_width=0)
    there = [torch.arange(90, device=DEV) < 64, torch.arange(25, device=DEV) < 64]
    b.table = b.table[:, :4].contiguous()
    b.check(b(max_new=30), there)


def test_lengths_that_do_not_fit_stay_inside():
    b = Trees([50, 20], [1, 1], 4, 2, 64, torch.float16, 16)
    b.seq_lens.copy_(torch.tensor([1 << 30, -5]))
    out = b(max_new=1)
    assert bool((out[1] == 0).all())
    for more in (2, 80):
        b = Trees([50, 20], [40, 40], 4, 2, 64, torch.float16, 16, words=[ancestors_of(chain(40))] * 2, extra_width=more)
        b.seq_lens.copy_(torch.tensor([3, 0]))  # fewer keys than new tokens: the first ones have none
        out = b()
        assert bool((out[:37] == 0).all()) and bool(out[37:40].isfinite().all()) and bool((out[40:] == 0).all())
        for cu in ([0, 1 << 30, -4], [70, 3, 80], [80, 80, 80]):
            b.cu.copy_(torch.tensor(cu))
            b()
            b.seq_lens.copy_(torch.tensor([1 << 30, 1 << 29]))
            b()
    many = Trees([0] * 60, [1] * 60, 4, 2, 64, torch.float16, 16, extra_width=80)  # offsets that go up and down
    many.cu.copy_(torch.tensor([0 if i % 2 == 0 else 60 for i in range(61)]))
    many()
    torch.cuda.synchronize()


def test_out_strides_and_streams():
    b = Trees([33, 200, 5], [10, 64, 2], 8, 2, 64, torch.float16, 16, pad=4)
    want = b(max_new=64)
    b.check(want)
    whole = torch.full((sum(b.new) + 4, 8, 72), 7.0, dtype=torch.float16, device=DEV)
    assert b(max_new=64, out=whole[..., :64]).data_ptr() == whole.data_ptr()
    assert torch.equal(whole[:76, :, :64], want[:76]) and bool((whole[76:] == 7).all()) and bool((whole[..., 64:] == 7).all())
    # Queries and caches with strides of their own, and another stream.
    wide = torch.zeros(b.q.shape[0], 2, 8, 64, dtype=torch.float16, device=DEV)
    wide[:, 1] = b.q
    keys = torch.zeros(b.cache_k.shape[0], 16, 2, 2, 64, dtype=torch.float16, device=DEV).permute(2, 0, 3, 1, 4)
    keys[0], keys[1] = b.cache_k, b.cache_v
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_tree_attention(wide[:, 1], keys[0], keys[1], b.table, b.cu, b.seq_lens, b.ancestors, max_new=64)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    scale = 1.0 / 64 ** 0.5
    assert torch.equal(torch.ops.kernelforge.paged_tree_attention(b.q, b.cache_k, b.cache_v, b.table, b.cu, b.seq_lens,
                                                                  b.ancestors, 64, scale), want)


@pytest.mark.parametrize("ctx,new", [([33, 200, 5], [10, 64, 2]), ([9000, 3000], [20, 64]), ([300], [4])])
def test_captured(ctx, new):
    """Replays follow lengths, words and caches; two graphs on the same inputs have workspaces of their own."""
    b = Trees(ctx, new, 8, 2, 64, torch.float16, 16)
    b(max_new=64)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(b(max_new=64))
        graphs.append(graph)
    for turn in range(3):
        b.q.mul_(-0.5)
        b.ancestors.copy_(torch.tensor([w & ~turn for w in b.ancestors.tolist()]))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = b(max_new=64)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@DTYPES
@pytest.mark.parametrize("ctx", [[64, 128, 300, 0], [64, 128, 1000, 0]], ids=["whole", "cut"])
def test_a_single_node_whose_word_lacks_its_own_bit(dtype, ctx):
    """All bits but its own, and no token in the cache: nothing is left to attend to."""
    new = [64, 9, 40, 1]
    words = [ancestors_of(t) for t in random_trees(new[:3], 7)] + [[-2]]
    for heads, kv_heads, d in ((8, 2, 64), (6, 2, 128), (2, 1, 256)):
        for max_new in (64, 1):
            b = Trees(ctx, new, heads, kv_heads, d, dtype, 16, words=words)
            out = b(max_new=max_new)
            b.check(out)
            assert bool((out[-1] == 0).all())


@DTYPES
def test_many_requests_beside_a_long_one(dtype):
    """More row tiles than workgroups that the card holds, of very different lengths."""
    rng = random.Random(8)
    ctx = [rng.choice([0, 17, 100, 400]) for _ in range(63)] + [20000]
    rng.shuffle(ctx)
    new = [rng.randrange(1, 17) for _ in ctx]
    b = Trees(ctx, new, 32, 8, 128, dtype, 16, pad=2)
    out = b(max_new=16)
    assert torch.equal(b(max_new=16), out)
    b.check(out)
