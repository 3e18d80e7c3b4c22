"""Attention of new tokens over a paged cache against float64 (needs a GPU): single tokens, chunks and both in one
batch; lengths at the edges of pages, tiles and splits; pages that are not there; caches of other layouts."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from attention_cases import attend64, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Batch:
    """Requests of ctx[r] + new[r] tokens over shuffled pages; unused slots hold NaN."""

    def __init__(self, ctx, new, heads, kv_heads, d, dtype, block, pad=0, extra_width=2, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed + heads + d + block + sum(ctx))
        self.ctx, self.new, self.block = ctx, new, block
        need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
        pages = sum(need) + 2
        perm = torch.randperm(pages, generator=g, device=DEV).int()
        self.table = torch.full((len(ctx), max(need) + extra_width), -1, dtype=torch.int32, device=DEV)
        self.cache_k = torch.full((pages, kv_heads, block, d), float("nan"), dtype=dtype, device=DEV)
        self.cache_v = self.cache_k.clone()
        self.k, self.v = [], []
        at = 0
        for r, (c, n) in enumerate(zip(ctx, new)):
            self.table[r, :need[r]] = perm[at:at + need[r]]
            at += need[r]
            k, v = (torch.randn(c + n, kv_heads, d, generator=g, device=DEV).to(dtype) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            i = torch.arange(c + n, device=DEV)
            page = self.table[r].long()[i // block]
            self.cache_k[page, :, i % block] = k
            self.cache_v[page, :, i % block] = v
        self.q = torch.randn(sum(new) + pad, heads, d, generator=g, device=DEV).to(dtype)
        self.cu = offsets(new, DEV)
        self.seq_lens = torch.tensor([c + n for c, n in zip(ctx, new)], dtype=torch.int32, device=DEV)

    def __call__(self, **kw):
        return ops.paged_attention(self.q, self.cache_k, self.cache_v, self.table, self.cu, self.seq_lens, **kw)

    def check(self, out, there=None):
        at, worst = 0, 0.0
        for r, n in enumerate(self.new):
            if n:
                ref, bound = attend64(self.q[at:at + n], self.k[r], self.v[r], None if there is None else there[r])
                worst = max(worst, check(out[at:at + n], ref, bound, f"request {r}"))
            at += n
        assert bool((out[at:] == 0).all())
        return worst


LAYOUTS = [(32, 4, 64), (12, 2, 128), (8, 8, 96), (16, 1, 80), (4, 2, 256), (3, 3, 8), (40, 1, 64), (24, 1, 200)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("block", [16, 64])
def test_decode(dtype, heads, kv_heads, d, block):
    b = Batch([0, 1, 15, 16, 31, 127, 128, 500, 1025], [1] * 9, heads, kv_heads, d, dtype, block, pad=2)
    b.check(b(max_new=1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("block", [16, 128])
def test_mixed(dtype, heads, kv_heads, d, block):
    b = Batch([0, 70, 300, 5, 640, 33], [130, 1, 17, 0, 3, 64], heads, kv_heads, d, dtype, block, pad=3)
    b.check(b(max_new=130))
    assert torch.equal(b(), b(max_new=130))


@pytest.mark.parametrize("ctx,new", [([20000], [1]), ([9000, 3], [1, 1]), ([4000], [300]), ([0], [777]), ([5000] * 3, [2] * 3),
                                     ([40] * 300, [1] * 300), ([3000, 0, 17], [1, 900, 2])],
                         ids=["long", "uneven", "chunk", "prompt", "few", "many", "both"])
def test_lengths(ctx, new):
    b = Batch(ctx, new, 8, 2, 64, torch.float16, 16)
    b.check(b(max_new=max(new)))


def test_hint_only_chooses_kernels():
    """A hint that is too small costs time, never rows."""
    b = Batch([100, 40], [90, 1], 8, 2, 64, torch.float16, 16)
    b.check(b(max_new=1))


def test_pages_that_are_not_there():
    """Holes in a table: their keys are not attended to, whatever number stands there; rows without any key are zeros."""
    for ctx, new in (([200, 64, 10], [1, 1, 1]), ([200, 0, 10], [100, 90, 6])):
        b = Batch(ctx, new, 8, 2, 128, torch.bfloat16, 16)
        there = [torch.ones(c + n, dtype=torch.bool, device=DEV) for c, n in zip(ctx, new)]
        for r, page, value in ((0, 0, -1), (0, 5, 1 << 30), (0, 12, b.cache_k.shape[0]), (2, 0, -7)):
            b.table[r, page] = value
            there[r][16 * page:16 * page + 16] = False
        out = b(max_new=max(new))
        b.check(out, there)
        assert bool((out[int(b.cu[2])] == 0).all()) or bool(there[2][:11].any())


def test_lengths_that_do_not_fit_stay_inside():
    """Wrong lengths and offsets give some result, from inside the arrays."""
    b = Batch([50, 20], [1, 1], 4, 2, 64, torch.float16, 16)
    b.seq_lens.copy_(torch.tensor([1 << 30, -5]))
    out = b(max_new=1)
    assert bool((out[1] == 0).all())
    b = Batch([50, 20], [40, 40], 4, 2, 64, torch.float16, 16)
    b.seq_lens.copy_(torch.tensor([3, 0]))  # fewer keys than new tokens: the first rows have none
    out = b()
    assert bool((out[:37] == 0).all()) and bool(out[37:40].isfinite().all()) and bool((out[40:] == 0).all())
    b.cu.copy_(torch.tensor([0, 1 << 30, -4]))
    b()
    torch.cuda.synchronize()


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_later_and_unused_slots_do_not_reach_a_row(new, bad):
    """Slots behind a request's last token hold NaN in every test here; a later token's value does not reach
    the rows before it."""
    b = Batch([37, 90], [new, new], 8, 2, 64, torch.float16, 16)
    want = b(max_new=new)
    last = 37 + new - 1
    page = int(b.table[0, last // 16])
    b.cache_v[page, 1, last % 16, 5] = bad
    out = b(max_new=new)
    hit = out[new - 1, 4:, 5]
    assert bool(hit.isnan().all()) if bad != bad else bool((hit == bad).all())
    out[new - 1, 4:, 5] = want[new - 1, 4:, 5]
    assert torch.equal(out, want)


def test_cache_layouts_and_strides():
    """Slots before heads, and both caches in one array: the same bits."""
    b = Batch([300, 12, 70], [1, 60, 2], 8, 2, 64, torch.float16, 32)
    want = b(max_new=60)
    k, v = b.cache_k, b.cache_v
    b.cache_k = k.transpose(1, 2).contiguous().transpose(1, 2)
    b.cache_v = v.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(b(max_new=60), want)
    both = torch.stack([k, v], 1)
    b.cache_k, b.cache_v = both[:, 0], both[:, 1]
    wide = torch.full((3, b.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide[:, :b.table.shape[1]]
    q = b.q
    b.q = torch.cat([q, q], 2)[..., :64]
    assert torch.equal(b(max_new=60), want)
    out = torch.full_like(q, 3.0)
    assert torch.equal(b(max_new=60, out=out), want)


def test_far_pages_pass_32_bits():
    """A cache of more than 2^32 bytes per array: the last pages are read."""
    pages = 70000
    k = torch.zeros(pages, 4, 64, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    b = Batch([500, 100], [1, 80], 8, 4, 128, torch.bfloat16, 64)
    n = b.cache_k.shape[0]
    k[pages - n:], v[pages - n:] = b.cache_k, b.cache_v
    want = b(max_new=80)
    b.cache_k, b.cache_v = k, v
    b.table = torch.where(b.table >= 0, b.table + (pages - n), b.table)
    assert torch.equal(b(max_new=80), want)


def test_captured_and_replayed():
    """Captured calls follow the lengths on the device; every replay equals the eager call, other work between."""
    b = Batch([600, 40, 0], [1, 1, 1], 8, 2, 64, torch.float16, 16, extra_width=40)
    b(max_new=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b(max_new=1)
        out2 = b()
    for lens in ([601, 41, 1], [3, 41, 1], [601, 2, 1], [17, 16, 0]):
        b.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        want = b(max_new=1)
        junk = torch.randn(1 << 20, device=DEV).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want) and bool(junk.isfinite())


def test_two_streams_at_once():
    """Two calls that may overlap have workspaces of their own."""
    a = Batch([9000, 100], [1, 1], 8, 2, 64, torch.float16, 16)
    b = Batch([70, 7000], [1, 1], 8, 2, 64, torch.float16, 16, seed=5)
    want = a(max_new=1), b(max_new=1)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        for x, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(x(max_new=1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (4, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("ctx,new", [([20000], [100]), ([9000, 0], [200, 90]), ([300, 5000, 40], [150, 70, 1]),
                                     ([700] * 30, [80] * 30)], ids=["cut", "cut2", "mixed", "ordered"])
def test_every_plan(heads, kv_heads, d, ctx, new):
    """Chunks over long contexts, cut over workgroups, beside short ones and single tokens."""
    b = Batch(ctx, new, heads, kv_heads, d, torch.bfloat16, 32, pad=2)
    b.check(b(max_new=max(new)))


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 64), (16, 8, 128), (8, 8, 96)])
@pytest.mark.parametrize("longest,new", [(15, 1), (500, 1), (980, 1), (980, 9)])
def test_many_short_requests(heads, kv_heads, d, longest, new):
    """An item or more for each of a few hundred CUs: whole ones and cut ones, one and two row tiles, pages missing."""
    count = 41
    b = Batch([(i * 37 * longest // 600) % longest if i % 9 else 0 for i in range(count)],
              [0 if i == 7 else 1 + i * 5 % new for i in range(count)], heads, kv_heads, d, torch.float16, 16, pad=1)
    lens = b.seq_lens.tolist()
    there = [torch.ones(n, dtype=torch.bool, device=DEV) for n in lens]
    long = max(range(count), key=lens.__getitem__)
    b.table[long, 0] = -1
    there[long][:16] = False
    b.check(b(max_new=new), there)


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 4, 64), (64, 8, 64), (32, 8, 128), (16, 16, 96)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_chunks_beside_single_tokens(heads, kv_heads, d, dtype):
    """Many row tiles of chunks, and single tokens over long contexts, in one launch: the rows at which a request goes to the
    other kind of workgroups, empty requests, pages that are missing in either kind, infinities behind a row's last key."""
    rep = heads // kv_heads
    edge = 64 // rep
    ctx = [0, 2900, 40, 700, 1300, 0, 16, 511, 1024, 5, 1900, 64]
    new = [300, 1, edge, edge + 1, 400, 0, 250, 1, 129, 2, 1, 333]
    b = Batch(ctx, new, heads, kv_heads, d, dtype, 16, pad=3)
    there = [torch.ones(c + n, dtype=torch.bool, device=DEV) for c, n in zip(ctx, new)]
    for r, page in ((1, 100), (4, 7), (8, 65)):
        b.table[r, page] = -1
        there[r][16 * page:16 * page + 16] = False
    out = b(max_new=400)
    b.check(out, there)
    assert torch.equal(out, b())
    last = ctx[4] + new[4] - 1
    b.cache_v[b.table[4, last // 16].long(), 0, last % 16, 3] = float("inf")
    got = b()
    row = sum(new[:5]) - 1
    assert bool((got[row, :rep, 3] == float("inf")).all())
    got[row, :rep, 3] = out[row, :rep, 3]
    assert torch.equal(got, out)


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 4, 64), (32, 8, 128), (8, 8, 96), (8, 2, 256)])
@pytest.mark.parametrize("pad", [0, 9])
def test_short_chunks(heads, kv_heads, d, pad):
    """A few requests of some tokens, single tokens for the most part: both sides of every bound on their rows."""
    rep = heads // kv_heads
    for most in (64 // rep, 64 // rep + 1, 128 // rep, 128 // rep + 1):
        new = [1, most, 0, 2, most // 2, 1, 1, 3, 1, 1, 1, 1]
        b = Batch([(i * 401 + 7) % 1500 for i in range(12)], new, heads, kv_heads, d, torch.bfloat16, 16, pad=pad)
        b.check(b(max_new=most))
        b.check(b())


def test_chunks_beside_single_tokens_of_many_requests():
    """More requests than are put in the order of their lengths."""
    count = 90
    ctx = [(i * 211) % 700 for i in range(count)]
    new = [1 if i % 3 else 30 + i for i in range(count)]
    b = Batch(ctx, new, 32, 8, 128, torch.float16, 32, pad=5)
    b.check(b(max_new=max(new)))


def test_chunks_beside_single_tokens_in_a_graph():
    """One captured call, whose requests change from chunks to single tokens and back between replays."""
    b = Batch([700] * 16, [90] * 16, 32, 8, 128, torch.float16, 16)
    b()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b()
    for new in ([90] * 16, [1] * 16, [1, 179] * 8, [0] * 15 + [1440]):
        b.cu.copy_(offsets(new, DEV))
        b.seq_lens.copy_(torch.tensor([max(n, 790 - n) for n in new], dtype=torch.int32))
        want = b()
        junk = torch.randn(1 << 20, device=DEV).sum()
        graph.replay()
        torch.cuda.synchronize()
        # Bits: the last request's keys go on into a page's unused slots, which hold NaN.
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and bool(junk.isfinite())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_holes_and_infinities_in_cut_items(bad):
    """A long item in pieces: a page that is missing in the middle, and values beyond a row's last key."""
    b = Batch([20000], [100], 8, 2, 64, torch.float16, 16)
    there = torch.ones(20100, dtype=torch.bool, device=DEV)
    b.table[0, 400] = -1
    there[6400:6416] = False
    out = b(max_new=100)
    b.check(out, [there])
    last = 20099
    b.cache_v[b.table[0, last // 16].long(), 1, last % 16, 5] = bad
    hit = b(max_new=100)
    got = hit[99, 4:, 5]
    assert bool(got.isnan().all()) if bad != bad else bool((got == bad).all())
    hit[99, 4:, 5] = out[99, 4:, 5]
    assert torch.equal(hit, out)


def test_registered_ops():
    b = Batch([40, 3], [1, 5], 4, 2, 64, torch.float16, 16)
    args = (b.q, b.cache_k.nan_to_num(), b.cache_v.nan_to_num(), b.table, b.cu, b.seq_lens, 5, 0.125)
    torch.library.opcheck(ops._paged_attention_op, args, test_utils=("test_schema", "test_faketensor"))
    assert torch.equal(torch.ops.kernelforge.paged_attention(*args), b(max_new=5))
    t = torch.zeros(2, 9, dtype=torch.int32, device=DEV)
    lens = torch.tensor([4, 0], dtype=torch.int32, device=DEV)
    free, count = torch.arange(9, dtype=torch.int32, device=DEV), torch.tensor([9], dtype=torch.int32, device=DEV)
    torch.library.opcheck(ops._paged_tables_op, (t, lens, lens, free, count, 16, 8),
                          test_utils=("test_schema", "test_faketensor"))
    pos, slots = torch.arange(4, device=DEV), torch.arange(4, device=DEV)
    cos = torch.ones(8, 64, device=DEV)
    caches = [torch.zeros(3, 2, 16, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    qkv = torch.randn(4, 512, device=DEV).half()
    torch.library.opcheck(ops._rope_paged_op, (qkv, cos, cos, pos, slots, *caches, 4),
                          test_utils=("test_schema", "test_faketensor"))
