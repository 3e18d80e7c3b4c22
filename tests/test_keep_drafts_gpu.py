"""What keep_drafts leaves in the cache and on the stack of free pages (needs a GPU), against moves one by one on the host, and the
operators of a drafted step in a row."""

from __future__ import annotations

import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from kernelforge import ops

from attention_cases import check
from draft_cases import ancestors_of, random_tree, random_trees, tree64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Step:
    """Requests of ctx tokens and new nodes over shuffled pages, and a path through each tree."""

    def __init__(self, ctx, new, block=16, arrays=3, kv_heads=2, d=64, dtype=torch.float16, seed=0, width=64, spare=5, extra=0):
        rng = random.Random(seed + len(ctx))
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.new, self.block = ctx, new, block
        need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g).tolist()
        self.table = [[-1] * (max(need) + 1 + extra) for _ in ctx]
        for r, n in enumerate(need):
            self.table[r][:n] = [perm.pop() for _ in range(n)]
        self.stack, self.free = perm + [-5] * (pages - spare), spare
        self.paths = []
        for n in new:
            tree, path = random_tree(n, rng, 4), []
            node = rng.randrange(n) if n else -1
            while node >= 0:
                path.append(node)
                node = tree[node]
            self.paths.append(path[::-1])
        self.width = width
        self.counts = [len(p) for p in self.paths]
        self.caches = torch.randn(arrays, pages, kv_heads, block, d, generator=g).to(dtype)

    def host(self):
        caches, stack, free, lens = self.caches.clone(), list(self.stack), self.free, []
        for r, path in enumerate(self.paths):
            moved = []
            for i, p in enumerate(path[:self.width]):
                moved.append((self.ctx[r] + p, self.ctx[r] + i))
            for a, b in moved:
                if a != b:
                    caches[:, self.table[r][b // self.block], :, b % self.block] = \
                        caches[:, self.table[r][a // self.block], :, a % self.block]
            lens.append(self.ctx[r] + len(moved))
            for j in range(-(-lens[-1] // self.block), -(-(self.ctx[r] + self.new[r]) // self.block)):
                if free < len(stack):
                    stack[free] = self.table[r][j]
                    free += 1
        return caches, stack, lens, free

    def args(self):
        path = i32([(p + [-1] * 64)[:self.width] for p in self.paths])
        return (i32(self.table), i32(self.ctx), i32([c + n for c, n in zip(self.ctx, self.new)]), i32(self.counts), path)

    def check(self, caches=None):
        caches = self.caches.to(DEV) if caches is None else caches
        stack = i32(self.stack)
        got = ops.keep_drafts(caches, *self.args(), stack, i32([self.free]))
        want = self.host()
        assert torch.equal(caches.reshape(want[0].shape).cpu(), want[0])
        assert stack.tolist() == want[1] and got.context_lens.tolist() == want[2] and got.free_count.tolist() == [want[3]]


@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0], [64]), ([15, 16, 17, 0], [1, 20, 64, 33]), ([100, 3, 50], [0, 64, 0]),
                                     ([7 * i for i in range(70)], [1 + i % 64 for i in range(70)])])
@pytest.mark.parametrize("block,kv_heads,d,dtype", [(16, 2, 64, torch.float16), (64, 1, 128, torch.bfloat16),
                                                    (16, 3, 8, torch.float16), (128, 2, 200, torch.bfloat16)])
def test_moves(ctx, new, block, kv_heads, d, dtype):
    Step(ctx, new, block, 5, kv_heads, d, dtype).check()


def test_more_requests_than_threads():
    rng = random.Random(1)
    Step([rng.randrange(40) for _ in range(700)], [rng.randrange(0, 65) for _ in range(700)], arrays=1, d=8).check()


def test_layouts():
    """Arrays of several dimensions, one alone, strides of their own, and lists of arrays."""
    step = Step([30, 5], [40, 64], arrays=6)
    step.check(step.caches.to(DEV).view(3, 2, *step.caches.shape[1:]))
    one = Step([30, 5], [40, 64], arrays=1)
    one.check(one.caches.to(DEV)[0])
    wide = torch.zeros(6, step.caches.shape[1], 2, 16, 80, dtype=torch.float16, device=DEV)[..., :64]
    wide.copy_(step.caches)
    step.check(wide)
    turned = torch.empty(step.caches.shape[1], 6, 16, 2, 64, dtype=torch.float16, device=DEV).permute(1, 0, 3, 2, 4)
    turned.copy_(step.caches)
    step.check(turned)
    parts, stack = [c.to(DEV) for c in step.caches], i32(step.stack)
    got = ops.keep_drafts(parts, *step.args(), stack, i32([step.free]))
    want = step.host()
    assert torch.equal(torch.stack(parts).cpu(), want[0]) and stack.tolist() == want[1]
    assert got.context_lens.tolist() == want[2] and got.free_count.tolist() == [want[3]]
    parts = [c.to(DEV) for c in step.caches]
    got = ops.keep_drafts(parts, *step.args())  # without a stack
    assert torch.equal(torch.stack(parts).cpu(), want[0]) and got.context_lens.tolist() == want[2] and got.free_count is None


def test_leading_dimensions_of_one():
    """Their strides say nothing."""
    step = Step([30, 5], [40, 64], arrays=6)
    whole = torch.zeros(6, 2, 1, *step.caches.shape[1:], dtype=torch.float16, device=DEV)
    step.check(whole[:, :1].copy_(step.caches[:, None, None]))
    step.check(whole[:, 1].copy_(step.caches[:, None]))


def test_counts_that_do_not_fit():
    step = Step([30, 5, 9], [4, 64, 2], width=4)
    step.counts = [1 << 30, 3, -2]
    step.paths = [[0, 2, 3, 1 << 30][:4], [0, 63, 64], []]
    args = step.args()
    caches = step.caches.to(DEV)
    got = ops.keep_drafts(caches, *args, i32(step.stack), i32([step.free]))
    assert got.context_lens.tolist() == [34, 8, 9]
    step.paths = [[0, 2, 3], [0, 63], []]  # the moves that there are
    want = step.host()[0]
    assert torch.equal(caches.cpu(), want)


def test_places_that_are_not_there():
    """Holes in a table, numbers that are no page, tables that are too narrow: such entries move nothing."""
    step = Step([10, 20], [64, 64])
    before = step.caches.to(DEV)
    for value in (-1, -9, step.caches.shape[1], 1 << 30):
        step.table[0] = [value] * len(step.table[0])
        step.table[1][2:] = [value] * len(step.table[1][2:])
        step.paths = [[0, 9, 20], [0, 40, 60]]
        step.counts = [3, 3]
        caches = before.clone()
        ops.keep_drafts(caches, *step.args(), i32(step.stack), i32([step.free]))
        assert torch.equal(caches, before)
    table, ctx, seq, counts, path = step.args()
    ops.keep_drafts(before, table[:, :1], i32([1 << 30, -5]), i32([1 << 30, 1 << 30]), counts, path, i32(step.stack), i32([-3]))
    torch.cuda.synchronize()


def test_a_full_stack():
    step = Step([0, 0], [64, 64])
    step.paths, step.counts = [[0], [0]], [1, 1]
    step.stack, step.free = step.stack[:step.free + 4], step.free
    step.check()


def test_registered_op_stream_and_capture():
    step = Step([33, 4, 70], [20, 64, 9], seed=3)
    want = step.host()
    args, stack, caches = step.args(), i32(step.stack), step.caches.to(DEV)
    kept = torch.ops.kernelforge.keep_drafts(caches, *args, stack, i32([step.free]))
    assert torch.equal(caches.cpu(), want[0]) and stack.tolist() == want[1] and kept.tolist() == [*want[2], want[3]]
    caches.copy_(step.caches)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.keep_drafts(caches, *args, i32(step.stack), i32([step.free]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(caches.cpu(), want[0])
    free = i32([step.free])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.keep_drafts(caches, *args, stack, free)
    for seed in (3, 4, 5):
        step = Step([33, 4, 70], [20, 64, 9], seed=seed)
        for old, new in zip((caches, *args, stack, free), (step.caches, *step.args(), i32(step.stack), i32([step.free]))):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = step.host()
        assert torch.equal(caches.cpu(), want[0]) and stack.tolist() == want[1]
        assert out.context_lens.tolist() == want[2] and out.free_count.tolist() == [want[3]]


def test_steps_in_a_row():
    """Tables, trees, writer, attention, verification and keeping, three steps as a server runs them: after each the cache holds
    exactly the accepted tokens of every request, and no page is lost."""
    heads, kv, d, block, vocab, dtype = 8, 2, 64, 16, 97, torch.float16
    g = torch.Generator(device=DEV).manual_seed(5)
    rng = random.Random(5)
    pages, b = 60, 4
    table = i32([[-1] * 20 for _ in range(b)])
    free, free_count = i32(list(range(pages))), i32([pages])
    caches = torch.zeros(2, pages, kv, block, d, dtype=dtype, device=DEV)
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    ang = torch.arange(400, dtype=torch.float64, device=DEV)[:, None] * inv
    cos, sin = torch.cat([ang.cos()] * 2, 1).float(), torch.cat([-ang.sin(), ang.sin()], 1).float()
    context = i32([0] * b)
    kept_k, kept_v = [[] for _ in range(b)], [[] for _ in range(b)]
    for turn in range(3):
        lens = [[40, 9, 64, 1], [5, 0, 64, 30], [1, 33, 0, 17]][turn]
        trees = random_trees(lens, turn, 2)
        parents = i32([p for t in trees for p in t] + [0, 0])
        new = i32(lens)
        step = ops.paged_tables(table, context, new, free, free_count, block_size=block, max_tokens=sum(lens) + 2)
        tree = ops.draft_trees(parents, step.cu_new, step.seq_lens)
        qkv = torch.randn(sum(lens) + 2, (heads + 2 * kv) * d, generator=g, device=DEV).to(dtype)
        q, k = ops.rope_paged_cache(qkv, cos, sin, tree.positions, step.slots, caches[0], caches[1], heads=heads)
        v = qkv.view(-1, heads + 2 * kv, d)[:, heads + kv:]
        out = ops.paged_tree_attention(q, caches[0], caches[1], table, step.cu_new, step.seq_lens, tree.ancestors, max_new=64)
        at = 0
        for r, t in enumerate(trees):
            if t:
                past = [torch.stack(x) if x else k[:0] for x in (kept_k[r], kept_v[r])]
                ref, bound = tree64(q[at:at + len(t)], torch.cat([past[0], k[at:at + len(t)]]),
                                    torch.cat([past[1], v[at:at + len(t)]]), ancestors_of(t))
                check(out[at:at + len(t)], ref, bound, f"step {turn}, request {r}")
            at += len(t)
        scores = torch.randn(sum(lens) + 2, vocab, generator=g, device=DEV)
        tokens = torch.randint(0, vocab, (sum(lens) + 2,), generator=g, device=DEV)
        at = 0
        for t in trees:  # the target agrees with most drafts
            for i, p in enumerate(t):
                if i and rng.random() < 0.8:
                    tokens[at + i] = scores[at + p].argmax()
            at += len(t)
        done = ops.verify_drafts(tokens, parents, step.cu_new, scores)
        kept = ops.keep_drafts(caches, table, context, step.seq_lens, done.counts, done.path, free, step.free_count)
        at = 0
        for r, t in enumerate(trees):
            for node in done.path[r, :int(done.counts[r])].tolist():
                kept_k[r].append(k[at + node])
                kept_v[r].append(v[at + node])
            at += len(t)
        context, free_count = kept.context_lens, kept.free_count
        assert context.tolist() == [len(x) for x in kept_k]
        held = []
        for r in range(b):
            used = -(-len(kept_k[r]) // block)
            held += table[r, :used].tolist()
            for i, (kk, vv) in enumerate(zip(kept_k[r], kept_v[r])):
                page = int(table[r, i // block])
                assert torch.equal(caches[0, page, :, i % block], kk) and torch.equal(caches[1, page, :, i % block], vv)
        assert sorted(held + free[:int(free_count)].tolist()) == list(range(pages))
    assert max(context.tolist()) > 4


@pytest.mark.parametrize("heads,kv,dtype", [(8, 4, torch.float16), (12, 2, torch.bfloat16)])
@pytest.mark.parametrize("mode", ["greedy", "drawn"])
def test_a_captured_step(heads, kv, dtype, mode):
    """A whole step in one graph, replayed over other lengths, trees and drafts, beside the same eager calls on a state of their own:
    all that it writes is bit for bit the same."""
    d, block, vocab, rows, pages, b = 64, 16, 211, 150, 100, 4
    g = torch.Generator(device=DEV).manual_seed(9)
    rng = random.Random(9)
    ang = torch.arange(600, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (
        -torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    cos, sin = torch.cat([ang.cos()] * 2, 1).float(), torch.cat([-ang.sin(), ang.sin()], 1).float()

    def state():
        return dict(caches=torch.zeros(2, pages, kv, block, d, dtype=dtype, device=DEV), table=torch.full_like(i32([[0] * 70] * b), -1),
                    context=i32([0] * b), free=i32(list(range(pages))), count=i32([pages]))

    inputs = dict(new=i32([0] * b), parents=i32([0] * rows), tokens=torch.zeros(rows, dtype=torch.int64, device=DEV),
                  qkv=torch.zeros(rows, (heads + 2 * kv) * d, dtype=dtype, device=DEV), target=torch.zeros(rows, vocab, device=DEV),
                  accept=torch.zeros(rows, device=DEV), sample=torch.zeros(b, device=DEV), draft=torch.zeros(rows, vocab, device=DEV))

    def run(s, x):
        step = ops.paged_tables(s["table"], s["context"], x["new"], s["free"], s["count"], block_size=block, max_tokens=rows)
        trees = ops.draft_trees(x["parents"], step.cu_new, step.seq_lens)
        q, _ = ops.rope_paged_cache(x["qkv"], cos, sin, trees.positions, step.slots, s["caches"][0], s["caches"][1], heads=heads)
        out = ops.paged_tree_attention(q, s["caches"][0], s["caches"][1], s["table"], step.cu_new, step.seq_lens, trees.ancestors)
        if mode == "greedy":
            done = ops.verify_drafts(x["tokens"], x["parents"], step.cu_new, x["target"])
        else:
            done = ops.verify_drafts(x["tokens"], x["parents"], step.cu_new, x["target"], x["accept"], x["sample"], draft=x["draft"])
        kept = ops.keep_drafts(s["caches"], s["table"], s["context"], step.seq_lens, done.counts, done.path, s["free"],
                               step.free_count)
        s["context"].copy_(kept.context_lens)
        s["count"].copy_(kept.free_count)
        return (*trees, out, *done)

    eager, captured = state(), state()
    run(state(), inputs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run(captured, inputs)
    for lens in ([64, 1, 30, 17], [5, 64, 0, 64], [0, 0, 0, 0], [1, 1, 1, 1], [33, 9, 64, 2], [16, 64, 3, 60]):
        trees = random_trees(lens, sum(lens), 3)
        inputs["new"].copy_(i32(lens))
        inputs["parents"].copy_(i32([p for t in trees for p in t] + [0] * (rows - sum(lens))))
        inputs["qkv"].normal_(generator=g)
        for name in ("target", "draft"):
            inputs[name].copy_(torch.softmax(3 * torch.randn(rows, vocab, generator=g, device=DEV), -1))
        for name in ("accept", "sample"):
            inputs[name].uniform_(generator=g)
        inputs["tokens"].copy_(torch.randint(0, vocab, (rows,), generator=g, device=DEV))
        at = 0
        for t in trees:
            for i, p in enumerate(t):
                if i and rng.random() < 0.8:
                    inputs["tokens"][at + i] = inputs["target"][at + p].argmax()
            at += len(t)
        graph.replay()
        want = run(eager, inputs)
        torch.cuda.synchronize()
        for x, y in zip((*static, *captured.values()), (*want, *eager.values())):
            assert torch.equal(x, y)
    assert int(eager["context"].max()) > 10


def test_a_cache_whose_offsets_pass_32_bits():
    """Attention and moves over the last pages of a large cache, against those pages alone."""
    kv, block, d, pages, few, heads = 4, 64, 128, 70000, 12, 8
    g = torch.Generator(device=DEV).manual_seed(2)
    small = torch.randn(2, few, kv, block, d, generator=g, device=DEV).half()
    large = torch.empty(2, pages, kv, block, d, dtype=torch.float16, device=DEV)
    assert large[0].numel() > 1 << 31
    large[:, -few:] = small
    lens, ctx = [40, 3], [500, 90]
    trees = random_trees(lens, 4, 2)
    table = i32([[3, 0, 5, 7, 1, 11, 2, 9, 4], [10, 6, -1, -1, -1, -1, -1, -1, -1]])
    far = torch.where(table >= 0, table + (pages - few), -1)
    cu, seq = i32([0, 40, 43]), i32([c + n for c, n in zip(ctx, lens)])
    words = torch.tensor([w for t in trees for w in ancestors_of(t)], dtype=torch.int64, device=DEV)
    q = torch.randn(43, heads, d, generator=g, device=DEV).half()
    for max_new in (None, 2):  # both kernels' plans
        rows = q if max_new is None else q[:, :4].repeat(1, 2, 1)
        near = ops.paged_tree_attention(rows, small[0], small[1], table, cu, seq, words, max_new=max_new)
        assert torch.equal(ops.paged_tree_attention(rows, large[0], large[1], far, cu, seq, words, max_new=max_new), near)
    path = i32([[0, 7, 20, 39] + [-1] * 60, [0, 2] + [-1] * 62])
    for cache, t in ((small, table), (large, far)):
        assert ops.keep_drafts(cache, t, i32(ctx), seq, i32([4, 2]), path).context_lens.tolist() == [504, 92]
    assert torch.equal(large[:, -few:], small)


def test_lists_of_arrays_that_share_places():
    """Views that meet are refused before anything moves; views of one tensor that do not are taken."""
    step = Step([30, 5], [40, 64], arrays=6)
    args, want = step.args(), step.host()
    caches, stack = step.caches.to(DEV), i32(step.stack)
    before = caches.clone()
    flat = caches.view(-1)
    shifted = flat[64:64 + 5 * caches[0].numel()].view(5, *caches.shape[1:])  # begins one token later
    for listed in ([caches, caches[1:]], [caches[5], caches[1:]], [caches[:4], caches[3:]], [caches[:, :9], caches[:, 8:]],
                   [caches[0], shifted], [caches[..., :64], caches[2:3, ..., 32:]]):
        with pytest.raises(ValueError, match="different arrays"):
            ops.keep_drafts(listed, *args, stack, i32([step.free]))
    assert torch.equal(caches, before) and stack.tolist() == step.stack
    turned = torch.empty(step.caches.shape[1], 6, 16, 2, 64, dtype=torch.float16, device=DEV).permute(1, 0, 3, 2, 4)
    for whole in (caches, turned):
        for parts in ([whole[i] for i in range(6)], [whole[:2], whole[2], whole[3:]], [whole[::2], whole[1::2]]):
            whole.copy_(step.caches)
            stack = i32(step.stack)
            got = ops.keep_drafts(parts, *args, stack, i32([step.free]))
            assert torch.equal(whole.cpu(), want[0]) and stack.tolist() == want[1] and got.context_lens.tolist() == want[2]


def test_a_list_with_an_array_elsewhere():
    """Nothing is moved before all arrays have been looked at."""
    step = Step([30, 5], [40, 64], arrays=2)
    caches, stack = step.caches.to(DEV), i32(step.stack)
    with pytest.raises(RuntimeError, match="must be on cuda"):
        ops.keep_drafts([caches[0], step.caches[1]], *step.args(), stack, i32([step.free]))
    assert torch.equal(caches.cpu(), step.caches) and stack.tolist() == step.stack


def test_a_list_in_a_traced_call():
    """Through the registered op: the same results, and views that meet are refused when it runs."""
    step = Step([30, 5], [40, 64], arrays=4)
    args, want = step.args(), step.host()
    caches, stack, free = step.caches.to(DEV), i32(step.stack), i32([step.free])

    def call(a, b, *rest):
        return ops.keep_drafts([a, b], *rest)

    mode = FakeTensorMode()
    fake = [mode.from_tensor(t) for t in (caches[:2], caches[2:], *args, stack, free)]
    with torch.no_grad(), mode:
        graph = make_fx(call)(*fake)
    got = graph(caches[:2], caches[2:], *args, stack, free)
    assert torch.equal(caches.cpu(), want[0]) and stack.tolist() == want[1]
    assert got.context_lens.tolist() == want[2] and got.free_count.tolist() == [want[3]]
    before = caches.clone()
    for a, b in ((caches, caches[1:]), (caches[1:3], caches[:2]), (caches[1:2], caches[1:2])):
        with pytest.raises(ValueError, match="different arrays"):
            graph(a, b, *args, stack, free)
    assert torch.equal(caches, before) and stack.tolist() == want[1]
