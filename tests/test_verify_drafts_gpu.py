"""Verification of drafted trees (needs a GPU) against a walk along each tree on the host in 64 bits: integers have to be equal.  A
test of acceptance compares products of 32-bit numbers, exact in 64 bits, and sums whose errors (vocab 2^-53) are some 10^8 times
smaller than the distance of random numbers from a border."""

from __future__ import annotations

import random

import pytest
import torch

from kernelforge import ops

from draft_cases import chain, random_trees, verify_on_host

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return i32(cu)


class Case:
    """Requests of lens nodes; drafts that the target often agrees with; on the host until a call."""

    def __init__(self, lens, vocab, mode, seed=0, width=3, pad=0, trees=None, dtype=torch.float32):
        g = torch.Generator().manual_seed(seed + vocab + sum(lens))
        rng = random.Random(seed)
        self.lens, self.pad, self.mode = lens, pad, mode
        trees = trees or random_trees(lens, seed + 1, width)
        self.parents = [p for t in trees for p in t] + [0] * pad
        rows = sum(lens) + pad
        scores = torch.randn(rows, vocab, generator=g)
        self.accept = self.sample = self.draft = None
        if mode == "greedy":
            self.target = scores.to(dtype)
        else:
            self.target = torch.softmax(3 * scores, -1)
            rough = torch.softmax(3 * scores + torch.randn(rows, vocab, generator=g), -1)
            self.accept, self.sample = torch.rand(rows, generator=g), torch.rand(len(lens), generator=g)
            if mode == "drawn":
                self.draft = rough
        self.tokens, at = [], 0
        for tree in trees:
            for i, p in enumerate(tree):
                row = at + max(p, 0)
                best = int(self.target[row].float().argmax())
                if mode == "drawn":
                    best = int(torch.multinomial(self.draft[row], 1, generator=g))
                self.tokens.append(best if rng.random() < 0.7 else rng.randrange(vocab))
            at += len(tree)
        self.tokens += [0] * pad

    def host(self, width=64):
        return verify_on_host(self.tokens, self.parents, self.lens, self.target, self.accept, self.sample, self.draft, width)

    def args(self, target=None, draft=None):
        dev = [None if t is None else t.to(DEV) for t in (self.accept, self.sample)]
        target = self.target.to(DEV) if target is None else target
        draft = self.draft.to(DEV) if draft is None and self.draft is not None else draft
        return (torch.tensor(self.tokens, dtype=torch.int64, device=DEV), i32(self.parents), offsets(self.lens), target, *dev), draft

    def call(self, max_new=None, **kw):
        args, draft = self.args(**kw)
        return ops.verify_drafts(*args, draft=draft, max_new=max_new)

    def check(self, got=None, width=64):
        got = got or self.call(None if width == 64 else width)
        want = self.host(width)
        assert got.counts.tolist() == want[0]
        assert got.path.tolist() == want[1]
        assert got.tokens.tolist() == want[2]
        return want[0]


MODES = pytest.mark.parametrize("mode", ["greedy", "given", "drawn"])


@MODES
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 4095, 4096, 4097, 32000])
@pytest.mark.parametrize("lens,pad", [([1], 0), ([16], 0), ([5, 0, 64, 1, 2], 3)])
def test_sizes(mode, vocab, lens, pad):
    Case(lens, vocab, mode, pad=pad).check()


@MODES
@pytest.mark.parametrize("width", [1, 2, 64], ids=["chains", "pairs", "bushes"])
def test_many_requests(mode, width):
    """Most ends that a path can have come up: rejected at once, after some, siblings taken, whole branches accepted."""
    rng = random.Random(width)
    counts = Case([rng.randrange(0, 20) for _ in range(120)], 300, mode, seed=width, width=width).check()
    assert min(counts) == 0 and max(counts) > 2


@MODES
def test_a_large_vocabulary(mode):
    """More pieces of a row than one round of the threads takes up."""
    Case([7, 3], 256 * 4096 + 4097, mode, seed=2).check()


@pytest.mark.parametrize("vocab", [41000, 65537, 131075, 262143, 262150, 400001])
def test_rows_added_up_again(vocab):
    """Rejected siblings, so that the sums of the present row's pieces are not those of the first launch; and rows of which the draft
    leaves nothing. Places all over the row."""
    g = torch.Generator().manual_seed(vocab)
    lens, ends = [4] * 12, [0.0, 1.0 - 2.0 ** -24]
    case = Case(lens, vocab, "drawn", trees=[[-1, 0, 0, 0]] * 12)
    case.sample = torch.cat([torch.tensor(ends), torch.rand(10, generator=g)])
    case.accept[:] = 1.0 - 2.0 ** -24
    for r in range(12):
        p, q = case.target[4 * r], case.draft[4 * r]
        if r % 4 == 3:
            p.copy_(0.5 * q)
        worse = (q > 4 * p).nonzero()[:, 0] if r % 4 != 3 else (q > 0).nonzero()[:, 0]
        case.tokens[4 * r + 1:4 * r + 4] = worse[torch.randperm(len(worse), generator=g)[:3]].tolist()
    counts = case.check()
    assert max(counts) == 1


def test_rows_added_up_by_several_workgroups():
    """Requests with and without further sums side by side, on several streams at once and again and again: always the same."""
    case = Case([1, 9, 0, 20, 3, 16, 2, 30] * 3, 90001, "drawn", seed=5, width=4, pad=1)
    case.check()
    args, draft = case.args()
    want = ops.verify_drafts(*args, draft=draft)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for side in streams:
        side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(40):
        for side in streams:
            with torch.cuda.stream(side):
                got.append(ops.verify_drafts(*args, draft=draft))
    torch.cuda.synchronize()
    for done in got:
        assert all(torch.equal(x, y) for x, y in zip(done, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [9, 2049, 20001])
def test_scores_of_every_type_and_stride(dtype, vocab):
    case = Case([9, 30], vocab, "greedy", dtype=dtype)
    case.check()
    for start, width in ((1, vocab + 1), (3, vocab + 8)):  # rows that begin anywhere
        wide = torch.full((39, width + start), 100.0, dtype=dtype, device=DEV)[:, start:start + vocab]
        wide.copy_(case.target)
        case.check(case.call(target=wide))
    across = case.target.t().contiguous().t().to(DEV)
    case.check(case.call(target=across))


def test_probabilities_with_strides():
    for mode in ("given", "drawn"):
        case = Case([9, 30], 5001, mode)
        wide = torch.full((39, 5004), 3.0, device=DEV)
        wide[:, 1:5002] = case.target.to(DEV)
        draft = None
        if mode == "drawn":
            draft = torch.full((39, 5100), 3.0, device=DEV)
            draft[:, 7:5008] = case.draft.to(DEV)
            draft = draft[:, 7:5008]
        case.check(case.call(target=wide[:, 1:5002], draft=draft))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
def test_equal_scores_infinities_and_nan(dtype):
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros(8, 9000)
    rows[1, [8999, 4100, 77]] = 5.0           # the first of equal ones
    rows[2] = -inf                            # all equal: index 0
    rows[3, 5000], rows[3, 6000] = inf, inf
    rows[4, 100], rows[4, 8000], rows[4, 50] = inf, nan, nan
    rows[5] = -rows[5]                        # -0 and 0 are equal
    rows[5, 3:] = 0.0
    rows[6] = -1.0
    rows[6, 8191] = -0.5
    rows[7, :] = nan
    cu = i32(list(range(9)))
    got = ops.verify_drafts(torch.zeros(8, dtype=torch.int64, device=DEV), i32([-1] * 8), cu, rows.to(dtype).to(DEV), max_new=1)
    assert got.tokens[:, 0].tolist() == [0, 77, 0, 5000, 50, 0, 8191, 0]
    assert got.counts.tolist() == [1] * 8 and got.path.tolist() == [[0]] * 8


def test_tokens_outside_the_vocabulary_and_siblings_that_agree():
    tree = [-1, 0, 0, 0, 0, 1, 2, 3, 4]
    for mode in ("greedy", "given", "drawn"):
        for seed in range(20):
            case = Case([9, 9], 50, mode, seed=seed, trees=[tree, tree])
            best = int(case.target[0].float().argmax())
            case.tokens[1:5] = [-1, 50, best, best]
            case.tokens[10:14] = [1 << 40, best, best, -(1 << 35)]
            case.check()


def test_uniforms_at_their_ends():
    below = 1.0 - 2.0 ** -24
    for mode in ("given", "drawn"):
        for accept, sample in ((0.0, 0.0), (0.0, below), (below, 0.0), (below, below)):
            case = Case([6, 6, 1], 4100, mode, seed=3)
            case.accept.fill_(accept)
            case.sample.fill_(sample)
            case.check()
        case = Case([6, 1], 9000, mode, seed=4)
        case.target[:, 8500:] = 0.0
        case.sample.fill_(2.0)  # not below 1: the last index with any mass
        case.check()


def test_rows_without_mass():
    """Nothing is left after a rejection: the token is drawn from the whole row; a row of nothing gives 0."""
    target = torch.zeros(4, 5000)
    target[0, 4321] = 1.0
    target[1, [1, 4500]] = 0.5
    target[2] = float("nan")
    for mode in ("given", "drawn"):
        case = Case([2, 1, 1], 5000, mode, trees=[[-1, 0], [-1], [-1]])
        case.target = target.clone()
        case.tokens = [0, 4321, 0, 0]
        case.accept = torch.tensor([0.0, 1.0, 0.0, 0.0])  # 1 is not below the probability of 1
        case.sample = torch.tensor([0.5, 0.75, 0.5])
        if mode == "drawn":
            case.draft = torch.zeros(4, 5000)
            case.draft[0, 4321] = 1.0
        got = case.call()
        case.check(got)
        assert got.tokens[:, 0].tolist() == [4321, 0, 0]  # rows 0, 2 and 3 are the last nodes'
        case.target[2] = target[1]
        got = case.call()
        case.check(got)
        assert got.tokens[:, 0].tolist() == [4321, 4500, 0]
    for bad in (float("nan"), -3.0):  # count as nothing
        for mode in ("given", "drawn"):
            case = Case([6, 6], 4500, mode, seed=9)
            case.target[:, ::7] = bad
            case.check()


@MODES
def test_width(mode):
    """Nodes past the width are not looked at."""
    case = Case([30, 3, 64], 40, mode, seed=5)
    for width in (1, 4, 31):
        case.check(width=width)
    case = Case([100, 66], 40, mode, seed=6)  # more new tokens than nodes
    case.check()
    case.check(case.call(max_new=1000))


@pytest.mark.parametrize("tree", [[-1], [-1, 0], [-1, 0, 1, 2], [-1, 0, 0, 0, 1, 1, 2, 3], [-1, 0, 0, 2, 2, 2]],
                         ids=["none", "one", "chain", "tree", "late"])
@pytest.mark.parametrize("mode", ["given", "drawn"])
def test_emitted_tokens_have_the_targets_distribution(tree, mode):
    """20000 requests, each with its own random numbers: the first token emitted is distributed as row 0 of the target says, the
    second as the row of the node that the first one led to (every node's row depends on its token only).  Counts are
    binomial: held to five standard deviations."""
    n, vocab, b = len(tree), 6, 20000
    g = torch.Generator(device=DEV).manual_seed(n)
    by_token = torch.softmax(torch.randn(vocab, vocab, generator=g, device=DEV), -1)  # what follows a token
    rough = torch.softmax(torch.randn(vocab, vocab, generator=g, device=DEV), -1)
    tokens = torch.zeros(b, n, dtype=torch.int64, device=DEV)
    for i in range(1, n):
        if mode == "drawn":
            tokens[:, i] = torch.multinomial(rough[tokens[:, tree[i]]], 1, generator=g)[:, 0]
        else:  # given: fixed by place
            tokens[:, i] = (2 * i + tree[i]) % vocab
    flat = tokens.reshape(-1)
    got = ops.verify_drafts(flat, i32(tree * b), offsets([n] * b), by_token[flat].contiguous(),
                            torch.rand(n * b, generator=g, device=DEV), torch.rand(b, generator=g, device=DEV),
                            draft=rough[flat].contiguous() if mode == "drawn" else None)

    def as_drawn(tokens, row):
        want = row.double() * tokens.numel()
        have = torch.bincount(tokens, minlength=vocab).double()
        assert bool(((have - want).abs() <= 5 * torch.sqrt(want * (1 - row.double())) + 1).all()), (have, want)

    as_drawn(got.tokens[:, 0], by_token[0])
    for first in range(vocab):
        second = got.tokens[(got.tokens[:, 0] == first) & (got.counts > 1), 1]
        as_drawn(second, by_token[first])


def test_offsets_that_do_not_fit_stay_inside():
    for mode in ("greedy", "given", "drawn"):
        case = Case([10, 10], 100, mode)
        args, draft = case.args()
        for cu in ([0, 1 << 30, -4], [15, 3, 20], [20, 20, 20]):
            args[2].copy_(i32(cu))
            ops.verify_drafts(*args, draft=draft)
        torch.cuda.synchronize()


@MODES
def test_no_tokens(mode):
    case = Case([0, 0], 11, mode)
    got = case.call()
    assert got.counts.tolist() == [0, 0] and bool((got.path == -1).all()) and bool((got.tokens == -1).all())


@MODES
def test_stream_registered_op_and_repeats(mode):
    case = Case([20, 7, 40], 9001, mode, seed=8)
    args, draft = case.args()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.verify_drafts(*args, draft=draft)
    torch.cuda.current_stream().wait_stream(side)
    case.check(got)
    case.check(ops.VerifiedDrafts(*torch.ops.kernelforge.verify_drafts(*args, draft, 64)))


@MODES
def test_captured(mode):
    """Replays follow everything on the device; two graphs have workspaces of their own."""
    cases = [Case([12, 20, 5], 5000, mode, seed=s) for s in range(4)]
    args, draft = cases[0].args()
    ops.verify_drafts(*args, draft=draft)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.verify_drafts(*args, draft=draft))
        graphs.append(graph)
    for case in cases[1:]:
        new, new_draft = case.args()
        for old, t in zip((*args, draft), (*new, new_draft)):
            if old is not None:
                old.copy_(t)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            case.check(out)


@pytest.mark.parametrize("vocab", [4500, 90001])
@pytest.mark.parametrize("bad,counts_as", [(float("nan"), 0.0), (float("-inf"), 0.0), (-3.0, 0.0), (float("inf"), 1.0), (7.0, 1.0)],
                         ids=["nan", "-inf", "negative", "inf", "seven"])
def test_draft_probabilities_that_are_none(vocab, bad, counts_as):
    """What a draft row holds beside numbers from 0 to 1 counts as the nearer end, NaN as 0: the target's mass there stays, and
    drafted tokens that the target does not have are not accepted. Rows of nodes without children may hold anything."""
    case = Case([6, 9, 2], vocab, "drawn", seed=11, trees=[[-1, 0, 0, 0, 1, 1], [-1, 0, 0, 0, 0, 1, 2, 3, 3], [-1, 0]])
    case.draft[:, ::7] = counts_as
    case.target[:, ::14] = 0.0
    for i in range(1, 17, 3):
        case.tokens[i] = 14 * (i + 1)  # neither has any
    case.accept[3::2] = 1.0 - 2.0 ** -24
    raw = case.draft.clone()
    raw[:, ::7] = bad
    for leaf in (2, 3, 4, 5, 10, 11, 12, 13, 14, 16):
        raw[leaf] = bad
    case.check(case.call(draft=raw.to(DEV)))


@pytest.mark.parametrize("mode", ["given", "drawn"])
def test_more_pieces_than_threads(mode):
    """Rows of more than 2^22 values, whose pieces' sums (4096 values each) the 1024 threads of a workgroup take in two rounds, and
    whose further sums one workgroup makes. Half of the mass is behind the first round's; places in both rounds and at the end."""
    first, vocab = 1024 * 4096, 1024 * 4096 + 4097
    g = torch.Generator().manual_seed(3)
    trees = [[-1, 0, 0], [-1, 0], [-1, 0, 0], [-1], [-1]]
    lens = [len(t) for t in trees]
    rows = sum(lens)

    def halves(x):
        x[:, :first] /= 2 * x[:, :first].double().sum(1, keepdim=True)
        x[:, first:] /= 2 * x[:, first:].double().sum(1, keepdim=True)
        return x

    case = Case(lens, 8, mode, trees=trees)
    case.target = halves(torch.rand(rows, vocab, generator=g))
    case.accept[:] = 1.0 - 2.0 ** -24
    case.sample = torch.tensor([0.21, 0.93, 2.0, 0.93, 0.0])
    case.tokens = [int(t) for t in torch.randint(0, first, (rows,), generator=g)]
    if mode == "drawn":
        case.draft = halves(case.target * (0.25 + 4 * torch.rand(rows, vocab, generator=g)))
        at = 0
        for tree in trees:  # tokens that the draft has more often are rejected
            worse = (case.draft[at] > 1.5 * case.target[at]).nonzero()[:, 0]
            for i in range(1, len(tree)):
                case.tokens[at + i] = int(worse[5 * i])
            at += len(tree)
    got = case.call()
    case.check(got)
    assert got.counts.tolist() == [1] * 5
    places = got.tokens[:, 0].tolist()
    assert places[0] < first <= min(places[1], places[2], places[3]) and places[4] < 100


@pytest.mark.parametrize("vocab", [50, 41000])
def test_tokens_without_probability_are_never_accepted(vocab):
    """Whatever the random numbers: behind siblings that leave less than nothing of their parent's mass, as numbers that are not
    below 1 and rows that sum to more can, and with negative numbers."""
    tree = [-1, 0, 0, 0, 0, 0]
    for u in (2.0, 1.5, 0.9, -1.0):
        target = torch.zeros(6, vocab)
        target[:, 1], target[:, 2], target[:, 3] = 0.6, 0.5, 0.7
        tokens = [0, 1, 2, vocab, -3, 7] if u > 0 else [0, vocab, -1, 7, 8, 1]
        got = ops.verify_drafts(torch.tensor(tokens, device=DEV), i32(tree), i32([0, 6]), target.to(DEV),
                                torch.full((6,), u, device=DEV), torch.full((1,), 0.5, device=DEV))
        emitted = got.tokens[0, :int(got.counts[0])].tolist()
        assert set(emitted) <= {1, 2, 3}, (u, emitted)
