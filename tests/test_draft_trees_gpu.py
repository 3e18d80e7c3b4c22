"""Ancestors and positions of drafted trees against a node-by-node construction (needs a GPU)."""

from __future__ import annotations

import random

import pytest
import torch

from kernelforge import ops

from draft_cases import ancestors_of, chain, positions_of, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def expected(trees, ctx, pad):
    bits = [b for t in trees for b in ancestors_of(t)] + [0] * pad
    pos = [p for t, c in zip(trees, ctx) for p in positions_of(t, c)] + [-1] * pad
    return bits, pos


def run(trees, ctx, pad=0):
    cu = [0]
    for t in trees:
        cu.append(cu[-1] + len(t))
    parents = i32([p for t in trees for p in t] + [0] * pad)
    return ops.draft_trees(parents, i32(cu), i32([c + len(t) for c, t in zip(ctx, trees)]))


@pytest.mark.parametrize("lens,pad", [([1], 0), ([64], 0), ([0], 3), ([2, 0, 64, 1, 33], 5), ([63, 64, 65, 130, 7], 0),
                                      ([1 + i % 64 for i in range(301)], 70)])
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_trees(lens, pad, kind):
    rng = random.Random(len(lens) + pad)
    make = {"random": lambda n: random_tree(n, rng, 6), "chain": chain, "star": lambda n: [-1] + [0] * (n - 1) if n else []}[kind]
    trees = [make(n) for n in lens]
    ctx = [rng.randrange(0, 100000) for _ in lens]
    got = run(trees, ctx, pad)
    bits, pos = expected(trees, ctx, pad)
    assert got.ancestors.tolist() == bits and got.positions.tolist() == pos
    assert got.positions.data_ptr() % 16 == 0


def test_parents_that_are_none_begin_a_tree():
    trees = [[-1, -1, 0, 5, 3, -7, 1 << 30, 6], [3, 0, 1]]
    got = run(trees, [10, 0])
    bits, pos = expected(trees, [10, 0], 0)
    assert got.ancestors.tolist() == bits and got.positions.tolist() == pos


def test_offsets_that_do_not_fit_stay_inside():
    parents = torch.zeros(6, dtype=torch.int32, device=DEV)
    ops.draft_trees(parents, i32([0, 1 << 30, -4]), i32([5, -3]))
    ops.draft_trees(parents, i32([3, 2, 1]), i32([1 << 30, 2]))
    torch.cuda.synchronize()


def test_no_tokens_registered_op_and_another_stream():
    empty = ops.draft_trees(i32([]), i32([0, 0]), i32([4]))
    assert empty.ancestors.shape == empty.positions.shape == (0,)
    parents, cu, lens = i32([-1, 0, 0, 2]), i32([0, 4]), i32([9])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.draft_trees(parents, cu, lens)
    torch.cuda.current_stream().wait_stream(side)
    b = torch.ops.kernelforge.draft_trees(parents, cu, lens)
    assert a.ancestors.tolist() == [1, 3, 5, 13] and a.positions.tolist() == [5, 6, 6, 7]
    assert torch.equal(a.ancestors, b[0]) and torch.equal(a.positions, b[1])


def test_captured():
    parents, cu, lens = i32([-1, 0, 1, 2, 9]), i32([0, 3, 5]), i32([3, 2])
    ops.draft_trees(parents, cu, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.draft_trees(parents, cu, lens)
    for trees, ctx in (([[-1, 0, 0], [-1, 0]], [7, 100]), ([[-1], [-1, 0, 1, 1]], [0, 3]), ([[], [-1, 0, 0, 0, 3]], [5, 6])):
        parents.copy_(i32([p for t in trees for p in t]))
        cu.copy_(i32([0, len(trees[0]), 5]))
        lens.copy_(i32([c + len(t) for c, t in zip(ctx, trees)]))
        graph.replay()
        torch.cuda.synchronize()
        assert (out.ancestors.tolist(), out.positions.tolist()) == expected(trees, ctx, 0)
        eager = ops.draft_trees(parents, cu, lens)
        assert torch.equal(eager.ancestors, out.ancestors)
