"""The paged decoder's steps with drafted tokens (needs a GPU): logits after every node against the single-stream model's, drafts
that are right, partly right and wrong, pages and lengths after them, and plain steps before and behind.  Logits are held to the bound of
test_paged_decoder_gpu.py, choices to twice of it."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops
from kernelforge import tinyllama as tl

from test_paged_decoder_gpu import BOUND, close, model, prompts, single  # noqa: F401 (model: a fixture)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def no_page_is_lost(dec):
    held = dec.block_table[dec.block_table >= 0].tolist()
    assert len(held) == sum(dec._pages(n) for n in dec.host_lens)
    assert sorted(dec.free_pages[:int(dec.free_count)].tolist() + held) == list(range(dec.num_pages))
    assert dec.context_lens.tolist() == dec.host_lens
    for row, n in enumerate(dec.host_lens):
        if n:
            assert int(dec.history[row, n]) == int(dec.tokens[row])


def choices_are_good(dec, row, prompt):
    """Each generated token is as good a choice as the single stream's, to within the bound."""
    assert torch.equal(dec.history[row, :prompt.numel()], prompt)
    for at in range(prompt.numel(), dec.host_lens[row] + 1):
        logits = single(dec.model, dec.history[row, :at])
        assert float(logits.max() - logits[dec.history[row, at]]) <= 2 * BOUND * float(logits.abs().max())


def test_logits_of_a_tree_against_the_single_stream(model):
    ps = prompts(70, 33, 1)
    dec = tl.PagedDecoder(model, DEV, requests=4, num_pages=60)
    dec.admit({0: ps[0], 2: ps[1], 3: ps[2]})
    parents = [[-1, 0, 0, 1, 1, 2, 3, 6], [-1, 0, 1, 2, 3], [-1]]
    g = torch.Generator(device=DEV).manual_seed(1)
    tokens = torch.randint(0, 2000, (14,), generator=g, device=DEV)
    flat = torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=DEV)
    step = ops.paged_tables(dec.block_table, dec.context_lens, torch.tensor([8, 0, 5, 1], dtype=torch.int32, device=DEV),
                            dec.free_pages, dec.free_count, block_size=16, max_tokens=14)
    trees = ops.draft_trees(flat, step.cu_new, step.seq_lens)
    logits = model.forward_paged(tokens, step, dec.cache, dec.rope, dec.block_table, max_new=8, trees=trees)
    assert logits.shape == (14, 2000)
    first = 0
    for p, tree in zip(ps, parents):
        for i in range(len(tree)):
            path, at = [], i
            while at >= 0:
                path.append(int(tokens[first + at]))
                at = tree[at]
            close(logits[first + i], single(model, torch.cat([p, torch.tensor(path[::-1], device=DEV)])))
        first += len(tree)


def test_drafts_that_are_right_wrong_and_both(model):
    ps = prompts(60, 21, 90)
    plain = tl.PagedDecoder(model, DEV, requests=3, num_pages=40)
    plain.admit(dict(enumerate(ps)))
    plain.decode(12, use_graph=False)
    want = [plain.generated(r, p.numel()) for r, p in enumerate(ps)]
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=40)
    dec.admit(dict(enumerate(ps)))
    # Row 0: the next five, in a tree beside wrong ones.  Row 1: two right, then a wrong one.  Row 2: none.
    right, wrong = want[0][1:6], (want[0][1:6] + 7) % 2000
    tree = torch.stack([wrong, right], 1).flatten()
    above = torch.tensor([-1, -1, 1, 1, 3, 3, 5, 5, 7, 7], device=DEV)
    chain = torch.cat([want[1][1:3], (want[1][3:4] + 1) % 2000, want[1][4:6]])
    got = dec.decode_drafts({0: (tree, above), 1: chain})
    assert all(1 <= g <= most for g, most in zip(got, (6, 6, 1))) and got[2] == 1
    no_page_is_lost(dec)
    for row, (p, n) in enumerate(zip(ps, got)):
        choices_are_good(dec, row, p)
        assert dec.host_lens[row] == p.numel() + n
        # The drafts are the model's own choices: they are taken up to where a rounding makes it choose otherwise.
        tokens = dec.generated(row, p.numel())
        if n < (6, 3, 1)[row]:
            logits = single(model, dec.history[row, :p.numel() + n])
            assert float(logits.max() - logits[want[row][n]]) <= 2 * BOUND * float(logits.abs().max())
        assert torch.equal(tokens[:n], want[row][:n])
    # Plain steps go on from there, captured ones too.
    dec.decode(2, use_graph=False)
    dec.capture()
    dec.decode(2)
    dec.decode_drafts({2: dec.tokens[:2]})
    dec.decode(1)
    no_page_is_lost(dec)
    for row, p in enumerate(ps):
        choices_are_good(dec, row, p)


def test_drafts_in_a_loop_and_rows_that_come_and_go(model):
    """Drafts looked up in the row's own text, the tokens that followed its last token's last place; several widths of tables."""
    ps = prompts(40, 17, 55)
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=36)
    dec.admit({0: ps[0], 1: ps[1]}, chunk=30)
    for turn in range(10):
        drafts = {}
        for row in (0, 1, 2):
            n = dec.host_lens[row]
            if n:
                before = (dec.history[row, :n] == dec.tokens[row]).nonzero()
                start = int(before[-1]) + 1 if len(before) else 0
                drafts[row] = dec.history[row, start:min(start + 3 + turn, n + 1)]
        if turn == 4:
            dec.finish(0)
            drafts.pop(0)
            dec.admit({2: ps[2]})
        dec.decode_drafts(drafts)
        no_page_is_lost(dec)
    for row, p in ((1, ps[1]), (2, ps[2])):
        choices_are_good(dec, row, p)
    dec.finish(1)
    dec.finish(2)
    assert int(dec.free_count) == 36 and dec.decode_drafts({}) == [0, 0, 0]


def test_sampled(model):
    """At a low temperature the choices are the greedy ones'; random numbers come from the generator; drawn drafts are taken."""
    ps = prompts(30, 50)
    out = []
    for _ in range(2):
        dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=30)
        dec.admit(dict(enumerate(ps)))
        g = torch.Generator(device=DEV).manual_seed(3)
        for _ in range(3):
            probs = torch.softmax(torch.randn(8, 2000, generator=g, device=DEV), -1)
            probs[2] = probs[1]  # siblings are drawn from one row
            tokens = torch.multinomial(probs, 1, generator=g)[:, 0]
            above = torch.tensor([-1, 0, 0, 1], device=DEV)
            dec.decode_drafts({0: (tokens[:4], above, probs[:4]), 1: (tokens[4:], None, probs[4:])}, temperature=0.8, generator=g)
            dec.decode_drafts({0: tokens[:3]}, temperature=1.3, generator=g)
            no_page_is_lost(dec)
        out.append(dec.history.clone())
    assert torch.equal(*out)
    cold = tl.PagedDecoder(model, DEV, requests=1, num_pages=30)
    cold.admit({0: ps[0]})
    for _ in range(4):
        cold.decode_drafts({0: cold.tokens[:1]}, temperature=1e-6)
    choices_are_good(cold, 0, ps[0])


def test_lowest_temperatures_and_drafts_of_no_tokens(model):
    """At temperatures whose quotients no float holds the choices are the greedy ones'; a draft with probabilities may be empty."""
    ps = prompts(30, 50)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=30)
    dec.admit(dict(enumerate(ps)))
    none, q = dec.tokens[:0], torch.full((1, 2000), 1 / 2000, device=DEV)
    for temperature in (1e-45, 1e-300, 1e-38):
        assert dec.decode_drafts({0: (none, none, q[:0])}, temperature=temperature) == [1, 1]
        dec.decode_drafts({0: (none, none, q[:0]), 1: (dec.tokens[:1], None, q)}, temperature=temperature)
    no_page_is_lost(dec)
    for row, p in enumerate(ps):
        choices_are_good(dec, row, p)


def test_a_step_that_fails(model, monkeypatch):
    """The rows are as before it, and go on."""
    p, = prompts(47)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=12)
    dec.admit({0: p})
    before = (dec.history.clone(), dec.tokens.clone(), dec.block_table.clone())

    def fail(*args, **kw):
        raise RuntimeError("no")

    for name in ("draft_trees", "verify_drafts", "keep_drafts"):
        with monkeypatch.context() as m, pytest.raises(RuntimeError, match="no"):
            m.setattr(ops, name, fail)
            dec.decode_drafts({0: p[:20]})
        no_page_is_lost(dec)
        for x, y in zip(before, (dec.history, dec.tokens, dec.block_table)):
            assert torch.equal(x, y)
    dec.decode_drafts({0: p[:20]})
    dec.decode(3, use_graph=False)
    no_page_is_lost(dec)
    choices_are_good(dec, 0, p)


def test_refusals(model):
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=8)
    a, = prompts(60)
    dec.admit({0: a})
    before = (dec.history.clone(), dec.context_lens.clone(), dec.free_count.clone(), dec.block_table.clone())
    t = torch.zeros(3, dtype=torch.long, device=DEV)
    for drafts, match in (({1: t}, "holds no request"), ({5: t}, "holds no request"), ({0: t.float()}, "1-D int64"),
                          ({0: t[None]}, "1-D int64"), ({0: t.cpu()}, "1-D int64"), ({0: (t, t[:2])}, "the parents"),
                          ({0: (t, t.float())}, "the parents"), ({0: t + 2000}, "outside of the vocabulary"),
                          ({0: t - 1}, "outside of the vocabulary"), ({0: (t, t - 2)}, "one before it"),
                          ({0: (t, t)}, "one before it"), ({0: (t, t + (1 << 40))}, "one before it"), ({0: t.new_zeros(64)}, "more than 63"),
                          ({0: (t, t - 1, torch.zeros(3, 7, device=DEV))}, "the probabilities"),
                          ({0: (t, t - 1, torch.zeros(3, 2000, device=DEV))}, "need a temperature")):
        with pytest.raises(ValueError, match=match):
            dec.decode_drafts(drafts)
    for draft in ([1, 2], (t, t, t, t), (), (None, t), (t, [-1, 0, 1]), {1: t}):
        with pytest.raises(TypeError, match="must be tokens"):
            dec.decode_drafts({0: draft})
    for temperature in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            dec.decode_drafts({}, temperature=temperature)
    small = tl.PagedDecoder(model, DEV, requests=2, num_pages=4)
    small.admit({0: a})
    with pytest.raises(ValueError, match="pages are needed"):
        small.decode_drafts({0: t.new_zeros(20)})
    long = tl.PagedDecoder(model, DEV, requests=1, num_pages=20)
    long.admit({0: prompts(190)[0]})
    with pytest.raises(ValueError, match="more than max_seq"):
        long.decode_drafts({0: t.new_zeros(30)})
    dec.admit({1: a})
    with pytest.raises(ValueError, match="or none"):
        dec.decode_drafts({0: (t, None, torch.zeros(3, 2000, device=DEV)), 1: t}, temperature=1.0)
    dec.finish(1)
    for x, y in zip(before, (dec.history, dec.context_lens, dec.free_count, dec.block_table)):
        assert torch.equal(x[0], y[0])
    assert dec.host_lens == [60, 0]


def test_drafts_of_one_parent_come_with_one_row(model):
    """Tokens behind one parent whose probabilities differ were not drawn as the rule of acceptance takes them to be: refused, and
    nothing is changed."""
    ps = prompts(30, 50)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=30)
    dec.admit(dict(enumerate(ps)))
    before = (dec.history.clone(), dec.context_lens.clone(), dec.free_count.clone(), dec.block_table.clone(), dec.tokens.clone())
    g = torch.Generator(device=DEV).manual_seed(4)
    probs = torch.softmax(torch.randn(5, 2000, generator=g, device=DEV), -1)
    tokens = torch.multinomial(probs, 1, generator=g)[:, 0]
    chain = (tokens[:2], None, probs[:2])
    for above in ([-1, -1, 0, 1, 2], [-1, 0, 1, 1, 3], [-1, 0, 1, 2, -1]):
        above = torch.tensor(above, device=DEV)
        for drafts in ({0: (tokens, above, probs), 1: chain}, {0: chain, 1: (tokens, above, probs)}):
            with pytest.raises(ValueError, match="one parent"):
                dec.decode_drafts(drafts, temperature=1.0, generator=g)
    for x, y in zip(before, (dec.history, dec.context_lens, dec.free_count, dec.block_table, dec.tokens)):
        assert torch.equal(x, y)
    probs[4], probs[2] = probs[0], probs[1]
    dec.decode_drafts({0: (tokens, torch.tensor([-1, 0, 0, 1, -1], device=DEV), probs), 1: chain}, temperature=1.0, generator=g)
    no_page_is_lost(dec)


def test_sampled_from_scores_that_are_infinite(model, monkeypatch):
    """A score of infinity has all of the probability, as it is the largest for greedy steps; scores that are all -inf are equal."""
    p, = prompts(30)
    forward = model.forward_paged

    def infinite(*args, **kw):
        logits = forward(*args, **kw)
        if kw.get("trees") is not None:
            logits[:] = -float("inf")
            logits[:, 7] = high
        return logits

    monkeypatch.setattr(model, "forward_paged", infinite)
    dec = tl.PagedDecoder(model, DEV, requests=1, num_pages=30)
    dec.admit({0: p})
    t = torch.tensor([7, 7, 8], device=DEV)
    for high in (float("inf"), 3.0):
        for temperature in (0.0, 1e-20, 0.8, 1e30):
            assert dec.decode_drafts({0: t}, temperature=temperature) == [3]
            assert dec.generated(0, 30)[-3:].tolist() == [7, 7, 7]
    high = -float("inf")
    g = torch.Generator(device=DEV).manual_seed(6)
    assert len({dec.decode_drafts({}, temperature=1.0, generator=g)[0] * int(dec.tokens[0]) for _ in range(8)}) > 4
    no_page_is_lost(dec)


def test_rows_of_probabilities_stand_at_the_parents(model, monkeypatch):
    """What verify_drafts is given: each node's row of the draft is what its children were drawn from, zeros without children."""
    ps = prompts(30, 50, 20)
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=30)
    dec.admit(dict(enumerate(ps)))
    seen, verify = [], ops.verify_drafts

    def spy(*args, **kw):
        seen.append(kw["draft"].clone())
        return verify(*args, **kw)

    monkeypatch.setattr(ops, "verify_drafts", spy)
    rows = torch.softmax(torch.randn(7, 2000, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV), -1)
    tokens = torch.arange(8, device=DEV)
    # Row 0: two tokens behind the last one, one behind each of them, two behind token 2.  Row 2: a chain of two.
    dec.decode_drafts({0: (tokens[:6], torch.tensor([-1, -1, 0, 1, 2, 2], device=DEV), rows[[0, 0, 1, 2, 3, 3]]),
                       2: (tokens[:2], None, rows[4:6])}, temperature=0.9)
    want = torch.zeros(7 + 1 + 3, 2000, device=DEV)
    want[0], want[1], want[2], want[3] = rows[0], rows[1], rows[2], rows[3]
    want[8], want[9] = rows[4], rows[5]
    assert len(seen) == 1 and torch.equal(seen[0], want)
    no_page_is_lost(dec)


def test_tokens_that_only_the_draft_has_are_rejected(model, monkeypatch):
    """A draft that is sure of tokens that the model never takes: none stays, in a chain and behind an accepted token."""
    ps = prompts(30)
    forward = model.forward_paged

    def without(*args, **kw):  # token 5 has no probability, token 6 nearly all
        logits = forward(*args, **kw)
        if kw.get("trees") is not None:
            logits[:, 5], logits[:, 6] = float("-inf"), logits.amax(-1) + 60
        return logits

    monkeypatch.setattr(model, "forward_paged", without)
    sure = torch.zeros(2, 2000, device=DEV)
    sure[0, 6] = sure[1, 5] = 1.0
    dec = tl.PagedDecoder(model, DEV, requests=1, num_pages=30)
    dec.admit({0: ps[0]})
    t = torch.tensor([6, 5], device=DEV)
    for _ in range(5):
        assert dec.decode_drafts({0: (t, None, sure)}, temperature=1.0) == [2]
        assert dec.generated(0, 30)[-2:].tolist() == [6, 6]
        assert dec.decode_drafts({0: (t[[1, 1]], t.new_full((2,), -1), sure[[1, 1]])}, temperature=1.0) == [1]
        assert dec.generated(0, 30)[-1].item() == 6
