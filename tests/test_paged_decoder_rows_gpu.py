"""Rows of the paged decoder that come and go, around its captured step (needs a GPU)."""

from __future__ import annotations

import pytest
import torch

from kernelforge import tinyllama as tl

from test_paged_decoder_gpu import BOUND, DEV, model, prompts, single  # noqa: F401  (model: a fixture)

pytestmark = pytest.mark.gpu

STATE = ("cache", "block_table", "context_lens", "active", "free_pages", "free_count", "tokens", "history")


def state(dec):
    return {name: getattr(dec, name).clone() for name in STATE}


def same(dec, before):
    for name, old in before.items():
        assert torch.equal(getattr(dec, name), old), name


def test_a_finished_row_keeps_its_history(model):
    a, b = prompts(20, 9)
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=20)
    dec.admit({0: a, 1: b})
    dec.decode(3, use_graph=False)
    want = dec.history[0].clone()
    dec.finish(0)
    dec.decode(2, use_graph=False)
    assert torch.equal(dec.history[0], want) and torch.equal(dec.history[0, :20], a)


def test_capture_needs_no_room(model):
    """Rows one token below max_seq and without a free page are captured, a large cache without a second one, and nothing
    of the requests changes."""
    last = model.cfg.max_seq - 1
    a, b = prompts(last, 16)
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=14)
    dec.admit({0: a, 2: b})
    assert int(dec.free_count) == 0
    before, lens = state(dec), list(dec.host_lens)
    dec.capture()
    same(dec, before)
    assert dec.host_lens == lens
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=8000)
    dec.admit({0: b})
    dec.decode(1, use_graph=False)
    size = dec.cache.numel() * dec.cache.element_size()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dec.capture()
    assert torch.cuda.max_memory_allocated() - held < size // 2


def test_a_capture_that_fails_leaves_the_requests(model, monkeypatch):
    a, b = prompts(20, 9)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=20)
    dec.admit({0: a, 1: b})
    before = state(dec)
    forward = model.forward_paged
    calls = []

    def failing(*args, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("planted")
        return forward(*args, **kw)
    monkeypatch.setattr(model, "forward_paged", failing)
    with pytest.raises(RuntimeError, match="planted"):
        dec.capture()
    same(dec, before)
    assert dec.graph is None


def test_a_negative_number_of_steps(model):
    (a,) = prompts(30)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=8)
    dec.admit({0: a})
    with pytest.raises(ValueError, match="steps"):
        dec.decode(-20, use_graph=False)
    assert dec.host_lens == [30, 0] and torch.equal(dec.decode(0, use_graph=False), dec.history)
    dec.finish(0)
    assert int(dec.free_count) == 8 and sorted(dec.free_pages.tolist()) == list(range(8))


@pytest.mark.parametrize("row", [-1, 2, 7])
def test_rows_that_there_are_not(model, row):
    a, b = prompts(20, 9)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=20)
    before = state(dec)
    for prompts_of in ({row: a}, {0: b, row: a}):
        with pytest.raises(ValueError, match=f"no row {row}"):
            dec.admit(prompts_of)
    same(dec, before)
    assert dec.host_lens == [0, 0]


def test_prompts_of_other_shapes(model):
    (a,) = prompts(20)
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=20)
    before = state(dec)
    for prompt in (a[None], a.float(), a.cpu()):
        with pytest.raises(ValueError, match="prompt of row 1"):
            dec.admit({1: prompt}, chunk=7)
    same(dec, before)


@torch.no_grad()
def test_whole_prompts_beside_running_rows(model, monkeypatch):
    """They are whole prompts whatever the other rows hold, which have no new tokens then."""
    a, b, c = prompts(40, 70, 33)
    dec = tl.PagedDecoder(model, DEV, requests=4, num_pages=40)
    dec.admit({1: a})
    dec.decode(2, use_graph=False)
    running = dec.history[1].clone()
    calls = []
    for name in ("prompt_attention", "paged_attention"):
        def counted(*args, op=getattr(tl.ops, name), name=name, **kw):
            calls.append(name)
            return op(*args, **kw)
        monkeypatch.setattr(tl.ops, name, counted)
    dec.admit({0: b, 3: c})
    assert calls == ["prompt_attention"] * model.cfg.layers
    assert torch.equal(dec.history[1], running) and dec.host_lens == [70, 42, 0, 33]
    dec.decode(3, use_graph=False)
    for row, p in ((0, b), (1, a), (3, c)):
        for at in range(p.numel(), dec.host_lens[row] + 1):
            logits = single(model, dec.history[row, :at])
            best, chosen = logits.max(), logits[dec.history[row, at]]
            assert float(best - chosen) <= 2 * BOUND * float(logits.abs().max())


def fail_at(monkeypatch, model, call):
    """The model's call number `call` from here on raises, before it computes anything."""
    forward, calls = model.forward_paged, []

    def failing(*args, **kw):
        calls.append(1)
        if len(calls) == call:
            raise RuntimeError("planted")
        return forward(*args, **kw)
    monkeypatch.setattr(model, "forward_paged", failing)


def test_an_admission_that_fails(model, monkeypatch):
    """Its rows are free again, with their pages; the others go on."""
    a, b, c = prompts(40, 70, 33)
    outs = []
    for fails in (False, True):
        dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=30)
        dec.admit({1: a})
        dec.decode(2, use_graph=False)
        if fails:
            with monkeypatch.context() as m:
                fail_at(m, model, 3)
                with pytest.raises(RuntimeError, match="planted"):
                    dec.admit({0: b, 2: c}, chunk=20)
            assert dec.host_lens == [0, 42, 0] and dec.context_lens.tolist() == [0, 42, 0]
            assert int(dec.free_count) == 27 and bool((dec.block_table[[0, 2]] == -1).all())
        dec.admit({0: b, 2: c}, chunk=20)
        dec.decode(4, use_graph=False)
        outs.append([dec.generated(r, p.numel()) for r, p in ((0, b), (1, a), (2, c))])
        assert int(dec.free_count) == 30 - sum(-(-n // 16) for n in dec.host_lens)
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_a_step_that_fails(model, monkeypatch):
    """The steps before it count, on the host as on the device, and the next call goes on from there."""
    a, b = prompts(30, 14)
    outs = []
    for fails in (False, True):
        dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=12)
        dec.admit({0: a, 1: b})
        done = 0
        if fails:
            with monkeypatch.context() as m:
                fail_at(m, model, 4)  # the step in which both rows take a new page
                with pytest.raises(RuntimeError, match="planted"):
                    dec.decode(6, use_graph=False)
            done = 3
            assert dec.host_lens == dec.context_lens.tolist() == [33, 17]
        dec.decode(6 - done, use_graph=False)
        assert dec.host_lens == dec.context_lens.tolist() == [36, 20]
        assert int(dec.free_count) == 12 - 3 - 2
        outs.append(dec.history.clone())
    assert torch.equal(*outs)


def test_rows_come_and_go_around_a_captured_step(model):
    """One capture, then requests that end and begin between its replays: what eager steps of the same rows give, with
    the model's other work between the replays."""
    ps = prompts(50, 21, 77, 5)
    outs = []
    for use_graph in (False, True):
        dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=30)
        if use_graph:
            dec.capture()  # before any request
        dec.admit({0: ps[0], 1: ps[1]})
        dec.decode(3, use_graph=use_graph)
        dec.finish(0)
        dec.decode(2, use_graph=use_graph)
        dec.admit({0: ps[2]}, chunk=30)
        dec.decode(2, use_graph=use_graph)
        dec.admit({2: ps[3]})
        dec.decode(5, use_graph=use_graph)
        outs.append({**state(dec), "lens": torch.tensor(dec.host_lens)})
        assert dec.host_lens == [84, 33, 10] == dec.context_lens.tolist()
    for name in outs[0]:
        if name != "cache":
            assert torch.equal(outs[0][name], outs[1][name]), name
