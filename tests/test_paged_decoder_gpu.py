"""The paged decoder (needs a GPU): its logits against the single-stream model's, prompts in chunks against whole
ones, graph replays against eager steps, rows that come and go.

Two paths through the same fp16 model differ by roundings only.  Each layer rounds its residual stream's value about ten
times on the way (norm, projections, RoPE, attention, output, gate, up, product, down, two sums), each by at most
2^-11 of the value, so logits of L layers are held to 10 (L + 1) 2^-11 of the largest one.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from kernelforge import tinyllama as tl

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
LAYERS = 3
BOUND = 10 * (LAYERS + 1) * 2.0 ** -11


def config():
    return dataclasses.replace(tl.TinyLlamaConfig(), layers=LAYERS, max_seq=200, vocab=2000)


@pytest.fixture(scope="module", params=["fused", "separate", "fp16"])
def model(request):
    cfg = config()
    if request.param == "fp16":
        with torch.device(DEV):
            m = tl.TinyLlama(cfg)
        return m.init_random_(4).half().eval()
    return tl.build_int4_model(cfg, DEV, seed=4, fuse=request.param == "fused")


def prompts(*lens):
    g = torch.Generator(device=DEV).manual_seed(sum(lens))
    return [torch.randint(0, 2000, (n,), generator=g, device=DEV) for n in lens]


@torch.no_grad()
def single(model, tokens):
    """Logits after the last token from the single-stream forward."""
    cfg = model.cfg
    pos = torch.arange(tokens.numel(), device=DEV)
    rope = tl._rope_tables(cfg, DEV)
    return model(tokens, pos, model.new_cache(DEV), rope, tl.causal_mask(pos, cfg.max_seq))


@torch.no_grad()
def next_logits(dec, tokens, new, max_new, whole):
    """One forward of the decoder's model without advancing anything but pages and cache."""
    from kernelforge import ops

    lens = torch.tensor(new, dtype=torch.int32, device=DEV)
    step = ops.paged_tables(dec.block_table, dec.context_lens, lens, dec.free_pages, dec.free_count,
                            block_size=dec.block_size, max_tokens=sum(new))
    return dec.model.forward_paged(tokens, step, dec.cache, dec.rope, dec.block_table, max_new=max_new, whole_prompts=whole)


def close(a, b):
    assert float((a.float() - b.float()).abs().max()) <= BOUND * float(b.float().abs().max())


def test_logits_against_the_single_stream(model):
    ps = prompts(70, 1, 33, 150)
    dec = tl.PagedDecoder(model, DEV, requests=4, num_pages=60)
    tokens = torch.cat(ps)
    for whole in (True, False):
        logits = next_logits(dec, tokens, [p.numel() for p in ps], 150, whole)
        for row, p in enumerate(ps):
            close(logits[row], single(model, p))


def test_chunks_and_steps_against_the_single_stream(model):
    ps = prompts(90, 17, 64)
    dec = tl.PagedDecoder(model, DEV, requests=4, num_pages=60, block_size=32)
    dec.admit({0: ps[0], 2: ps[1], 3: ps[2]}, chunk=40)
    dec.decode(3, use_graph=False)
    for row, p in ((0, ps[0]), (2, ps[1]), (3, ps[2])):
        seen = dec.history[row, :dec.host_lens[row]]
        assert torch.equal(seen[:p.numel()], p) and seen.numel() == p.numel() + 3
        assert int(dec.context_lens[row]) == seen.numel()
        # Each generated token is as good a choice as the single stream's, to within the bound.
        for at in range(p.numel(), seen.numel() + 1):
            logits = single(model, dec.history[row, :at])
            best, chosen = logits.max(), logits[dec.history[row, at]]
            assert float(best - chosen) <= 2 * BOUND * float(logits.abs().max())
    assert int(dec.free_count) == 60 - sum(-(-n // 32) for n in dec.host_lens)


def test_graph_steps_equal_eager_ones(model):
    ps = prompts(40, 9, 120)
    out = []
    for use_graph in (False, True):
        dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=40)
        dec.admit(dict(enumerate(ps)))
        if use_graph:
            dec.capture()
        for _ in range(3):  # replays with eager work between them
            dec.decode(4, use_graph=use_graph)
            torch.randn(1000, device=DEV).sum().item()
        out.append((dec.history.clone(), dec.context_lens.clone(), dec.free_count.clone()))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_rows_come_and_go(model):
    """A row's tokens do not depend on the others: alone, beside others, and in a row and pages that were used before."""
    ps = prompts(50, 21, 77)
    alone = []
    for p in ps:
        dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=30)
        dec.admit({1: p}, chunk=200)
        dec.decode(6, use_graph=False)
        alone.append(dec.generated(1, p.numel()))
    dec = tl.PagedDecoder(model, DEV, requests=3, num_pages=30)
    dec.admit({0: ps[0]}, chunk=200)
    dec.admit({1: ps[1]}, chunk=200)
    dec.decode(2, use_graph=False)
    dec.finish(0)
    dec.admit({0: ps[2]}, chunk=200)
    dec.decode(4, use_graph=False)
    # Batches of other sizes run other kernels for the projections, so tokens are compared where the choice is clear.
    for row, p, want in ((1, ps[1], alone[1]), (0, ps[2], alone[2])):
        got = dec.generated(row, p.numel())
        n = min(got.numel(), want.numel())
        for i in range(n):
            if got[i] == want[i]:
                continue
            logits = single(model, dec.history[row, :p.numel() + i])
            assert float(logits.max() - logits[got[i]]) <= 2 * BOUND * float(logits.abs().max())
            break
    assert sorted(dec.free_pages[:int(dec.free_count)].tolist() +
                  dec.block_table[dec.block_table >= 0].tolist()) == list(range(30))


def test_refusals(model):
    dec = tl.PagedDecoder(model, DEV, requests=2, num_pages=8)
    a, b = prompts(60, 70)
    with pytest.raises(ValueError, match="capture first"):
        dec.decode(1)
    with pytest.raises(ValueError, match="pages are needed"):
        dec.admit({0: a, 1: b})
    dec.admit({0: a})
    with pytest.raises(ValueError, match="holds a request"):
        dec.admit({0: b})
    with pytest.raises(ValueError, match="is empty"):
        dec.admit({1: a[:0]})
    with pytest.raises(ValueError, match="holds no request"):
        dec.finish(1)
    with pytest.raises(ValueError, match="more than max_seq"):
        dec.decode(200, use_graph=False)
    with pytest.raises(ValueError, match="pages are needed"):
        dec.decode(100, use_graph=False)
    assert dec.host_lens == [60, 0] and int(dec.context_lens[0]) == 60
