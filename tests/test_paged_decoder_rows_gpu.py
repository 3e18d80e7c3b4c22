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
