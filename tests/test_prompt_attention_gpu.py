"""Causal attention of packed prompts against float64 (needs a GPU): head layouts and sizes that fill tiles and do not,
lengths at the edges of rows and keys, empty sequences, strided views, infinities and NaN in keys that a
row does not attend to."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from attention_cases import attend64, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lens, heads, kv_heads, d, dtype, pad=0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * heads + d + sum(lens))
    t = sum(lens) + pad
    qk = torch.randn(t, heads + kv_heads, d, generator=g, device=DEV).to(dtype)
    qkv = torch.randn(t, heads + 2 * kv_heads, d, generator=g, device=DEV).to(dtype)
    return qk[:, :heads], qk[:, heads:], qkv[:, heads + kv_heads:], offsets(lens, DEV)


def against64(lens, q, k, v, out, scale=None):
    at, worst = 0, 0.0
    for n in lens:
        if n:
            ref, bound = attend64(q[at:at + n], k[at:at + n], v[at:at + n], scale=scale)
            worst = max(worst, check(out[at:at + n], ref, bound, f"sequence of {n} at {at}"))
        at += n
    return worst


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 4, 64), (12, 2, 128), (8, 8, 96), (16, 1, 80), (4, 2, 256),
                                              (3, 3, 8), (5, 1, 136), (2, 1, 200), (6, 2, 40)])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0, 17, 1], [64], [65, 63, 130], [300, 0, 7]],
                         ids=["one", "short", "tile", "edges", "longer"])
def test_against_float64(dtype, heads, kv_heads, d, lens):
    q, k, v, cu = make(lens, heads, kv_heads, d, dtype)
    against64(lens, q, k, v, ops.prompt_attention(q, k, v, cu))


@pytest.mark.parametrize("lens", [[1531], [2049, 1, 700], [1] * 200, [3, 0] * 70], ids=["odd", "long", "ones", "many"])
def test_lengths(lens):
    q, k, v, cu = make(lens, 8, 2, 64, torch.float16)
    against64(lens, q, k, v, ops.prompt_attention(q, k, v, cu))


def test_scale_and_large_scores():
    # Scores of hundreds, the largest ones late and early: the maximum moves by far more than its slack.
    lens = [200, 90]
    q, k, v, cu = make(lens, 4, 2, 64, torch.float16)
    k = (k * torch.linspace(0.1, 20, k.shape[0], device=DEV)[:, None, None]).half()
    against64(lens, q, k, v, ops.prompt_attention(q, k, v, cu, scale=0.5), scale=0.5)
    k = k.flip(0).contiguous()
    against64(lens, q, k, v, ops.prompt_attention(q, k, v, cu, scale=0.01), scale=0.01)


def test_rows_behind_the_last_sequence():
    lens, pad = [9, 40], 150
    q, k, v, cu = make(lens, 4, 2, 64, torch.bfloat16, pad)
    out = ops.prompt_attention(q, k, v, cu)
    assert bool((out[49:] == 0).all())
    mine = torch.full((49 + pad, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ops.prompt_attention(q, k, v, cu, out=mine)
    assert got.data_ptr() == mine.data_ptr() and bool((mine[49:] == 7).all())
    assert torch.equal(mine[:49], out[:49])


def test_strides_and_output_layout():
    lens = [33, 70]
    q, k, v, cu = make(lens, 4, 2, 64, torch.float16)
    ref = ops.prompt_attention(q, k, v, cu)
    # Heads outermost, odd element offsets (copied), an output inside a larger tensor.
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    k2 = torch.zeros(k.numel() + 3, dtype=k.dtype, device=DEV)[3:].view(k.shape)
    k2.copy_(k)
    big = torch.zeros(103, 4, 80, dtype=torch.float16, device=DEV)
    got = ops.prompt_attention(q2, k2, v, cu, out=big[..., 8:72])
    assert torch.equal(got, ref) and bool((big[..., :8] == 0).all()) and bool((big[..., 72:] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [64, 72, 128, 256])
def test_later_keys_do_not_reach_a_row(dtype, bad, d):
    """Key 40 of 90 is not finite: rows before it are what they are without it, rows from it on are not finite
    where the value is met."""
    q, k, v, cu = make([90, 20], 4, 2, d, dtype)
    k, v = k.contiguous(), v.contiguous()
    clean = ops.prompt_attention(q, k, v, cu)
    v2 = v.clone()
    v2[40, 1, 3] = bad
    out = ops.prompt_attention(q, k, v2, cu)
    assert torch.equal(out[:40], clean[:40]) and torch.equal(out[90:], clean[90:])
    assert torch.equal(out[:90, :2], clean[:90, :2])  # the other KV head
    hit = out[40:90, 2:, 3]
    assert bool(hit.isnan().all()) if bad != bad else bool((hit == bad).all())
    rest = torch.cat([out[40:90, 2:, :3], out[40:90, 2:, 4:]], -1)
    assert torch.equal(rest, torch.cat([clean[40:90, 2:, :3], clean[40:90, 2:, 4:]], -1))
    k2 = k.clone()
    k2[40, 1] = bad
    out = ops.prompt_attention(q, k2, v, cu)
    assert torch.equal(out[:40], clean[:40]) and torch.equal(out[90:], clean[90:])


def test_captured_and_replayed():
    """A captured call follows the lengths it is given, and equals the eager one on every replay."""
    q, k, v, cu = make([100, 28], 8, 2, 64, torch.float16)
    ops.prompt_attention(q, k, v, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.prompt_attention(q, k, v, cu)
    for lens in ([100, 28], [1, 127], [0, 128], [64, 10]):
        cu.copy_(offsets(lens, DEV))
        want = ops.prompt_attention(q, k, v, cu)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_another_stream():
    q, k, v, cu = make([700], 8, 2, 64, torch.float16)
    want = ops.prompt_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.prompt_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_many_small_probabilities(dtype):
    """One key far above the others: their probabilities are subnormal in fp16 against it, and add up to as much
    as it has."""
    n = 3001
    q, k, v, cu = make([n], 2, 1, 64, dtype)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0
    k = k.contiguous() * 0.01
    k[0, 0, 0] = 8.0 * 1.29  # score 10.3: the others' probabilities are about 3.3e-5 of its
    against64([n], q, k, v, ops.prompt_attention(q, k, v, cu))


def test_far_apart_tokens():
    """Keys 128 MiB apart: offsets within a copy pass 31 bits, those of tokens 32."""
    n, step = 33, 1 << 26
    q, k, v, cu = make([n], 2, 1, 64, torch.float16)
    want = ops.prompt_attention(q, k, v, cu)
    big = torch.empty((n - 1) * step + 64, dtype=torch.float16, device=DEV)
    far = big.as_strided((n, 1, 64), (step, 64, 1))
    far.copy_(k)
    assert torch.equal(ops.prompt_attention(q, far, v, cu), want)
    far.copy_(v)
    assert torch.equal(ops.prompt_attention(q, k, far, cu), want)
    with pytest.raises(ValueError, match="token strides"):
        big.resize_(0)
        big = torch.empty((n - 1) * (step + 8) + 64, dtype=torch.float16, device=DEV)
        ops.prompt_attention(q, big.as_strided((n, 1, 64), (step + 8, 64, 1)), v, cu)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (4, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("lens", [[2000], [6000], [900, 1, 1700], [40] * 30 + [333] * 20, [1, 2500, 7, 0, 600]],
                         ids=["groups", "cut", "few", "ordered", "uneven"])
def test_every_plan(heads, kv_heads, d, lens):
    """Row tiles whole, shared by two groups of wavefronts, cut over workgroups, and in the order of their lengths: prompts
    of few and many row tiles, against 64 bits."""
    q, k, v, cu = make(lens, heads, kv_heads, d, torch.bfloat16, pad=3)
    out = ops.prompt_attention(q, k, v, cu)
    against64(lens, q, k, v, out)
    assert bool((out[sum(lens):] == 0).all())


def test_registered_op():
    q, k, v, cu = make([20, 9], 4, 2, 64, torch.float16)
    torch.library.opcheck(ops._prompt_attention_op, (q, k, v, cu, 0.125), test_utils=("test_schema", "test_faketensor"))
    assert torch.equal(torch.ops.kernelforge.prompt_attention(q, k, v, cu, 0.125), ops.prompt_attention(q, k, v, cu))
