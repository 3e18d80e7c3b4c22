"""The paged-cache operators without a GPU: what they refuse, in Python and at the C ABI (before any launch), and the
shapes of their registered ops under a tracer."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kernelforge import _lib, ops

H = torch.float16


def attention_args(dtype=H, t=6, heads=4, kv=2, d=64, block=16, b=2, width=3, pages=5, device="cpu"):
    i32 = dict(dtype=torch.int32, device=device)
    return dict(q=torch.zeros(t, heads, d, dtype=dtype, device=device),
                cache_k=torch.zeros(pages, kv, block, d, dtype=dtype, device=device),
                cache_v=torch.zeros(pages, kv, block, d, dtype=dtype, device=device),
                block_table=torch.zeros(b, width, **i32), cu_new=torch.zeros(b + 1, **i32), seq_lens=torch.zeros(b, **i32))


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(6, 4, 64)), TypeError, "fp16 or bf16"),
    (dict(q=torch.zeros(6, 256, dtype=H)), TypeError, "3-D"),
    (dict(q=torch.zeros(6, 3, 64, dtype=H)), ValueError, "must divide"),
    (dict(q=torch.zeros(6, 4, 32, dtype=H)), ValueError, "head_dim"),
    (dict(cache_v=torch.zeros(5, 2, 16, 64)), TypeError, "cache_v must have the type"),
    (dict(cache_v=torch.zeros(5, 2, 32, 64, dtype=H)), ValueError, "must be .num_pages"),
    (dict(cache_k=torch.zeros(0, 2, 16, 64, dtype=H), cache_v=torch.zeros(0, 2, 16, 64, dtype=H)), ValueError, "empty"),
    (dict(cache_k=torch.zeros(5, 2, 24, 64, dtype=H), cache_v=torch.zeros(5, 2, 24, 64, dtype=H)), ValueError, "power of two"),
    (dict(cache_k=torch.zeros(5, 2, 8, 64, dtype=H), cache_v=torch.zeros(5, 2, 8, 64, dtype=H)), ValueError, "power of two"),
    (dict(cache_k=torch.zeros(5, 2, 64, 16, dtype=H).transpose(2, 3)), ValueError, "contiguous last dimension"),
    (dict(cache_k=torch.zeros(5, 2, 16, 68, dtype=H)[..., :64]), ValueError, "multiples of 8"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "block_table"),
    (dict(cu_new=torch.zeros(2, dtype=torch.int32)), ValueError, "cu_new"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(max_new=0), ValueError, "max_new"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(scale=-1.0), ValueError, "scale"),
    (dict(out=torch.zeros(6, 4, 64)), ValueError, "out must be"),
    (dict(out=torch.zeros(6, 4, 65, dtype=H)[..., 1:]), ValueError, "out must be"),
    (dict(out=torch.zeros(6, 1, 64, dtype=H).expand(6, 4, 64)), ValueError, "none of them 0"),
])
def test_paged_attention_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.paged_attention(**{**attention_args(), **change})


def test_no_requests_and_no_gpu():
    a = attention_args(b=0)
    with pytest.raises(ValueError, match="at least one request"):
        ops.paged_attention(**a)
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.paged_attention(**attention_args())


def prompt_args():
    return dict(q=torch.zeros(6, 4, 64, dtype=H), k=torch.zeros(6, 2, 64, dtype=H), v=torch.zeros(6, 2, 64, dtype=H),
                cu_seqlens=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(6, 4, 64, dtype=torch.float64)), TypeError, "fp16 or bf16"),
    (dict(k=torch.zeros(5, 2, 64, dtype=H)), ValueError, "k and v must be"),
    (dict(v=torch.zeros(6, 1, 64, dtype=H)), ValueError, "k and v must be"),
    (dict(k=torch.zeros(6, 3, 64, dtype=H), v=torch.zeros(6, 3, 64, dtype=H)), ValueError, "must divide"),
    (dict(k=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), TypeError, "type of q"),
    (dict(q=torch.zeros(6, 4, 60, dtype=H), k=torch.zeros(6, 2, 60, dtype=H), v=torch.zeros(6, 2, 60, dtype=H)), ValueError,
     "multiple of 8"),
    (dict(q=torch.zeros(6, 4, 264, dtype=H), k=torch.zeros(6, 2, 264, dtype=H), v=torch.zeros(6, 2, 264, dtype=H)),
     ValueError, "up to 256"),
    (dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)), ValueError, "B >= 1"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), ValueError, "cu_seqlens"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(out=torch.zeros(5, 4, 64, dtype=H)), ValueError, "out must be"),
    (dict(), RuntimeError, "CUDA device"),
])
def test_prompt_attention_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.prompt_attention(**{**prompt_args(), **change})


def rope_args():
    return dict(qkv=torch.zeros(6, 8 * 64, dtype=H), cos=torch.zeros(9, 64), sin=torch.zeros(9, 64),
                positions=torch.zeros(6, dtype=torch.int64), slots=torch.zeros(6, dtype=torch.int64),
                cache_k=torch.zeros(5, 2, 16, 64, dtype=H), cache_v=torch.zeros(5, 2, 16, 64, dtype=H), heads=4)


@pytest.mark.parametrize("change,error,match", [
    (dict(qkv=torch.zeros(6, 512)), TypeError, "fp16 or bf16"),
    (dict(qkv=torch.zeros(6, 520, dtype=H)), ValueError, "columns"),
    (dict(heads=3), ValueError, "must divide"),
    (dict(cos=torch.zeros(9, 64, dtype=H)), ValueError, "cos"),
    (dict(sin=torch.zeros(8, 64)), ValueError, "sin"),
    (dict(cos=torch.zeros(0, 64), sin=torch.zeros(0, 64)), ValueError, "cos"),
    (dict(positions=torch.zeros(6, dtype=torch.int32)), ValueError, "positions"),
    (dict(slots=torch.zeros(7, dtype=torch.int64)), ValueError, "slots"),
    (dict(cache_k=torch.zeros(5, 2, 16, 64)), TypeError, "cache_k"),
    (dict(cache_v=torch.zeros(1, 2, 16, 64, dtype=H).expand(5, 2, 16, 64)), ValueError, "must not be expanded"),
    (dict(), RuntimeError, "CUDA device"),
])
def test_rope_paged_cache_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.rope_paged_cache(**{**rope_args(), **change})


def tables_args():
    i32 = dict(dtype=torch.int32)
    return dict(block_table=torch.zeros(2, 3, **i32), context_lens=torch.zeros(2, **i32), new_lens=torch.zeros(2, **i32),
                free_pages=torch.zeros(4, **i32), free_count=torch.zeros(1, **i32), block_size=16, max_tokens=8)


@pytest.mark.parametrize("change,error,match", [
    (dict(block_table=torch.zeros(6, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError, "block_table"),
    (dict(context_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "context_lens"),
    (dict(new_lens=torch.zeros(2)), ValueError, "new_lens"),
    (dict(free_pages=torch.zeros(4, dtype=torch.int64)), ValueError, "free_pages"),
    (dict(free_count=torch.zeros(2, dtype=torch.int32)), ValueError, "free_count"),
    (dict(block_size=17), ValueError, "power of two"),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), ValueError, "must not overlap"),
    (dict(max_tokens=-1), ValueError, "max_tokens"),
    (dict(), RuntimeError, "CUDA device"),
])
def test_paged_tables_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.paged_tables(**{**tables_args(), **change})


@pytest.mark.parametrize("op,args", [(ops.paged_attention, attention_args), (ops.prompt_attention, prompt_args),
                                     (ops.rope_paged_cache, rope_args)])
def test_gradients_and_transforms_are_refused(op, args):
    a = args()
    first = next(iter(a))
    a[first] = a[first].requires_grad_()
    with pytest.raises(RuntimeError, match="inference only"):
        op(**a)
    a = args()
    x = a.pop(first)
    with pytest.raises(RuntimeError, match="cannot be transformed"):
        torch.func.vmap(lambda y: op(**{first: y}, **a))(x[None])


def test_shapes_under_a_tracer():
    with FakeTensorMode(), torch.no_grad():
        a = attention_args(device="cuda")
        assert ops.paged_attention(**a).shape == (6, 4, 64)
        with pytest.raises(RuntimeError, match="no traceable form"):
            ops.paged_attention(**a, out=torch.empty_like(a["q"]))
        a = {k: v.cuda() for k, v in prompt_args().items()}
        assert ops.prompt_attention(**a).shape == (6, 4, 64)
        a = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in rope_args().items()}
        q, k = ops.rope_paged_cache(**a)
        assert q.shape == (6, 4, 64) and k.shape == (6, 2, 64)
        a = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in tables_args().items()}
        step = ops.paged_tables(**a)
        assert [t.shape[0] for t in step] == [3, 2, 8, 8, 1] and step.slots.dtype == torch.int64


def _err(status, match):
    assert status != 0
    assert re.search(match, _lib.last_error()), _lib.last_error()


def _struct(cls, **change):
    """A struct whose checks pass up to what `change` breaks: pointers that are never dereferenced."""
    values = dict(tokens=4, seqs=2, heads=4, kv_heads=2, head_dim=64, dtype=1, scale=0.125, table_width=3, num_pages=5,
                  block_size=16, max_pos=9, free_capacity=4, max_tokens=8)
    out = cls()
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p:
            setattr(out, name, 0x1000 * (1 + [n for n, _ in cls._fields_].index(name)))
        elif kind is ctypes.c_int64:
            setattr(out, name, 64)
        elif name in values:
            setattr(out, name, values[name])
    for name, value in change.items():
        setattr(out, name, value)
    return out


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "non-null"), (dict(cu_seqlens=None), "non-null"), (dict(k=0x1008), "16-byte"), (dict(seqs=0), "seqs >= 1"),
    (dict(tokens=-1), "tokens >= 0"), (dict(kv_heads=3), "divide"), (dict(head_dim=12), "multiple of 8"),
    (dict(head_dim=264), "up to 256"), (dict(dtype=0), "dtype"), (dict(scale=float("nan")), "scale"), (dict(scale=0.0), "scale"),
    (dict(q_head=12), "multiples of 8"), (dict(out_token=-8), "multiples of 8"), (dict(k_token=1 << 27), "token strides"),
    (dict(tokens=1 << 30, heads=64, kv_heads=1), "more than one launch"),
])
def test_prompt_attention_abi(change, match):
    _err(_lib.load().kf_prompt_attention(ctypes.byref(_struct(_lib.PromptAttentionArgs, **change)), None, 0, None), match)


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "non-null"), (dict(block_table=None), "non-null"), (dict(cache_v=0x1002), "16-byte"),
    (dict(block_size=48), "power of two"), (dict(block_size=8), "power of two"), (dict(table_width=0), "table_width"),
    (dict(num_pages=0), "num_pages"), (dict(max_new=-1), "max_new"), (dict(table_width=1 << 28), "too long"),
    (dict(k_page=4), "multiples of 8"), (dict(v_token=1 << 27), "token strides"),
])
def test_paged_attention_abi(change, match):
    args = _struct(_lib.PagedAttentionArgs, **change)
    _err(_lib.load().kf_paged_attention(ctypes.byref(args), 0x1000, 1 << 40, None), match)


@pytest.mark.parametrize("change,match", [
    (dict(qkv=None), "non-null"), (dict(qk=0x1004), "16-byte"), (dict(tokens=-1), "negative"), (dict(heads=0), "divide"),
    (dict(max_pos=0), "max_pos"), (dict(num_pages=0), "num_pages"), (dict(block_size=20), "power of two"),
    (dict(qkv_stride=3), "multiples of 8"), (dict(tokens=1 << 28), "more than one launch"), (dict(dtype=7), "dtype"),
])
def test_rope_paged_cache_abi(change, match):
    _err(_lib.load().kf_rope_paged_cache(ctypes.byref(_struct(_lib.RopePagedArgs, **change)), None), match)


@pytest.mark.parametrize("change,match", [
    (dict(slots=None), "non-null"), (dict(seqs=0), "seqs"), (dict(max_tokens=-1), "max_tokens"), (dict(block_size=0), "power of two"),
    (dict(free_left=0x5000, free_count=0x5000), "must not be free_count"), (dict(seqs=(1 << 16) + 1), "up to"),
    (dict(table_stride=2), "overlap"),
])
def test_paged_tables_abi(change, match):
    _err(_lib.load().kf_paged_tables(ctypes.byref(_struct(_lib.PagedTablesArgs, **change)), None), match)


def test_null_arguments_and_empty_batches():
    lib = _lib.load()
    for fn in (lib.kf_rope_paged_cache, lib.kf_paged_tables):
        _err(fn(None, None), "args must be non-null")
    _err(lib.kf_prompt_attention(None, None, 0, None), "args must be non-null")
    assert lib.kf_prompt_attention_workspace_bytes(None) == 0
    _err(lib.kf_paged_attention(None, None, 0, None), "args must be non-null")
    assert lib.kf_paged_attention_workspace_bytes(None) == 0
    assert lib.kf_prompt_attention(ctypes.byref(_struct(_lib.PromptAttentionArgs, tokens=0, q=None)), None, 0, None) == 0
    assert lib.kf_rope_paged_cache(ctypes.byref(_struct(_lib.RopePagedArgs, tokens=0, qkv=None)), None) == 0


@pytest.mark.parametrize("cls,pack", [
    (_lib.PagedTablesArgs, _lib.pack_paged_tables), (_lib.RopePagedArgs, _lib.pack_rope_paged),
    (_lib.PromptAttentionArgs, _lib.pack_prompt_attention), (_lib.PagedAttentionArgs, _lib.pack_paged_attention),
])
def test_packed_arguments_are_the_structure(cls, pack):
    values = [0.375 if kind is ctypes.c_float else (1 << 40) + i if kind is not ctypes.c_int else i - 3
              for i, (_, kind) in enumerate(cls._fields_)]
    assert pack(*values) == bytes(cls(*values))
    values[-1] = 1 << 32  # cut off in a structure
    with pytest.raises(ValueError, match="more than one call takes"):
        pack(*values)
