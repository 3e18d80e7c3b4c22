"""Arguments of the paged-cache operators that are refused before a launch (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernelforge import _lib, ops

from test_paged_cpu import _struct, attention_args, prompt_args


@pytest.mark.parametrize("op,args", [(ops.paged_attention, attention_args), (ops.prompt_attention, prompt_args)])
def test_an_output_that_requires_a_gradient(op, args):
    """It would be written without its graph knowing."""
    a = args()
    out = torch.zeros_like(a["q"], requires_grad=True)
    with pytest.raises(RuntimeError, match="inference only"):
        op(**a, out=out)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA device"):
        op(**a, out=out)


@pytest.mark.parametrize("scale", [2.4e38, 2.9e38])
def test_scales_whose_exponents_are_not_finite(scale):
    """Scores are taken in units of the exponent to base 2, scale x 1.4427: past 2^128 even a score of zero is NaN."""
    for op, args in ((ops.paged_attention, attention_args), (ops.prompt_attention, prompt_args)):
        with pytest.raises(ValueError, match="at most 2.35e38"):
            op(**args(), scale=scale)
        with pytest.raises(RuntimeError, match="CUDA device"):
            op(**args(), scale=2.3e38)
    lib = _lib.load()
    for fn, cls, rest in ((lib.kf_prompt_attention, _lib.PromptAttentionArgs, (None, 0, None)),
                          (lib.kf_paged_attention, _lib.PagedAttentionArgs, (0x1000, 1 << 40, None))):
        assert fn(ctypes.byref(_struct(cls, scale=scale)), *rest) != 0 and "at most 2.35e38" in _lib.last_error()
