"""Arguments of the paged-cache operators that are refused before a launch (no GPU)."""

from __future__ import annotations

import pytest
import torch

from kernelforge import ops

from test_paged_cpu import attention_args, prompt_args


@pytest.mark.parametrize("op,args", [(ops.paged_attention, attention_args), (ops.prompt_attention, prompt_args)])
def test_an_output_that_requires_a_gradient(op, args):
    """It would be written without its graph knowing."""
    a = args()
    out = torch.zeros_like(a["q"], requires_grad=True)
    with pytest.raises(RuntimeError, match="inference only"):
        op(**a, out=out)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA device"):
        op(**a, out=out)
