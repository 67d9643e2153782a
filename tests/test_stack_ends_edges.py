"""Ends of a `MoeStack` that could not be served are refused before a step runs."""
import dataclasses

import pytest
import torch

from test_stack_attention_bind import NE, Notes, stack
from test_stack_ends import ends

from moe4all_b200 import DType


@pytest.mark.parametrize("dtype", [DType.F16, DType.BF16])
def test_a_head_of_16_bits_is_refused_before_a_step(dtype):
    """`linear` has no weights of 16 bits: a step would end at its last op, its keys and values written."""
    be = Notes()
    with pytest.raises(ValueError, match="head_dtype"):
        stack(be, 2, None, ends=dataclasses.replace(ends(be, 2), head_dtype=dtype))
    # (a table of them is fine)
    stack(be, 2, None, ends=dataclasses.replace(ends(be, 2), table_dtype=dtype))


def test_a_norm_that_is_something_else_is_refused():
    """The library sees its bytes only: one of f64 would be read as f32, one of 16 bits refused behind the layers."""
    be = Notes()
    for norm in (torch.ones(NE).double(), torch.ones(NE).half(), torch.ones(NE - 1), torch.ones(2 * NE)[::2]):
        with pytest.raises(ValueError, match="norm"):
            stack(be, 2, None, ends=dataclasses.replace(ends(be, 2), norm=norm))
