"""Ends of a `MoeStack` that could not be served are refused before a step runs; a stack may be built behind work that is still under way."""
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


@pytest.mark.gpu
def test_a_stack_built_behind_work_under_way(backend):
    """What a step needs of its inputs is there; only the stack's own buffers are made while torch's stream is busy.  Nothing of them arrives in the middle of a step."""
    import test_gpu_stack_attention as g
    from test_stack_ends import PROMPTS, build, write

    from moe4all_b200.stack import MoeStack

    be = backend
    chunk, steps, _, t = build(be, PROMPTS)
    n = len(PROMPTS)
    cu = [0]
    for p in PROMPTS:
        cu.append(cu[-1] + p - 1)
    write(chunk.attn, cu, [p - 1 for p in PROMPTS])
    chunk.step()
    be.sync()
    write(chunk.attn, list(range(n + 1)), PROMPTS)
    first = t["last"].clone()
    steps.step()
    be.sync()
    want = t["last"].clone(), steps.hidden.clone(), steps.ends.logits.clone()
    t["last"].copy_(first)
    busy = torch.zeros(1 << 28, device="cuda")
    torch.cuda.synchronize()
    for _ in range(200):
        busy.add_(1.0)
    late = MoeStack(be, steps.layers, steps._nw, n, g.NE, g.E, g.K, g.NFF, attn=steps.attn, ends=steps.ends._ends)
    late.step()
    be.sync()
    torch.cuda.synchronize()
    for a, b in zip((t["last"], late.hidden, late.ends.logits), want):
        assert torch.equal(a, b)
