"""A GGUF layer whose tensors have a type that only token tables may have is refused when it is loaded, nothing uploaded."""
from types import SimpleNamespace

import pytest

from moe4all_b200 import DType
from moe4all_b200.gguf import moe_layer_op

DIMS = {"ffn_gate_inp": (256, 8), "ffn_gate_exps": (256, 512, 8), "ffn_up_exps": (256, 512, 8), "ffn_down_exps": (512, 256, 8)}


class File:
    """One layer's tensors, their types by name."""

    def __init__(self, **types):
        self.types, self.uploaded = {"ffn_gate_inp": 0, "ffn_gate_exps": 12, "ffn_up_exps": 12, "ffn_down_exps": 14, **types}, []

    def find(self, name):
        t = name.split(".")[2]
        return SimpleNamespace(dims=DIMS[t], dtype=self.types[t]) if t in DIMS and name.endswith(".weight") else None

    def meta_u64(self, key):
        return 2

    def meta_f64(self, key):
        return None

    def upload(self, be, name):
        self.uploaded.append(name)
        return SimpleNamespace(handle=1)


def test_types_of_a_layer():
    f = File()
    op, _ = moe_layer_op(None, f, 0, "any")
    assert (op.router_dtype, op.gate_dtype, op.up_dtype, op.down_dtype) == (DType.F32, DType.Q4K, DType.Q4K, DType.Q6K) and len(f.uploaded) == 4


@pytest.mark.parametrize("tensor", DIMS)
@pytest.mark.parametrize("dtype", [1, 30, 29])
def test_16_bits_are_refused(tensor, dtype):
    f = File(**{tensor: dtype})
    with pytest.raises(ValueError):
        moe_layer_op(None, f, 0, "any")
    assert not f.uploaded
