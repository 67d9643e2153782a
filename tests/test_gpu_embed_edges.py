"""GPU: rows of a table that another op has just written, on the same stream and in recorded plans."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("writer", ["embed", "rms_norm"])
def test_rows_of_a_table_that_was_just_written(backend, writer, recorded):
    """A table that changes between two lookups, by kernels beside whose ends the lookups may start: every lookup has the rows that are there when it is due.  All CTAs read the
    same few rows, so that every SM has had the old ones."""
    import torch

    from moe4all_b200 import Embed

    be, w = backend, backend.wrap_tensor
    R, ne, V = 1184, 256, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    sources = [torch.randn(V, ne, generator=g, device="cuda") for _ in range(6)]
    table = torch.zeros(V, ne, device="cuda")
    outs = [torch.zeros(R, ne, device="cuda") for _ in sources]
    rows = torch.arange(V, dtype=torch.int32, device="cuda")
    ids = (torch.arange(R, device="cuda") % V).int()
    ones = torch.ones(ne, device="cuda")
    torch.cuda.synchronize()
    b_table, b_ones = w(table), w(ones)
    fill = [Embed(table=w(s), ids=w(rows), dst=b_table, rows=V, ne=ne, n_vocab=V) for s in sources]
    look = [Embed(table=b_table, ids=w(ids), dst=w(o), rows=R, ne=ne, n_vocab=V) for o in outs]
    b_sources = [w(s) for s in sources]

    def step():
        for i in range(len(sources)):
            if writer == "embed":
                be.embed(fill[i])
            else:
                be.rms_norm(b_sources[i], b_ones, b_table, V, ne, 1e-6)
            be.embed(look[i])

    step()
    be.sync()
    if recorded:
        be.graph_begin()
        step()
        plan = be.graph_end()
    for _ in range(10):
        for o in outs:
            o.fill_(7.5)
        torch.cuda.synchronize()
        be.execute(plan) if recorded else step()
        be.sync()
        for s, o in zip(sources, outs):
            want = s
            if writer == "rms_norm":
                # (f32 by a rounded factor: 2^-20 of the value)
                want = (s.double() / torch.sqrt((s.double() ** 2).mean(-1, keepdim=True) + 1e-6)).float()
            off = (o - want[ids.long()]).abs()
            assert bool((off <= (0.0 if writer == "embed" else 2.0 ** -20) * want[ids.long()].abs()).all())
