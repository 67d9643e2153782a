"""One `StackAttention` in several `MoeStack`s: each stack's ops work on the stack's own rows.  On the CPU by a backend that writes the calls
down, buffers named by their addresses; on the GPU against stacks that have an attention of their own."""
import dataclasses
import gc
from types import SimpleNamespace

import pytest
import torch

from moe4all_b200 import Buffer
from moe4all_b200.stack import AttnWeights, MoeStack, StackAttention

NE, E, K, NFF, H, KV, HD, PAGE, LAYERS = 64, 8, 2, 32, 4, 2, 16, 16, 2


class Notes:
    """A backend that notes what it is asked for."""

    def __init__(self):
        self.calls = []

    def wrap(self, ptr, nbytes):
        return Buffer(self, ptr, nbytes)

    def wrap_tensor(self, t):
        b = self.wrap(t.data_ptr(), t.numel() * t.element_size())
        b._owner = t
        return b

    def __getattr__(self, name):
        if name.startswith("_"):
            raise AttributeError(name)
        return lambda *args: self.calls.append((name, args))


def attention(be):
    z = torch.zeros
    layers = [AttnWeights(norm=z(NE), wqkv=be.wrap_tensor(z((H + 2 * KV) * HD, NE)), wo=be.wrap_tensor(z(NE, H * HD)), q_norm=z(HD), k_norm=z(HD)) for _ in range(LAYERS)]
    i32 = lambda *s: z(*s, dtype=torch.int32)
    return StackAttention(layers, H, KV, HD, i32(3), i32(2), i32(2, 8), PAGE, [(z(20, KV, PAGE, HD).half(), z(20, KV, PAGE, HD).half()) for _ in range(LAYERS)], window=40)


def stack(be, rows, attn, **kw):
    t = [be.wrap_tensor(torch.zeros(4)) for _ in range(4)]
    layers = [SimpleNamespace(b=dict(zip(("router", "gate", "up", "down"), t))) for _ in range(LAYERS)]
    return MoeStack(be, layers, [torch.ones(NE) for _ in range(LAYERS)], rows, NE, E, K, NFF, attn=attn, **kw)


def holds_together(be, st, li, rows):
    """The sub-layer's six calls: each reads what the one before wrote, from and to the stack's own hidden."""
    be.calls.clear()
    st.layer(li)
    (n0, norm), (n1, qkv), (n2, (rope,)), (n3, (att,)), (n4, proj), (n5, add) = be.calls[:6]
    assert [n0, n1, n2, n3, n4, n5] == ["rms_norm", "linear", "rope_kv", "attention", "linear", "add"]
    hidden = st.hidden.data_ptr()
    at = lambda b: b.handle
    assert at(norm[0]) == hidden and norm[3] == rows and at(norm[2]) == at(qkv[2]) and qkv[4] == rows
    wide = at(qkv[3])
    assert rope.rows == att.rows == rows and [at(x) for x in (rope.q, rope.k, rope.v)] == [wide, wide + 4 * H * HD, wide + 4 * (H + KV) * HD]
    assert at(rope.q_out) == at(att.q) and at(att.out) == at(proj[2]) and proj[4] == rows
    assert at(add[0]) == at(add[2]) == hidden and at(add[1]) == at(proj[3]) and add[3] == rows * NE
    assert [at(rope.k_cache), at(rope.v_cache)] == [at(att.k), at(att.v)] == [c.data_ptr() for c in st.attn.caches[li]]
    assert at(rope.kv_len) == at(att.kv_len) == st.attn.kv_len.data_ptr()
    return {wide, at(rope.q_out), at(att.out), at(proj[3]), at(norm[2])}


def test_each_stack_has_rows_of_its_own():
    be = Notes()
    attn = attention(be)
    stacks = [(stack(be, 60, attn), 60), (stack(be, 1, attn), 1), (stack(be, 7, attn, fused=False), 7)]
    gc.collect()
    used = [set().union(*(holds_together(be, st, li, rows) for li in range(LAYERS))) for st, rows in stacks]
    assert [len(u) for u in used] == [5, 5, 5] and len(set().union(*used)) == 15
    assert [u for u in used] == [set().union(*(holds_together(be, st, li, rows) for li in range(LAYERS))) for st, rows in stacks]


def test_layer_of_the_attention_itself():
    be = Notes()
    attn = attention(be)
    with pytest.raises(RuntimeError, match="0 stacks"):
        attn.layer(0)
    first = stack(be, 5, attn)
    attn.layer(1)
    assert [n for n, _ in be.calls] == ["rms_norm", "linear", "rope_kv", "attention", "linear", "add"] and be.calls[0][1][0].handle == first.hidden.data_ptr()
    second = stack(be, 3, attn)
    with pytest.raises(RuntimeError, match="2 stacks"):
        attn.layer(0)
    be.calls.clear()
    second.attn_layer(0)
    assert be.calls[0][1][0].handle == second.hidden.data_ptr()
    del first
    be.calls.clear()
    gc.collect()
    attn.layer(0)
    assert be.calls[0][1][0].handle == second.hidden.data_ptr()
    # a copy for another batch is bound to nothing yet
    with pytest.raises(RuntimeError, match="0 stacks"):
        dataclasses.replace(attn, max_q=1).layer(0)


def test_arrays_and_caches_that_are_something_else_are_refused():
    be = Notes()
    ok = attention(be)
    stack(be, 4, ok)
    z, f16 = torch.zeros, torch.float16
    pair = lambda *s, dtype=f16: (z(*s, dtype=dtype), z(*s, dtype=dtype))
    for match, kw in (("kv_len must be int32", dict(kv_len=ok.kv_len.long())), ("cu_q must be int32", dict(cu_q=ok.cu_q.float())), ("page_table must be int32", dict(page_table=ok.page_table.long())),
                      (r"cu_q is \[n_seq", dict(cu_q=ok.cu_q[:2])), (r"page_table \[n_seq", dict(page_table=ok.page_table.view(-1))), (r"page_table \[n_seq", dict(page_table=ok.page_table[:1])),
                      ("a .k, v. pair", dict(caches=ok.caches[:1])), ("float16", dict(caches=[ok.caches[0], pair(20, PAGE, KV, HD)])), ("float16", dict(caches=[pair(20, KV, PAGE, HD, dtype=torch.float32)] * 2)),
                      ("float16", dict(caches=[ok.caches[0], pair(19, KV, PAGE, HD)])), ("attention for 1", dict(layers=ok.layers[:1], caches=ok.caches[:1]))):
        with pytest.raises(ValueError, match=match):
            stack(be, 4, dataclasses.replace(ok, **kw))


@pytest.mark.gpu
def test_chunks_and_steps_over_one_attention(backend):
    """A prompt by one stack, then tokens by another (fused or not, recorded or not) over the same `StackAttention`, in turns: bit for bit what
    stacks with an attention each give over caches that start alike."""
    import test_gpu_stack_attention as g

    be = backend

    def arrays(attn, cu, kv):
        attn.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
        attn.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))

    x = torch.randn(42, g.NE, generator=torch.Generator(device="cuda").manual_seed(21), device="cuda")
    turns = [(40, [0, 30, 40], [30, 17]), (2, [0, 1, 2], [31, 18]), (40, [0, 5, 38], [36, 51]), (2, [0, 1, 2], [37, 52]), (2, [0, 1, 2], [38, 53])]
    results = []
    for shared in (False, True):
        chunks, a, _ = g.build(be, [0, 7], [30, 10])
        steps, b, _ = g.build(be, [0, 7], [1, 1])
        if shared:
            b = a
            layers, nws = steps.layers, steps._nw
            steps = MoeStack(be, layers, nws, 2, g.NE, g.E, g.K, g.NFF, attn=a)
            plain = MoeStack(be, layers, nws, 2, g.NE, g.E, g.K, g.NFF, attn=a, fused=False)  # bound, and once used
            before = [tuple(c.clone() for c in l) for l in a.caches]
            arrays(a, [0, 1, 2], [31, 18])
            torch.cuda.synchronize()
            plain.step()
            steps.record()
            be.sync()
            for l, old in zip(a.caches, before):
                for c, o in zip(l, old):
                    c.copy_(o)
        outs = []
        for i, (rows, cu, kv) in enumerate(turns):
            st, at, other = (chunks, a, b) if rows == 40 else (steps, b, a)
            arrays(at, cu, kv)
            st.hidden.copy_(x[:rows] + i)
            torch.cuda.synchronize()
            st.replay() if shared and rows == 2 else st.step()
            be.sync()
            n = cu[-1]
            outs.append(st.hidden[:n].clone())
            if other is not at:
                for l, m in zip(at.caches, other.caches):
                    for c, o in zip(l, m):
                        o.copy_(c)
            torch.cuda.synchronize()
        results.append((outs, [c.clone() for l in a.caches for c in l]))
    for p, q in zip(results[0][0], results[1][0]):
        assert torch.equal(p, q) and bool(p.isfinite().all())
    for p, q in zip(results[0][1], results[1][1]):
        assert torch.equal(p, q)
