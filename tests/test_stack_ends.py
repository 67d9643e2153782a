"""A `MoeStack` from tokens to tokens over pages of 8 bits.  On the CPU by a backend that writes the calls down; on the GPU each stage against its formula in 64
bits, and recorded steps, each of which goes on from the answer before, against the same steps called op by op.

Tolerances: an attention sub-layer's are those of test_gpu_stack_attention.py, over the values that the pages hold after it.  Logits, a Linear of NE values in f32
behind a norm: rows off by 2^-21, the product by NE 2^-24 of sum |w| |x| at most."""
import dataclasses

import pytest
import torch

from test_stack_attention_bind import E, H, HD, K, KV, LAYERS, NE, NFF, PAGE, Notes, attention, stack

from moe4all_b200 import DType
from moe4all_b200.stack import StackEnds

V = 1001


def bits8(n_pages=20, device="cpu"):
    z = lambda last: torch.zeros(n_pages, KV, PAGE, last, dtype=torch.uint8, device=device)
    return [(z(HD), z(HD), z(HD // 16), z(HD // 16)) for _ in range(LAYERS)]


def ends(be, rows, **kw):
    w = lambda: be.wrap_tensor(torch.zeros(4))
    kw = {**dict(norm=torch.ones(NE), head=w(), u=torch.zeros(rows), temperature=torch.ones(rows), top_k=torch.zeros(rows, dtype=torch.int32)), **kw}
    return StackEnds(table=w(), tokens=torch.zeros(rows, dtype=torch.int32), n_vocab=V, scale=2.0, **kw)


def test_calls_of_a_step_hold_together():
    be = Notes()
    attn = dataclasses.replace(attention(be), caches=bits8())
    e = ends(be, 2)
    st = stack(be, 2, attn, ends=e)
    st.step()
    names = [n for n, _ in be.calls]
    assert names == ["embed"] + ["rms_norm", "linear", "rope_kv", "attention", "linear", "add", "moe_ffn"] * LAYERS + ["rms_norm", "linear", "sample"]
    at = lambda b: b.handle
    embed, sample = be.calls[0][1][0], be.calls[-1][1][0]
    assert at(embed.ids) == at(sample.ids) == e.tokens.data_ptr() and at(embed.dst) == st.hidden.data_ptr()
    assert (embed.rows, embed.ne, embed.n_vocab, embed.scale) == (2, NE, V, 2.0) and (sample.rows, sample.n_vocab) == (2, V)
    norm, head = be.calls[-3][1], be.calls[-2][1]
    assert at(norm[0]) == st.hidden.data_ptr() and at(norm[2]) == at(head[2]) and at(head[1]) == at(e.head) and at(head[3]) == at(sample.logits) and head[4:] == (2, NE, V)
    assert at(sample.u) == e.u.data_ptr() and at(sample.temperature) == e.temperature.data_ptr() and at(sample.top_k) == e.top_k.data_ptr() and sample.top_p is None and sample.min_p is None
    for li in range(LAYERS):
        rope, att = be.calls[3 + 7 * li][1][0], be.calls[4 + 7 * li][1][0]
        assert [at(x) for x in (rope.k_cache, rope.v_cache, rope.k_scale, rope.v_scale)] == [at(x) for x in (att.k, att.v, att.k_scale, att.v_scale)] == [c.data_ptr() for c in attn.caches[li]]


def test_a_stack_without_a_head_ends_with_its_layers():
    be = Notes()
    st = stack(be, 2, attention(be), ends=ends(be, 2, head=None, norm=None, u=None, temperature=None, top_k=None))
    st.step()
    assert [n for n, _ in be.calls] == ["embed"] + ["rms_norm", "linear", "rope_kv", "attention", "linear", "add", "moe_ffn"] * LAYERS


def test_ends_that_are_something_else_are_refused():
    be = Notes()
    for match, kw in (("tokens", dict(tokens=torch.zeros(3, dtype=torch.int32))), ("tokens", dict(tokens=torch.zeros(2, dtype=torch.int64))), ("u is", dict(u=torch.zeros(2).double())),
                      ("u is", dict(u=torch.zeros(4)[::2])), ("top_k", dict(top_k=torch.zeros(2))), ("temperature", dict(temperature=torch.ones(1))), ("norm", dict(norm=None)),
                      ("random", dict(u=None)), ("without a head", dict(head=None))):
        with pytest.raises(ValueError, match=match):
            stack(be, 2, None, ends=dataclasses.replace(ends(be, 2), **kw))


def test_caches_of_8_bits_that_are_something_else_are_refused():
    be = Notes()
    ok = dataclasses.replace(attention(be), caches=bits8())
    stack(be, 4, ok)
    f16 = attention(be).caches
    stack(be, 4, dataclasses.replace(ok, caches=[f16[0], ok.caches[1]]))  # a layer each as it likes
    a, b = ok.caches
    for match, bad in (("not 3 tensors", a[:3]), ("8 bits", (*a[:2], *f16[0])), ("8 bits", (a[2], a[3], a[0], a[1])), ("8 bits", (*a[:3], a[3][:19])), ("float16", a[:2])):
        with pytest.raises(ValueError, match=match):
            stack(be, 4, dataclasses.replace(ok, caches=[b, bad]))


# ---- on the GPU

def build(be, prompts):
    """Stacks of one model over the same pages: one for the prompts but for their last tokens, one for a token of each."""
    import test_gpu_stack_attention as g
    from moe4all_b200.stack import MoeStack

    n = len(prompts)
    first, attn, host = g.build(be, [0] * n, [p - 1 for p in prompts])
    z = lambda last: torch.full((attn.caches[0][0].shape[0], g.KV, g.PAGE, last), 0xEE, dtype=torch.uint8, device="cuda")
    attn = dataclasses.replace(attn, caches=[(z(g.HD), z(g.HD), z(g.HD // 16), z(g.HD // 16)) for _ in range(g.LAYERS)])
    r = torch.Generator(device="cuda").manual_seed(31)
    table = torch.randn(V, g.NE, generator=r, device="cuda") / 8
    head = torch.randn(V, g.NE, generator=r, device="cuda") * (3 * g.NE ** -0.5)
    norm = 1 + 0.1 * torch.randn(g.NE, generator=r, device="cuda")
    f = lambda *v: torch.tensor(v, device="cuda")
    tokens = torch.randint(0, V, (sum(prompts),), generator=r, device="cuda", dtype=torch.int32)
    lead = torch.cat([t[:-1] for t in tokens.split(prompts)]).contiguous()
    last = torch.stack([t[-1] for t in tokens.split(prompts)]).contiguous()
    both = dict(table=be.wrap_tensor(table), n_vocab=V, scale=8.0)
    rows = sum(prompts) - n
    chunk = MoeStack(be, first.layers, first._nw, rows, g.NE, g.E, g.K, g.NFF, attn=attn, ends=StackEnds(tokens=lead, **both))
    steps = MoeStack(be, first.layers, first._nw, n, g.NE, g.E, g.K, g.NFF, attn=dataclasses.replace(attn, max_q=1),
                     ends=StackEnds(tokens=last, norm=norm, head=be.wrap_tensor(head), u=torch.zeros(n, device="cuda"), temperature=f(0.0, 1.0, 0.7, 1.3), top_k=f(0, 0, 40, 5).int(),
                                    top_p=f(1.0, 0.9, 1.0, 0.8), **both))
    torch.cuda.synchronize()
    return chunk, steps, host, dict(table=table, head=head, norm=norm, lead=lead, last=last)


def write(attn, cu, kv):
    attn.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
    attn.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))
    torch.cuda.synchronize()


def plain_attention(attn, host, li, hidden):
    """The sub-layer in 64 bits over the values that are in the pages, and its tolerance."""
    import test_gpu_stack_attention as g
    from test_gpu_kv_q8 import values

    keep = attn.caches
    kc, vc, ks, vs = keep[li]
    kc, vc = values(kc, ks), values(vc, vs)
    t = {k: v.double() for k, v in host[li].items()}
    h = hidden.double()
    x = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * t["norm"]
    rows = x.shape[0]
    q = (x @ t["wqkv"].T).view(rows, g.H + 2 * g.KV, g.HD)[:, : g.H]
    q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6) * t["q_norm"]
    cu, kv = attn.cu_q.tolist(), attn.kv_len.tolist()
    pos = torch.cat([torch.arange(kv[s] - cu[s + 1] + cu[s], kv[s], device="cuda") for s in range(len(kv))]).double()
    ang = pos[:, None, None] * 1e6 ** (-torch.arange(0, g.HD, 2, device="cuda").double() / g.HD)
    a, b = q[..., : g.HD // 2], q[..., g.HD // 2 :]
    q = torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    out = torch.zeros(rows, g.H, g.HD, dtype=torch.float64, device="cuda")
    S = M = 0.0
    for s in range(len(kv)):
        i = torch.arange(kv[s], device="cuda")
        pages = attn.page_table[s].long()[i // g.PAGE]
        keys, vals = (c[pages, :, i % g.PAGE].repeat_interleave(g.H // g.KV, 1) for c in (kc, vc))
        new = cu[s + 1] - cu[s]
        score = torch.einsum("rhd,khd->rhk", q[cu[s] : cu[s + 1]], keys) * g.HD ** -0.5
        ahead = i[None, :] > (kv[s] - new + torch.arange(new, device="cuda"))[:, None]
        out[cu[s] : cu[s + 1]] = torch.einsum("rhk,khd->rhd", torch.softmax(score.masked_fill(ahead[:, None], -float("inf")), -1), vals)
        S, M = max(S, float(q.norm(dim=-1).max() * keys.norm(dim=-1).max()) * g.HD ** -0.5), max(M, float(vals.abs().max()))
    assert bool(out.isfinite().all())
    return h + out.view(rows, -1) @ t["wo"].T, 3 * M * (2 * 2.0 ** -11 * S + 2.0 ** -11 + g.NE * 2.0 ** -22)


PROMPTS = [50, 2, 17, 33]


@pytest.mark.gpu
def test_each_stage_of_a_step(backend):
    import test_gpu_stack_attention as g
    from test_gpu_token_ends import reference

    be = backend
    chunk, steps, host, t = build(be, PROMPTS)
    n = len(PROMPTS)
    r = torch.Generator(device="cuda").manual_seed(41)
    cu = [0]
    for p in PROMPTS:
        cu.append(cu[-1] + p - 1)
    for step in range(4):
        st = chunk if step == 0 else steps
        write(chunk.attn, cu if step == 0 else list(range(n + 1)), [p - 1 + step for p in PROMPTS])
        tokens = (t["lead"] if step == 0 else t["last"]).clone()
        steps.ends._ends.u.copy_(torch.rand(n, generator=r, device="cuda"))
        torch.cuda.synchronize()
        st.ends.embed()
        be.sync()
        assert torch.equal(st.hidden, 8 * t["table"][tokens.long()])
        for li in range(g.LAYERS):
            h = st.hidden.clone()
            torch.cuda.synchronize()
            st.attn_layer(li)
            be.sync()
            want, tol = plain_attention(st.attn, host, li, h)
            assert float((st.hidden - want).abs().max()) <= tol
            be.moe_ffn(st.ops[li])
            be.sync()
        st.ends.answer()
        be.sync()
        if step == 0:
            assert torch.equal(tokens, t["lead"])
            continue
        h, w = st.hidden.double(), t["head"].double()
        x = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * t["norm"].double()
        assert bool(((st.ends.logits - x @ w.T).abs() <= (2.0 ** -21 + g.NE * 2.0 ** -24) * (x.abs() @ w.abs().T)).all())
        e, logits = st.ends._ends, st.ends.logits.cpu().numpy()
        for i in range(n):
            assert int(t["last"][i]) == reference(logits[i], float(e.u[i]), float(e.temperature[i]), int(e.top_k[i]), float(e.top_p[i]))[0]


@pytest.mark.gpu
def test_recorded_steps_answer_themselves(backend):
    be = backend
    results = []
    for recorded in (False, True):
        chunk, steps, _, t = build(be, PROMPTS)
        n = len(PROMPTS)
        cu = [0]
        for p in PROMPTS:
            cu.append(cu[-1] + p - 1)
        write(chunk.attn, cu, [p - 1 for p in PROMPTS])
        chunk.step()
        be.sync()
        write(chunk.attn, list(range(n + 1)), PROMPTS)
        if recorded:
            last = t["last"].clone()
            torch.cuda.synchronize()
            steps.record()  # (its one run writes the places that the first replay writes)
            be.sync()
            t["last"].copy_(last)
        r = torch.Generator(device="cuda").manual_seed(51)
        ids = []
        for step in range(24):
            write(chunk.attn, list(range(n + 1)), [p + step for p in PROMPTS])
            steps.ends._ends.u.copy_(torch.rand(n, generator=r, device="cuda"))
            torch.cuda.synchronize()
            steps.replay() if recorded else steps.step()
            be.sync()
            ids.append(t["last"].clone())
        ids = torch.stack(ids)
        assert bool((ids >= 0).all()) and bool((ids < V).all()) and all(len(set(ids[:, i].tolist())) > 3 for i in (1, 2, 3))
        results.append((ids, [c.clone() for l in chunk.attn.caches for c in l]))
    assert torch.equal(results[0][0], results[1][0])
    for a, b in zip(results[0][1], results[1][1]):
        assert torch.equal(a, b)
