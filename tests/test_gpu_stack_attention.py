"""GPU: whole layers - attention over pages, then the MoE sub-layer - as `MoeStack` runs them, step after step.

Tolerance of an attention sub-layer, relative to the largest magnitude M of each of its stages: a Linear of n values in f32 is off by
n 2^-24 of sum |w| |x| at most, here sqrt(n) max|x| times the weights' 1 / sqrt(n) spread (3 standard deviations: 3 max|x|); the norm by 2^-21;
keys and values are rounded to f16, 2^-11 of them, the former also on scores of size S: weights off by 2^-11 S, results by twice that."""
import numpy as np
import pytest

from moe4all_b200 import DType
from moe4all_b200.devgen import DeviceLayer
from moe4all_b200.stack import AttnWeights, MoeStack, StackAttention

pytestmark = pytest.mark.gpu
NE, E, K, NFF, H, KV, HD, PAGE, LAYERS = 512, 16, 4, 256, 8, 2, 64, 16, 2


def build(be, lens, new, width=8):
    """A stack of LAYERS layers for sequences with lens tokens in their caches and new ones to come."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    rows, n = sum(new), len(new)
    layers = [DeviceLayer(be, 700 + i, NE, E, NFF, router_std=0.05) for i in range(LAYERS)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    weights, host = [], []
    for _ in range(LAYERS):
        t = dict(norm=1.0 + 0.1 * r(NE), wqkv=r((H + 2 * KV) * HD, NE) * NE ** -0.5, wo=r(NE, H * HD) * (H * HD) ** -0.5, q_norm=1.0 + 0.1 * r(HD), k_norm=1.0 + 0.1 * r(HD))
        host.append(t)
        weights.append(AttnWeights(norm=t["norm"], wqkv=be.wrap_tensor(t["wqkv"]), wo=be.wrap_tensor(t["wo"]), q_norm=t["q_norm"], k_norm=t["k_norm"], dtype=DType.F32))
    n_pages = n * width + 1
    table = torch.randperm(n_pages, generator=g, device="cuda")[: n * width].int().view(n, width).contiguous()
    caches = [tuple(r(n_pages, KV, PAGE, HD).half() for _ in range(2)) for _ in range(LAYERS)]
    attn = StackAttention(weights, H, KV, HD, i32([sum(new[:i]) for i in range(n + 1)]), i32([a + b for a, b in zip(lens, new)]), table, PAGE, caches, max_q=max(new), rope_base=1e6)
    nws = [1.0 + 0.1 * r(NE) for _ in range(LAYERS)]
    st = MoeStack(be, layers, nws, rows, NE, E, K, NFF, attn=attn)
    torch.cuda.synchronize()
    return st, attn, host


def plain_attention(attn, host, li, hidden, kc, vc):
    """The sub-layer in 64 bits: hidden after it, the new k and v, and its largest stage."""
    import torch

    h, t = hidden.double(), {k: v.double() for k, v in host[li].items()}
    x = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * t["norm"]
    rows = x.shape[0]
    q, k, v = (x @ t["wqkv"].T).view(rows, H + 2 * KV, HD).split([H, KV, KV], 1)
    norm = lambda y, w: y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
    cu, kv = attn.cu_q.tolist(), attn.kv_len.tolist()
    pos = torch.cat([torch.arange(kv[s] - cu[s + 1] + cu[s], kv[s], device="cuda") for s in range(len(kv))]).double()
    ang = pos[:, None, None] * 1e6 ** (-torch.arange(0, HD, 2, device="cuda").double() / HD)

    def turn(y):
        a, b = y[..., : HD // 2], y[..., HD // 2 :]
        return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)

    q, k = turn(norm(q, t["q_norm"])), turn(norm(k, t["k_norm"]))
    out = torch.zeros(rows, H, HD, dtype=torch.float64, device="cuda")
    for s in range(len(kv)):
        n = cu[s + 1] - cu[s]
        i = torch.arange(kv[s] - n, device="cuda")
        pages = attn.page_table[s].long()[i // PAGE]
        keys, vals = (torch.cat([c[pages, :, i % PAGE].double(), y[cu[s] : cu[s + 1]]]) for c, y in ((kc, k), (vc, v)))
        for j in range(n):
            m = kv[s] - n + j + 1
            for head in range(H):
                w = torch.softmax(keys[:m, head // (H // KV)] @ q[cu[s] + j, head] * HD ** -0.5, 0)
                out[cu[s] + j, head] = w @ vals[:m, head // (H // KV)]
    S = float((q.norm(dim=-1).max() * max(float(k.norm(dim=-1).max()), float(kc.double().norm(dim=-1).max())))) * HD ** -0.5
    M = max(float(v.abs().max()), float(vc.double().abs().max()))
    tol = 3 * M * (2 * 2.0 ** -11 * S + 2.0 ** -11 + NE * 2.0 ** -22)
    return h + out.view(rows, -1) @ t["wo"].T, tol


@pytest.mark.parametrize("lens,new", [([0, 40, 7, 100], [1, 1, 1, 1]), ([0, 3, 50], [40, 1, 7])])
def test_layer_is_attention_then_moe(backend, lens, new):
    import torch

    be = backend
    st, attn, host = build(be, lens, new)
    h0 = torch.randn(sum(new), NE, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    for li in range(LAYERS):
        before = [c.clone() for c in attn.caches[li]]
        want, tol = plain_attention(attn, host, li, h0, *before)
        st.hidden.copy_(h0)
        torch.cuda.synchronize()
        attn.layer(li)
        be.sync()
        after = st.hidden.clone()
        assert float((after - want).abs().max()) <= tol
        assert not torch.equal(before[0], attn.caches[li][0]) and not torch.equal(before[1], attn.caches[li][1])
        torch.cuda.synchronize()
        be.moe_ffn(st.ops[li])
        be.sync()
        both = st.hidden.clone()
        st.hidden.copy_(h0)
        torch.cuda.synchronize()
        st.layer(li)
        be.sync()
        assert torch.equal(st.hidden, both)


def test_recorded_steps_follow_the_sequences(backend):
    """Tokens generated by one recorded step, its lengths written between replays, against the same steps called op by op."""
    import torch

    be = backend
    results = []
    for recorded in (False, True):
        st, attn, _ = build(be, [0, 15, 31, 60], [1, 1, 1, 1])
        start = attn.kv_len.clone()
        if recorded:
            st.hidden.zero_()
            caches = [tuple(x.clone() for x in c) for c in attn.caches]
            torch.cuda.synchronize()
            st.record()
            be.sync()
            for c, old in zip(attn.caches, caches):
                for x, y in zip(c, old):
                    x.copy_(y)
        x = torch.randn(4, NE, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda")
        outs = []
        for step in range(20):
            attn.kv_len.copy_(start + step)
            st.hidden.copy_(x)
            torch.cuda.synchronize()
            st.replay() if recorded else st.step()
            be.sync()
            x = st.hidden / st.hidden.norm(dim=-1, keepdim=True) * NE ** 0.5
            outs.append(st.hidden.clone())
        results.append(torch.stack(outs))
        assert bool(results[-1].isfinite().all())
    assert torch.equal(results[0], results[1])


def test_prompt_at_once_or_in_chunks(backend):
    """A prompt through the attention sub-layer in one call, or in pieces over the growing cache: the same keys, the same rows."""
    import torch

    be = backend
    x = torch.randn(60, NE, generator=torch.Generator(device="cuda").manual_seed(13), device="cuda")
    whole, attn, host = build(be, [0], [60])
    whole.hidden.copy_(x)
    torch.cuda.synchronize()
    attn.layer(0)
    be.sync()
    want, tol = whole.hidden.clone(), None
    _, tol = plain_attention(attn, host, 0, x, *[torch.zeros_like(c) for c in attn.caches[0]])
    done = 0
    got = torch.zeros_like(x)
    pieces, first = [25, 1, 1, 33], None
    for n in pieces:
        st, a, _ = build(be, [done], [n])
        if first is not None:
            for c, old in zip(a.caches[0], first):
                c.copy_(old)
        st.hidden.copy_(x[done : done + n])
        torch.cuda.synchronize()
        a.layer(0)
        be.sync()
        got[done : done + n] = st.hidden
        first = [c.clone() for c in a.caches[0]]
        done += n
    # (two ways to the same numbers, each within the bound)
    assert float((got - want).abs().max()) <= 2 * tol
