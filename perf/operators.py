"""The attention half of a mixture-of-experts layer, as timed cases: what runs between two `moe_ffn` calls.

Three operators, each case is one call of one of them:

  rope    `CudaBackend.rope_kv`: per-head RMS norm and rotary embedding of a batch's new q and k rows, and their k and v
          rounded to f16 into a paged cache.
  paged   `CudaBackend.attention` over the pages: single tokens, speculative windows, chunks of a prompt behind a past.
  prompt  `CudaBackend.attention` over packed f16 rows: whole prompts of different lengths, causal.

Rows are f32 as everywhere in this framework, the cache is f16 [pages, kv heads, page size, head size].  Sizes are generic
ones for layers of the benchmark's hidden sizes (2048 to 7168): heads of 64, 128 and 256 (and sizes between), 1 to 16 query heads per kv head.
"""
import itertools
import math
import random

import torch

own = False

EPS = 1e-6


def case(op, name=None, **kw):
    c = dict(op=op, heads=32, kv_heads=4, hd=128, n_seq=1, rows=1, past_lo=0, past_hi=0, page=64, window=0, n_rot=0, interleaved=False, norm=False, base=1e6)
    c.update(kw)
    if op != "rope":
        for k in ("n_rot", "interleaved", "norm", "base"):
            del c[k]
    return dict(c, name=name) if name else c


def listed():
    return [
        # A decode step of 32 streams: one new row each, with the per-head norms of the models that have them.
        case("rope", "rope_step_32", n_seq=32, rows=32, past_lo=100, past_hi=2000, n_rot=128, norm=True),
        # A ragged batch of prompt chunks of a model that rotates a quarter of its wide heads, pairs side by side.
        case("rope", "rope_partial_777", heads=16, kv_heads=2, hd=256, n_seq=3, rows=777, past_lo=1, past_hi=900, n_rot=64, interleaved=True, page=16),
        # Four prompts of a prefill batch.
        case("rope", "rope_prompts_8192", n_seq=4, rows=8192, n_rot=128, norm=True),
        # One chat stream early in its conversation: the smallest call, latency alone.
        case("paged", "step_1x513", past_lo=512, past_hi=512, page=16),
        # A full decode batch with contexts of all lengths.
        case("paged", "step_64x8k", n_seq=64, rows=64, past_lo=700, past_hi=8000),
        # One stream over a long document.
        case("paged", "step_1x131072", past_lo=131071, past_hi=131071),
        # Decode on wide heads, 8 query heads to a kv head.
        case("paged", "step_16x16k_hd256", heads=16, kv_heads=2, hd=256, n_seq=16, rows=16, past_lo=1000, past_hi=16000, page=32),
        # A speculative window of five tokens per stream, on a layer with a sliding window.
        case("paged", "window_24x5", heads=64, kv_heads=8, hd=64, n_seq=24, rows=120, past_lo=50, past_hi=4000, window=1024, page=16),
        # Chunked prefill: 512 new tokens or so each behind long pasts.
        case("paged", "chunk_4x512", n_seq=4, rows=2048, past_lo=3000, past_hi=16000),
        # A short question.
        case("prompt", "prompt_61", rows=61),
        # A prefill batch of prompts of different lengths.
        case("prompt", "prompts_16_hd64", heads=64, kv_heads=8, hd=64, n_seq=16, rows=8192),
        # One long prompt.
        case("prompt", "prompt_8192", rows=8192),
    ]


def _lengths(c):
    """New tokens and tokens in the cache after them, by sequence: fixed by the case."""
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    n, rows = c["n_seq"], c["rows"]
    ends = list(itertools.accumulate(r.uniform(0.2, 1.8) for _ in range(n)))
    ends = [i + 1 + int(round((rows - n) * e / ends[-1])) for i, e in enumerate(ends)]  # at least one each; the rest by weight
    q = [b - a for a, b in zip([0] + ends[:-1], ends)]
    lo, hi = c["past_lo"], c["past_hi"]
    past = [int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))) if 0 < lo < hi else lo for _ in range(n)]
    return q, [a + b for a, b in zip(q, past)]


def _pairs(q, kv, window):
    """Visible (row, key) pairs of a sequence, and its visible keys."""
    first = kv - q
    if not window:
        return q * first + q * (q + 1) // 2, kv
    pairs = sum(min(window, p + 1) for p in range(first, kv))
    return pairs, kv - max(0, first - window + 1)


def work(c):
    H, K, hd, rows = c["heads"], c["kv_heads"], c["hd"], c["rows"]
    if c["op"] == "rope":
        return {"bytes": rows * hd * (4 * (H + 2 * K) + 4 * H + 4 * K), "flops": rows * (H + K) * (4 * hd * c["norm"] + 3 * c["n_rot"])}
    pairs = [_pairs(q, kv, c["window"]) for q, kv in zip(*_lengths(c))]
    return {"bytes": rows * H * hd * 8 + sum(k for _, k in pairs) * K * hd * 4, "flops": 4 * hd * H * sum(p for p, _ in pairs)}


def draw(rng):
    between = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["rope", "paged", "paged", "paged", "prompt", "prompt"])
        hd = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 7, 8, 8, 12, 16])
        if heads * hd > 8192:
            continue
        kw = dict(heads=heads, kv_heads=kv_heads, hd=hd, page=rng.choice([16, 32, 48, 64, 128, 256]))
        if op == "rope":
            kw.update(n_seq=between(1, 64), n_rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                      base=rng.choice([1e4, 5e5, 1e6, 1e7]), past_lo=between(1, 50), past_hi=between(60, 2000))
            kw["rows"] = max(kw["n_seq"], between(1, 8192))
        elif op == "paged":
            per = rng.choice([1, 1, rng.randint(2, 8), between(9, 512)])
            kw.update(n_seq=between(1, 128), past_lo=between(1, 2000), past_hi=between(2001, 65536), window=rng.choice([0, 0, 0, between(32, 4096)]))
            kw["rows"] = kw["n_seq"] * per
        else:
            kw.update(n_seq=between(1, 24), window=rng.choice([0, 0, 0, between(32, 4096)]))
            kw["rows"] = max(kw["n_seq"], between(8, 8192))
        c = case(op, **kw)
        q, kv = _lengths(c)
        # room for the plain form's scores, and for its padded keys
        plain = 4 * len(q) * max(kv) * (heads * max(q) + 2 * kv_heads * hd)
        if op != "rope" and plain > 9e9 or sum(kv) * kv_heads * hd * 4 > 2e9:
            continue
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


_backend = []


def _be():
    """The program's one backend: device, stream and workspace."""
    if not _backend:
        from moe4all_b200 import CudaBackend

        _backend.append(CudaBackend(0))
    return _backend[0]


def prepare(c, seed):
    H, K, hd, rows, n = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["n_seq"]
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    q_len, kv_len = _lengths(c)
    s = {"c": c, "max_q": max(q_len), "max_kv": max(kv_len), "scale": hd ** -0.5}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s["cu_q"] = i32([sum(q_len[:i]) for i in range(n + 1)])
    if c["op"] != "prompt":
        # pages handed out in no order, as an allocator that has run for a while leaves them
        page = c["page"]
        need = [-(-k // page) for k in kv_len]
        n_pages, width = sum(need) + 3, max(need)
        ids = torch.randperm(n_pages, generator=gen, device="cuda").int()
        at = torch.arange(width, device="cuda")[None, :] + i32([sum(need[:i]) for i in range(n)])[:, None]
        s["page_table"] = torch.where(torch.arange(width, device="cuda")[None, :] < i32(need)[:, None], ids[at.clamp(max=n_pages - 1)], -1).int().contiguous()
        s["kv_len"] = i32(kv_len)
        s["k_cache"], s["v_cache"] = (normal(n_pages, K, page, hd).half() for _ in range(2))
    if c["op"] == "rope":
        # what one Linear for q, k and v leaves: rows of all three, side by side
        s["qkv"] = normal(rows, (H + 2 * K) * hd)
        s["q_norm"], s["k_norm"] = (1.0 + 0.2 * normal(hd) for _ in range(2))
        s["out"] = torch.zeros(rows, H * hd, device="cuda")
    else:
        # heads that look around and heads that look at a few keys
        s["q"] = (normal(rows, H, hd) * (0.5 + 2.5 * torch.rand(H, 1, generator=gen, device="cuda"))).reshape(rows, H * hd)
        s["out"] = torch.zeros(rows, H * hd, device="cuda")
        if c["op"] == "prompt":
            s["k"], s["v"] = (normal(rows, K, hd).half() for _ in range(2))
    if own:
        s["op"] = _op(s)
    return s


def _op(s):
    """The op that a program builds once for its buffers and calls every step."""
    from moe4all_b200 import Attention, RopeKv

    c, be = s["c"], _be()
    torch.cuda.synchronize()
    H, K, hd, rows = c["heads"], c["kv_heads"], c["hd"], c["rows"]
    w = be.wrap_tensor
    batch = dict(cu_q=w(s["cu_q"]), rows=rows, n_seq=c["n_seq"], n_head=H, n_kv=K, head_dim=hd)
    if c["op"] != "prompt":
        n_pages, _, page, _ = s["k_cache"].shape
        batch.update(kv_len=w(s["kv_len"]), page_table=w(s["page_table"]), n_pages=n_pages, page_size=page, max_pages=s["page_table"].shape[1])
    if c["op"] == "rope":
        wide = (H + 2 * K) * hd
        part = lambda first: be.wrap(s["qkv"].data_ptr() + 4 * first, 4 * (s["qkv"].numel() - first))
        norms = dict(q_norm=w(s["q_norm"]), k_norm=w(s["k_norm"]), norm_eps=EPS) if c["norm"] else {}
        return RopeKv(q=part(0), k=part(H * hd), v=part((H + K) * hd), q_stride=wide, k_stride=wide, v_stride=wide, q_out=w(s["out"]),
                      k_cache=w(s["k_cache"]), v_cache=w(s["v_cache"]), n_rot=c["n_rot"], interleaved=c["interleaved"], rope_base=c["base"], **norms, **batch)
    k, v = (s["k"], s["v"]) if c["op"] == "prompt" else (s["k_cache"], s["v_cache"])
    return Attention(q=w(s["q"]), k=w(k), v=w(v), out=w(s["out"]), scale=s["scale"], max_q=s["max_q"], window=c["window"], **batch)


def run(s):
    if own:
        if s["c"]["op"] == "rope":
            _be().rope_kv(s["op"])
            return [s["out"], s["k_cache"], s["v_cache"]]
        _be().attention(s["op"])
        return s["out"]
    return _plain_rope(s) if s["c"]["op"] == "rope" else _plain_attention(s)


def _places(s):
    """Each row's sequence, place among the sequence's new tokens, and position in it."""
    row = torch.arange(s["c"]["rows"], device="cuda")
    seq = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
    cu = s["cu_q"].long()
    t = row - cu[seq]
    q_len = cu[1:] - cu[:-1]
    past = s["kv_len"].long() - q_len if "kv_len" in s else torch.zeros_like(q_len)
    return seq, t, past[seq] + t, past, q_len


def _plain_rope(s):
    c = s["c"]
    H, K, hd, rows, rot = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["n_rot"]
    seq, _, pos, _, _ = _places(s)
    q, k, v = s["qkv"].view(rows, H + 2 * K, hd).split([H, K, K], 1)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    # angles in 64 bits: a far position times a frequency keeps few of 32
    freq = c["base"] ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        y = x.clone()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c["interleaved"] else (y[..., : rot // 2], y[..., rot // 2 : rot])
        first, second = a * cos - b * sin, a * sin + b * cos
        a.copy_(first)
        b.copy_(second)
        return y

    page = s["k_cache"].shape[2]
    at = s["page_table"].long()[seq, pos // page]
    s["k_cache"][at, :, pos % page] = turn(k).half()
    s["v_cache"][at, :, pos % page] = v.half()
    return [turn(q).reshape(rows, H * hd), s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    c = s["c"]
    H, K, hd, rows, n = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["n_seq"]
    g, max_q = H // K, s["max_q"]
    seq, t, _, past, q_len = _places(s)
    q = s["q"].new_zeros(n, max_q, K, g, hd)
    q[seq, t] = s["q"].view(rows, K, g, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, K, g * max_q, hd)
    if c["op"] == "prompt":
        k, v = s["q"].new_zeros(2, n, max_q, K, hd)
        k[seq, t], v[seq, t] = s["k"].float(), s["v"].float()
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    else:
        table = s["page_table"].long().clamp(min=0)
        k, v = (x[table].permute(0, 2, 1, 3, 4).reshape(n, K, -1, hd).float() for x in (s["k_cache"], s["v_cache"]))
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"])
    at = past[:, None] + torch.arange(max_q, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    hidden = key > at[..., None]
    if c["window"]:
        hidden |= key <= at[..., None] - c["window"]
    scores.view(n, K, g, max_q, -1).masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, v).div_(total)
    return out.view(n, K, g, max_q, hd).permute(0, 3, 1, 2, 4)[seq, t].reshape(rows, H * hd)


def exact(c, seed):
    s = prepare(c, seed)
    H, K, hd, rows = c["heads"], c["kv_heads"], c["hd"], c["rows"]
    g = H // K
    q_len, kv_len = _lengths(c)
    table = s["page_table"].tolist() if "page_table" in s else None
    if c["op"] == "rope":
        x = s["qkv"].double().view(rows, H + 2 * K, hd)
        out = torch.empty(rows, H, hd, dtype=torch.float64, device="cuda")
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        half = c["n_rot"] // 2
        freq = torch.tensor([float(c["base"]) ** (-2.0 * i / c["n_rot"]) for i in range(half)], dtype=torch.float64, device="cuda")
        where = torch.arange(half, device="cuda")
        first, second = (2 * where, 2 * where + 1) if c["interleaved"] else (where, where + half)

        def rotated(y, w, positions):
            if c["norm"]:
                y = y / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
            turned = torch.complex(y[..., first], y[..., second]) * z
            y = y.clone()
            y[..., first], y[..., second] = turned.real, turned.imag
            return y

        row = 0
        for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
            part, positions = x[row : row + nq], torch.arange(nk - nq, nk, device="cuda")
            out[row : row + nq] = rotated(part[:, :H], s["q_norm"], positions)
            pages = torch.tensor(table[i], device="cuda")[positions // c["page"]]
            kc[pages, :, positions % c["page"]] = rotated(part[:, H : H + K], s["k_norm"], positions)
            vc[pages, :, positions % c["page"]] = part[:, H + K :]
            row += nq
        return [out.view(rows, H * hd), kc, vc]
    out = torch.zeros(rows, H, hd, dtype=torch.float64, device="cuda")
    row = 0
    for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
        for h in range(K):
            if c["op"] == "prompt":
                k, v = s["k"][row : row + nq, h].double(), s["v"][row : row + nq, h].double()
            else:
                pages = torch.tensor(table[i][: -(-nk // c["page"])], device="cuda")
                k, v = (y[pages, h].reshape(-1, hd)[:nk].double() for y in (s["k_cache"], s["v_cache"]))
            step = max(1, min(nq, int(2e8 / (g * nk))))
            for a in range(0, nq, step):
                b = min(nq, a + step)
                q = s["q"].view(rows, H, hd)[row + a : row + b, h * g : (h + 1) * g].double()
                p = torch.arange(nk - nq + a, nk - nq + b, device="cuda")[:, None, None]
                j = torch.arange(nk, device="cuda")
                seen = (j <= p) & (j > p - c["window"]) if c["window"] else j <= p
                w = torch.softmax(torch.where(seen, (q @ k.T) * s["scale"], -math.inf), -1)
                out[row + a : row + b, h * g : (h + 1) * g] = w @ v
        row += nq
    return out.view(rows, H * hd)
