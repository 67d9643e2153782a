"""A decode step from token to token over a cache in 8 bits, as timed cases.

Five operators, each case is one pass through one of them:

  write   `CudaBackend.rope_kv` into 8-bit pages: per-head RMS norm and rotary embedding of a batch's new rows, their k and v quantised into
          the cache; and `CudaBackend.kv_read` of the rows that were put there, as a program does that goes on with what the cache holds.
  read    `CudaBackend.kv_read`: whole sequences out of 8-bit pages, to be kept elsewhere or handed to another program.
  paged   `CudaBackend.attention` over 8-bit pages: single tokens, speculative windows, chunks of a prompt behind a past.
  embed   `CudaBackend.embed`: rows of a quantised token table by number, scaled.
  sample  `CudaBackend.sample`: a token of each row of logits from given random numbers, with temperature, top-k, top-p and min-p by row.

The cache: codes u8 [pages, kv heads, page size, head size] and scale bytes u8 [.., head size / 16], one for 16 values.  A scale byte s is the f16 number
with the bits s << 7 (four significant bits), a value is (code - 128) times it.  Rows are f32 as everywhere in this framework.  Sizes are generic
ones for layers of the benchmark's hidden sizes (2048 to 7168): heads of 64, 128 and 256 (and sizes between), 1 to 16 query heads per kv head.
"""
import itertools
import math
import random

import numpy
import torch

own = False

EPS = 1e-6
FORMATS = {"f16": (1, 2), "q8_0": (32, 34), "q4_k": (256, 144), "q6_k": (256, 210)}  # values and bytes of a block


def case(op, name=None, **kw):
    if op == "embed":
        c = dict(op=op, rows=1, ne=2048, vocab=32000, format="q6_k", scale=1.0)
    elif op == "sample":
        c = dict(op=op, rows=1, vocab=32000, temperature=0.7, top_k=20, top_p=0.8, min_p=0.0, mixed=False)
    else:
        c = dict(op=op, heads=32, kv_heads=4, hd=128, n_seq=1, rows=1, past_lo=0, past_hi=0, page=64, window=0, n_rot=0, interleaved=False, norm=False, base=1e6, half=True)
    c.update(kw)
    for k in {"write": ("window", "half"), "read": ("heads", "window", "n_rot", "interleaved", "norm", "base"), "paged": ("n_rot", "interleaved", "norm", "base", "half")}.get(op, ()):
        del c[k]
    return dict(c, name=name) if name else c


def listed():
    return [
        # A decode step of 32 streams: one new row each, with the per-head norms of the models that have them.
        case("write", "write_step_32", n_seq=32, rows=32, past_lo=100, past_hi=2000, n_rot=128, norm=True),
        # The ragged last chunks of three prompts, of a model that rotates a quarter of its wide heads, pairs side by side.
        case("write", "write_chunks_4099", heads=16, kv_heads=2, hd=256, n_seq=3, rows=4099, past_lo=1, past_hi=900, n_rot=64, interleaved=True, page=16),
        # A short conversation that is put aside.
        case("read", "read_1x777", rows=777, page=16),
        # A batch of streams that move to another program, as f32 rows.
        case("read", "read_16x2000", n_seq=16, rows=32000, kv_heads=8, half=False),
        # One chat stream early in its conversation: the smallest call, latency alone.
        case("paged", "step_1x513", past_lo=512, past_hi=512, page=16),
        # A full decode batch with contexts of all lengths.
        case("paged", "step_64x8k", n_seq=64, rows=64, past_lo=700, past_hi=8000),
        # One stream over a long document.
        case("paged", "step_1x131072", past_lo=131071, past_hi=131071),
        # Chunked prefill: 512 new tokens or so each behind long pasts.
        case("paged", "chunk_4x512", n_seq=4, rows=2048, past_lo=3000, past_hi=16000),
        # The tokens of a decode step of 32 streams.
        case("embed", "embed_step_32", rows=32, vocab=150000),
        # A prompt batch of a model that scales its embeddings by the root of their width.
        case("embed", "embed_prompts_8191", rows=8191, ne=7168, format="q8_0", scale=math.sqrt(7168.0)),
        # Single-stream chat with the usual settings.
        case("sample", "sample_1x150000", vocab=150000),
        # A decode batch whose requests each have settings of their own, greedy ones among them.
        case("sample", "sample_64x150001", rows=64, vocab=150001, mixed=True),
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
    rows = c["rows"]
    if c["op"] == "embed":
        values, size = FORMATS[c["format"]]
        return {"bytes": rows * (c["ne"] // values * size + 4 * c["ne"] + 4), "flops": rows * c["ne"] * 2}
    if c["op"] == "sample":
        return {"bytes": rows * (4 * c["vocab"] + 28), "flops": rows * c["vocab"] * 4}
    K, hd = c["kv_heads"], c["hd"]
    token = 2 * K * (hd + hd // 16)  # bytes of k and v in the cache
    if c["op"] == "read":
        return {"bytes": rows * (token + 2 * K * hd * (2 if c["half"] else 4)), "flops": rows * 2 * K * hd}
    H = c["heads"]
    if c["op"] == "write":
        return {"bytes": rows * (4 * hd * (H + 2 * K) + 4 * H * hd + 2 * token + 4 * K * hd), "flops": rows * ((H + K) * (4 * hd * c["norm"] + 3 * c["n_rot"]) + 10 * K * hd)}
    pairs = [_pairs(q, kv, c["window"]) for q, kv in zip(*_lengths(c))]
    return {"bytes": rows * H * hd * 8 + sum(k for _, k in pairs) * token, "flops": 4 * hd * H * sum(p for p, _ in pairs)}


def draw(rng):
    between = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    most = {}
    for c in listed():
        for k, v in work(c).items():
            most[c["op"], k] = max(most.get((c["op"], k), 0), v)
    while True:
        op = rng.choice(["write", "read", "paged", "paged", "paged", "embed", "sample", "sample"])
        if op == "embed":
            f = rng.choice(list(FORMATS))
            c = case(op, rows=between(1, 8192), ne=256 * rng.randint(2, 28), vocab=between(2000, 150000), format=f, scale=rng.choice([1.0, 1.0, 0.5, 12.0, 45.25]))
            if c["vocab"] * c["ne"] > 4e8:
                continue
        elif op == "sample":
            c = case(op, rows=between(1, 64), vocab=between(1000, 150000), temperature=rng.choice([0.0, 0.6, 0.7, 1.0, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 20, 40, 50, between(1, 1000)]),
                     top_p=rng.choice([1.0, 1.0, 0.5, 0.8, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.02, 0.05, 0.1]), mixed=rng.random() < 0.4)
        else:
            hd = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 7, 8, 8, 12, 16])
            if heads * hd > 8192:
                continue
            kw = dict(heads=heads, kv_heads=kv_heads, hd=hd, page=rng.choice([16, 32, 48, 64, 128, 256]))
            if op == "write":
                kw.update(n_seq=between(1, 64), n_rot=rng.choice([hd, hd, hd // 2, 0]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                          base=rng.choice([1e4, 5e5, 1e6, 1e7]), past_lo=between(1, 50), past_hi=between(60, 2000))
                kw["rows"] = max(kw["n_seq"], between(1, 4099))
            elif op == "read":
                kw.update(n_seq=between(1, 64), half=rng.random() < 0.6)
                kw["rows"] = max(kw["n_seq"], between(1, 32000))
            else:
                per = rng.choice([1, 1, rng.randint(2, 8), between(9, 512)])
                kw.update(n_seq=between(1, 128), past_lo=between(1, 2000), past_hi=between(2001, 65536), window=rng.choice([0, 0, 0, between(32, 4096)]))
                kw["rows"] = kw["n_seq"] * per
            c = case(op, **kw)
            q, kv = _lengths(c)
            # room for the plain form's scores, and for its padded keys
            if op == "paged" and (4 * len(q) * max(kv) * (heads * max(q) + 2 * kv_heads * hd) > 9e9 or sum(kv) * kv_heads * hd * 4 > 2e9):
                continue
        if all(v <= most[op, k] for k, v in work(c).items()):
            return c


_backend = []


def _be():
    """The program's one backend: device, stream and workspace."""
    if not _backend:
        from moe4all_b200 import CudaBackend

        _backend.append(CudaBackend(0))
    return _backend[0]


def _scale_of(s):
    """Scale bytes as the numbers that they are (f16 numbers, in 32 bits)."""
    e, m = (s >> 3).int(), (s & 7).float()
    return torch.where(e > 0, torch.ldexp(8.0 + m, e - 18), torch.ldexp(m, torch.full_like(e, -17)))


def _quantise(x):
    """[.., hd] f32 -> codes [.., hd] and scale bytes [.., hd / 16]: a 16th part of a row has the least scale of four significant bits that 127 of
    reach its largest magnitude."""
    x = x.unflatten(-1, (-1, 16))
    t = x.abs().amax(-1) / 127.0
    normal = ((t.contiguous().view(torch.int32) + 0xFFFFF) >> 20) - (112 << 3)
    s = torch.where(t < 2.0 ** -14, torch.ceil(t * 2.0 ** 17).int(), normal)
    d = _scale_of(s)
    q = torch.round(x * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))[..., None]).clamp(-127, 127)
    return (q + 128).flatten(-2).to(torch.uint8), s.to(torch.uint8)


def _values(codes, s):
    """The numbers that codes and scale bytes stand for, in 32 bits."""
    return ((codes.float() - 128).unflatten(-1, (-1, 16)) * _scale_of(s)[..., None]).flatten(-2)


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s = {"c": c}
    rows = c["rows"]
    if c["op"] == "embed":
        values, size = FORMATS[c["format"]]
        blocks = c["vocab"] * (c["ne"] // values)
        if c["format"] == "f16":
            s["table"] = normal(c["vocab"], c["ne"]).mul_(0.02).half().view(torch.uint8)
        else:
            t = torch.randint(0, 256, (blocks, size), generator=gen, device="cuda", dtype=torch.uint8)
            d = (1e-4 + 9e-4 * uniform(blocks, 2)).half().view(torch.uint8)
            if c["format"] == "q6_k":
                t[:, 208:] = d[:, :2]
            else:
                t[:, : 4 if c["format"] == "q4_k" else 2] = d[:, : 4 if c["format"] == "q4_k" else 2]
            s["table"] = t.view(c["vocab"], -1)
        # few tokens often, many seldom
        s["ids"] = (c["vocab"] * uniform(rows) ** 4).int().clamp_(max=c["vocab"] - 1)
        s["out"] = torch.zeros(rows, c["ne"], device="cuda")
        return s
    if c["op"] == "sample":
        V = c["vocab"]
        # a bulk, a slope towards the likely tokens, and a few of these far ahead; rows more and less sure
        x = normal(rows, V) * 2.2 + 6.0 * uniform(rows, V) ** 12
        head = torch.randint(0, V, (rows, 24), generator=gen, device="cuda")
        x.scatter_add_(1, head, (5.0 + 8.0 * uniform(rows, 24)) * uniform(rows, 1))
        s["logits"], s["u"] = x, uniform(rows)
        pick = lambda options, each: torch.tensor(options, device="cuda")[torch.randint(0, len(options), (rows,), generator=gen, device="cuda")] if c["mixed"] else torch.tensor([each] * rows, device="cuda")
        s["temperature"] = pick([0.0, 0.6, 0.7, 1.0, 1.0, 1.3], c["temperature"]).float()
        s["top_k"] = pick([0, 0, 20, 40, 50, 200, 1000], c["top_k"]).int()
        s["top_p"] = pick([1.0, 1.0, 0.8, 0.9, 0.95], c["top_p"]).float()
        s["min_p"] = pick([0.0, 0.0, 0.0, 0.02, 0.05], c["min_p"]).float()
        s["ids"], s["prob"] = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        return s
    K, hd, n, page = c["kv_heads"], c["hd"], c["n_seq"], c["page"]
    q_len, kv_len = _lengths(c)
    s.update(max_q=max(q_len), max_kv=max(kv_len), scale=hd ** -0.5)
    s["cu_q"] = i32([sum(q_len[:i]) for i in range(n + 1)])
    # pages handed out in no order, as an allocator that has run for a while leaves them
    need = [-(-k // page) for k in kv_len]
    n_pages, width = sum(need) + 3, max(need)
    ids = torch.randperm(n_pages, generator=gen, device="cuda").int()
    at = torch.arange(width, device="cuda")[None, :] + i32([sum(need[:i]) for i in range(n)])[:, None]
    s["page_table"] = torch.where(torch.arange(width, device="cuda")[None, :] < i32(need)[:, None], ids[at.clamp(max=n_pages - 1)], -1).int().contiguous()
    s["kv_len"] = i32(kv_len)
    # (keys have channels that are larger than others)
    wide = 0.5 + 2.0 * uniform(hd) ** 6
    for name, by in (("k", wide), ("v", torch.ones_like(wide))):
        s[name + "_cache"], s[name + "_scale"] = _quantise(normal(n_pages, K, page, hd) * by)
    if c["op"] == "paged":
        H = c["heads"]
        # heads that look around and heads that look at a few keys
        s["q"] = (normal(rows, H, hd) * (0.5 + 2.5 * uniform(H, 1))).reshape(rows, H * hd)
        s["out"] = torch.zeros(rows, H * hd, device="cuda")
        return s
    if c["op"] == "write":
        H = c["heads"]
        # what one Linear for q, k and v leaves: rows of all three, side by side
        s["qkv"] = normal(rows, (H + 2 * K) * hd)
        s["q_norm"], s["k_norm"] = (1.0 + 0.2 * normal(hd) for _ in range(2))
        s["out"] = torch.zeros(rows, H * hd, device="cuda")
    s["k_rows"], s["v_rows"] = (torch.zeros(rows, K * hd, device="cuda", dtype=torch.float16 if c.get("half", True) else torch.float32) for _ in range(2))
    return s


def _ops(s):
    """The ops that a program builds once for its buffers and calls every step."""
    from moe4all_b200 import Attention, DType, Embed, KvRead, RopeKv, Sample

    c, w, be = s["c"], _be().wrap_tensor, _be()
    torch.cuda.synchronize()
    rows = c["rows"]
    if c["op"] == "embed":
        form = {"f16": DType.F16, "q8_0": DType.Q8_0, "q4_k": DType.Q4K, "q6_k": DType.Q6K}[c["format"]]
        return [Embed(table=w(s["table"]), dtype=form, ids=w(s["ids"]), dst=w(s["out"]), rows=rows, ne=c["ne"], n_vocab=c["vocab"], scale=c["scale"])]
    if c["op"] == "sample":
        return [Sample(logits=w(s["logits"]), u=w(s["u"]), ids=w(s["ids"]), prob=w(s["prob"]), rows=rows, n_vocab=c["vocab"], temperature=w(s["temperature"]), top_k=w(s["top_k"]),
                       top_p=w(s["top_p"]), min_p=w(s["min_p"]))]
    K, hd = c["kv_heads"], c["hd"]
    kc, vc, ks, vs = (w(s[k]) for k in ("k_cache", "v_cache", "k_scale", "v_scale"))
    batch = dict(cu_q=w(s["cu_q"]), rows=rows, n_seq=c["n_seq"], n_kv=K, head_dim=hd, kv_len=w(s["kv_len"]), page_table=w(s["page_table"]), n_pages=s["k_cache"].shape[0],
                 page_size=c["page"], max_pages=s["page_table"].shape[1], k_scale=ks, v_scale=vs)
    if c["op"] == "paged":
        return [Attention(q=w(s["q"]), k=kc, v=vc, out=w(s["out"]), scale=s["scale"], max_q=s["max_q"], window=c["window"], n_head=c["heads"], **batch)]
    read = KvRead(k_cache=kc, v_cache=vc, k=w(s["k_rows"]), v=w(s["v_rows"]), f16=c.get("half", True), **batch)
    if c["op"] == "read":
        return [read]
    H = c["heads"]
    wide = (H + 2 * K) * hd
    part = lambda first: be.wrap(s["qkv"].data_ptr() + 4 * first, 4 * (s["qkv"].numel() - first))
    norms = dict(q_norm=w(s["q_norm"]), k_norm=w(s["k_norm"]), norm_eps=EPS) if c["norm"] else {}
    return [RopeKv(q=part(0), k=part(H * hd), v=part((H + K) * hd), q_stride=wide, k_stride=wide, v_stride=wide, q_out=w(s["out"]), k_cache=kc, v_cache=vc, n_head=H,
                   n_rot=c["n_rot"], interleaved=c["interleaved"], rope_base=c["base"], **norms, **batch), read]


def run(s):
    op = s["c"]["op"]
    if own:
        if "ops" not in s:
            s["ops"] = _ops(s)
        be, ops = _be(), s["ops"]
        if op == "embed":
            be.embed(ops[0])
            return s["out"]
        if op == "sample":
            be.sample(ops[0])
            return [s["ids"], s["prob"]]
        if op == "paged":
            be.attention(ops[0])
            return s["out"]
        if op == "read":
            be.kv_read(ops[0])
            return [s["k_rows"], s["v_rows"]]
        be.rope_kv(ops[0])
        be.kv_read(ops[1])
        return [s["out"], s["k_rows"], s["v_rows"]]
    return {"embed": _plain_embed, "sample": _plain_sample, "paged": _plain_attention, "read": _plain_read, "write": _plain_write}[op](s)


def _plain_embed(s):
    c = s["c"]
    b = s["table"][s["ids"].long()]
    if c["format"] == "f16":
        return b.view(torch.float16).float() * c["scale"]
    values, size = FORMATS[c["format"]]
    b = b.view(c["rows"], c["ne"] // values, size)
    half = lambda at: b[..., at : at + 2].contiguous().view(torch.float16).float()
    if c["format"] == "q8_0":
        x = half(0) * b[..., 2:].contiguous().view(torch.int8).float()
    elif c["format"] == "q4_k":
        # eight groups of 32: six bits of scale and of minimum each, the last four's upper two bits with the first four
        g = b[..., 4:16].int()
        sc = torch.cat([g[..., 0:4] & 63, (g[..., 8:12] & 15) | (g[..., 0:4] >> 6 << 4)], -1).float()
        mn = torch.cat([g[..., 4:8] & 63, (g[..., 8:12] >> 4) | (g[..., 4:8] >> 6 << 4)], -1).float()
        n = b[..., 16:].unflatten(-1, (4, 32))
        n = torch.stack([n & 15, n >> 4], -2).flatten(-3, -2).float()
        x = (half(0) * sc)[..., None] * n - (half(2) * mn)[..., None]
    else:
        # two halves of 128: 64 bytes of low bits, 32 of upper ones, eight scales
        lo, hi, sc = b[..., :128].unflatten(-1, (2, 2, 32)), b[..., 128:192].unflatten(-1, (2, 32)), b[..., 192:208].contiguous().view(torch.int8).float()
        q = torch.stack([lo[..., 0, :] & 15, lo[..., 1, :] & 15, lo[..., 0, :] >> 4, lo[..., 1, :] >> 4], -2).int()
        q = q | (torch.stack([hi & 3, hi >> 2 & 3, hi >> 4 & 3, hi >> 6], -2).int() << 4)
        x = (half(208) * sc).repeat_interleave(16, -1) * (q - 32).flatten(-3).float()
    return x.reshape(c["rows"], c["ne"]) * c["scale"]


def _plain_sample(s):
    # in 64 bits: a sum of 32 decides differently next to a border
    x = s["logits"].double()
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    T = s["temperature"].double()[:, None]
    greedy = T <= 0
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / torch.where(greedy, torch.ones_like(T), T)))
    order = x.sort(dim=1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    rank = torch.arange(V, device="cuda")
    k = torch.where(greedy[:, 0], torch.ones_like(s["top_k"]), torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], V)))
    keep = rank < k[:, None]
    sums = (ws * keep).cumsum(1)
    p = s["top_p"].double()[:, None]
    before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], 1)
    keep &= (p >= 1) | (before < p * sums[:, -1:])
    keep &= ws >= s["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, ws * keep)
    cdf = kept.cumsum(1)
    ids = torch.searchsorted(cdf, s["u"].double()[:, None] * cdf[:, -1:], right=True)
    last = (kept > 0).long().mul_(rank + 1).amax(1, keepdim=True) - 1
    ids = torch.minimum(ids, last)
    return [ids[:, 0].int(), (kept.gather(1, ids) / cdf[:, -1:])[:, 0].float()]


def _places(s):
    """Each row's sequence, place among the sequence's new tokens, and position in it."""
    row = torch.arange(s["c"]["rows"], device="cuda")
    seq = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
    cu = s["cu_q"].long()
    t = row - cu[seq]
    past = s["kv_len"].long() - (cu[1:] - cu[:-1])
    return seq, t, past[seq] + t, past


def _plain_read(s):
    page = s["k_cache"].shape[2]
    seq, _, pos, _ = _places(s)
    at = s["page_table"].long()[seq, pos // page]
    return [_values(s[n + "_cache"][at, :, pos % page], s[n + "_scale"][at, :, pos % page]).flatten(1).to(s[n + "_rows"].dtype) for n in "kv"]


def _plain_write(s):
    c = s["c"]
    H, K, hd, rows, rot = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["n_rot"]
    seq, _, pos, _ = _places(s)
    q, k, v = s["qkv"].view(rows, H + 2 * K, hd).split([H, K, K], 1)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    # angles in 64 bits: a far position times a frequency keeps few of 32
    freq = c["base"] ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
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
    s["k_cache"][at, :, pos % page], s["k_scale"][at, :, pos % page] = _quantise(turn(k))
    s["v_cache"][at, :, pos % page], s["v_scale"][at, :, pos % page] = _quantise(v)
    return [turn(q).reshape(rows, H * hd)] + _plain_read(s)


def _plain_attention(s):
    c = s["c"]
    H, K, hd, rows, n = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["n_seq"]
    g, max_q = H // K, s["max_q"]
    seq, t, _, past = _places(s)
    q = s["q"].new_zeros(n, max_q, K, g, hd)
    q[seq, t] = s["q"].view(rows, K, g, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, K, g * max_q, hd)
    table = s["page_table"].long().clamp(min=0)
    k, v = (_values(s[x + "_cache"][table], s[x + "_scale"][table]).permute(0, 2, 1, 3, 4).reshape(n, K, -1, hd) for x in "kv")
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


def _exact_values(codes, scales):
    """The same numbers by way of the f16 bits that a scale byte stands for, in 64 bits."""
    d = (scales.to(torch.int16) << 7).contiguous().view(torch.float16).double()
    return (codes.double() - 128.0) * d.repeat_interleave(16, -1)


def _exact_rounded(x):
    """What a cache holds of x [.., hd]: 16 at a time the nearest multiples of the least scale that reaches, in 64 bits."""
    y = x.reshape(-1, 16)
    a = y.abs().max(-1).values / 127.0
    e = torch.floor(torch.log2(a.clamp(min=1e-30))).clamp(min=-14.0) - 3
    d = torch.ceil(a / 2.0 ** e) * 2.0 ** e
    return (torch.round(y / d.clamp(min=1e-30)[:, None]) * d[:, None]).view(x.shape)


def _exact_sample(s):
    x = s["logits"].cpu().numpy().astype(numpy.float64)
    T, k, p, m, u = (s[n].cpu().numpy().astype(numpy.float64) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    ids, prob = [], []
    for i in range(x.shape[0]):
        if T[i] <= 0:
            ids.append(int(numpy.argmax(x[i])))
            prob.append(1.0)
            continue
        order = numpy.lexsort((numpy.arange(x.shape[1]), -x[i]))
        w = numpy.exp((x[i][order] - x[i].max()) / T[i])
        n = min(int(k[i]), w.size) if k[i] > 0 else w.size
        sums = numpy.cumsum(w[:n])
        if p[i] < 1:
            n = min(n, 1 + int(numpy.sum(sums < p[i] * sums[-1])))
        n = int(numpy.sum(w[:n] >= m[i]))
        chosen = numpy.sort(order[:n])
        w = numpy.exp((x[i][chosen] - x[i].max()) / T[i])
        cdf = numpy.cumsum(w)
        j = min(int(numpy.sum(cdf <= u[i] * cdf[-1])), int(numpy.flatnonzero(w)[-1]))
        ids.append(int(chosen[j]))
        prob.append(w[j] / cdf[-1])
    return [torch.tensor(ids, dtype=torch.int32), torch.tensor(prob, dtype=torch.float64)]


def _exact_embed(s):
    c = s["c"]
    rows = s["table"].cpu().numpy()[s["ids"].cpu().numpy()]
    if c["format"] == "f16":
        return torch.from_numpy(rows.view(numpy.float16).astype(numpy.float64) * c["scale"])
    values, size = FORMATS[c["format"]]
    b = rows.reshape(-1, size)
    out = numpy.empty((b.shape[0], values))
    f16 = lambda at: numpy.ascontiguousarray(b[:, at : at + 2]).view(numpy.float16).astype(numpy.float64)[:, 0]
    if c["format"] == "q8_0":
        out[:] = f16(0)[:, None] * b[:, 2:].view(numpy.int8)
    elif c["format"] == "q4_k":
        for j in range(8):
            if j < 4:
                sc, mn = b[:, 4 + j] & 63, b[:, 8 + j] & 63
            else:
                sc, mn = (b[:, 8 + j] & 15) + 16 * (b[:, j] >> 6), (b[:, 8 + j] >> 4) + 16 * (b[:, 4 + j] >> 6)
            byte = b[:, 16 + 32 * (j // 2) : 48 + 32 * (j // 2)]
            out[:, 32 * j : 32 * j + 32] = (f16(0) * sc)[:, None] * (byte >> 4 if j & 1 else byte & 15) - (f16(2) * mn)[:, None]
    else:
        scales = numpy.ascontiguousarray(b[:, 192:208]).view(numpy.int8).astype(numpy.float64)
        for i in range(256):
            half, part, lane = i // 128, i % 128 // 32, i % 32
            low = b[:, 64 * half + 32 * (part % 2) + lane] >> (4 * (part // 2)) & 15
            high = b[:, 128 + 32 * half + lane] >> (2 * part) & 3
            out[:, i] = f16(208) * scales[:, i // 16] * (low + 16.0 * high - 32.0)
    return torch.from_numpy(out.reshape(c["rows"], c["ne"]) * c["scale"])


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] in ("embed", "sample"):
        return (_exact_embed if c["op"] == "embed" else _exact_sample)(s)
    K, hd, rows = c["kv_heads"], c["hd"], c["rows"]
    q_len, kv_len = _lengths(c)
    table = s["page_table"].tolist()
    if c["op"] == "read":
        out = []
        for n in "kv":
            parts = []
            for i, nk in enumerate(kv_len):
                pages = torch.tensor(table[i][: -(-nk // c["page"])], device="cuda")
                parts.append(_exact_values(s[n + "_cache"][pages], s[n + "_scale"][pages]).transpose(1, 2).reshape(-1, K * hd)[nk - q_len[i] : nk])
            out.append(torch.cat(parts))
        return out
    H = c["heads"]
    if c["op"] == "write":
        x = s["qkv"].double().view(rows, H + 2 * K, hd)
        half = c["n_rot"] // 2
        freq = torch.tensor([float(c["base"]) ** (-2.0 * i / c["n_rot"]) for i in range(half)], dtype=torch.float64, device="cuda")
        where = torch.arange(half, device="cuda")
        first, second = (2 * where, 2 * where + 1) if c["interleaved"] else (where, where + half)
        positions = torch.cat([torch.arange(nk - nq, nk, device="cuda") for nq, nk in zip(q_len, kv_len)])

        def rotated(y, w):
            if c["norm"]:
                y = y / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
            turned = torch.complex(y[..., first], y[..., second]) * z
            y = y.clone()
            y[..., first], y[..., second] = turned.real, turned.imag
            return y

        return [rotated(x[:, :H], s["q_norm"]).reshape(rows, -1), _exact_rounded(rotated(x[:, H : H + K], s["k_norm"])).reshape(rows, -1),
                _exact_rounded(x[:, H + K :].contiguous()).reshape(rows, -1)]
    g = H // K
    out = torch.zeros(rows, H, hd, dtype=torch.float64, device="cuda")
    row = 0
    for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
        for h in range(K):
            pages = torch.tensor(table[i][: -(-nk // c["page"])], device="cuda")
            k, v = (_exact_values(s[n + "_cache"][pages, h], s[n + "_scale"][pages, h]).reshape(-1, hd)[:nk] for n in "kv")
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
