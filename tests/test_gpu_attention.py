"""GPU: rope_kv and attention through the C ABI against the formulas in 64 bits.

Tolerances count roundings.  Attention, with M = the largest |v|: the scores' error dS is that of q's two f16 pieces (2^-22 of it), of hd / 8
accumulations in f32 (2^-23 each) and of the exponent's argument, all relative to scale * sum |q| |k|; it enters numerator and denominator
once each.  The weights' two pieces and the exponential add 2^-20, the accumulation over n keys n / 8 steps of 2^-23 at most:
    |error| <= M (2 dS + 2^-20 + n / 8 2^-23),  dS = scale max sum |q| |k| (2^-21 + hd / 8 2^-23).
rope_kv: a dozen f32 operations on a pair, 2^-20 of its magnitude; the cache another half step of f16 (2^-11, 2^-25 among subnormals)."""
import dataclasses
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NAN = float("nan")


class Batch:
    """A batch of sequences on the GPU.  Whatever no row may see is NaN: stale tokens, pages nobody owns, rows of no sequence."""

    def __init__(self, q_lens, pasts, H, K, hd, page=0, seed=0, lead=0, tail=0, spare=2, q_pad=0, out_pad=0, spread=1.0):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.q_lens, self.pasts, self.H, self.K, self.hd, self.page = q_lens, pasts, H, K, hd, page
        self.kv = [max(0, a + b) for a, b in zip(q_lens, pasts)]
        n = len(q_lens)
        self.cu = [lead + sum(q_lens[:i]) for i in range(n + 1)]
        self.rows = self.cu[-1] + tail
        self.q_stride, self.out_stride = H * hd + q_pad, H * hd + out_pad
        self.q = torch.full((self.rows, self.q_stride), NAN, device="cuda")
        self.q[lead : self.cu[-1], : H * hd] = spread * r(self.cu[-1] - lead, H * hd)
        self.out = torch.full((self.rows, self.out_stride), 7.5, device="cuda")
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        self.cu_t, self.kv_t = i32(self.cu), i32(self.kv)
        if page:
            need = [-(-k // page) for k in self.kv]
            self.n_pages, self.width = max(1, sum(need) + spare), max(1, max(need))
            ids = torch.randperm(self.n_pages, generator=g, device="cuda").int().tolist()
            self.tables, at = [], 0
            for m in need:
                self.tables.append(ids[at : at + m])
                at += m
            self.table_t = i32([t + [-1] * (self.width - len(t)) for t in self.tables])
            self.k, self.v = (torch.full((self.n_pages, K, page, hd), NAN, device="cuda", dtype=torch.float16) for _ in range(2))
            for s in range(n):
                for c in (self.k, self.v):
                    self.put(c, s, r(self.kv[s], K, hd).half())
        else:
            self.k, self.v = (torch.full((self.rows, K, hd), NAN, device="cuda", dtype=torch.float16) for _ in range(2))
            for c in (self.k, self.v):
                c[lead : self.cu[-1]] = r(self.cu[-1] - lead, K, hd).half()

    def at(self, s):
        """Index of sequence s's tokens in a cache, as (page, slot) or rows."""
        import torch

        i = torch.arange(self.kv[s], device="cuda")
        if not self.page:
            return (self.cu[s] + i,)
        return torch.tensor(self.tables[s], device="cuda", dtype=torch.long)[i // self.page], i % self.page

    def put(self, cache, s, x):
        if not self.kv[s]:
            return
        if self.page:
            a, b = self.at(s)
            cache[a, :, b] = x
        else:
            cache[self.at(s)[0]] = x

    def get(self, cache, s):
        """[tokens, kv heads, hd]"""
        if not self.kv[s]:
            return cache.new_zeros(0, self.K, self.hd)
        if self.page:
            a, b = self.at(s)
            return cache[a, :, b]
        return cache[self.at(s)[0]]

    def fields(self, be):
        w = be.wrap_tensor
        f = dict(cu_q=w(self.cu_t), rows=self.rows, n_seq=len(self.q_lens), n_head=self.H, n_kv=self.K, head_dim=self.hd)
        if self.page:
            f.update(kv_len=w(self.kv_t), page_table=w(self.table_t), n_pages=self.n_pages, page_size=self.page, max_pages=self.width)
        return f

    def op(self, be, **kw):
        from moe4all_b200 import Attention

        w = be.wrap_tensor
        f = dict(q=w(self.q), k=w(self.k), v=w(self.v), out=w(self.out), scale=self.hd ** -0.5, q_stride=self.q_stride, out_stride=self.out_stride, max_q=max(self.q_lens))
        return Attention(**{**f, **self.fields(be), **kw})

    def ref(self, window=0, scale=None):
        """Attention in 64 bits, and the bound of the error: the rows' results, by (row, head, value)."""
        import torch

        scale = self.hd ** -0.5 if scale is None else scale
        out = self.out.clone().double()
        worst = 0.0
        for s, (n, cu) in enumerate(zip(self.q_lens, self.cu)):
            if not n:
                continue
            g = self.H // self.K
            q = self.q[cu : cu + n, : self.H * self.hd].double().view(n, self.K, g, self.hd)
            k, v = self.get(self.k, s).double(), self.get(self.v, s).double()
            pos = torch.arange(n, device="cuda")[:, None] + self.kv[s] - n
            j = torch.arange(self.kv[s], device="cuda")
            seen = (j <= pos) & ((j > pos - window) if window else True)
            for h in range(self.K):
                sc = torch.einsum("tgd,jd->tgj", q[:, h], k[:, h]) * scale
                sc = torch.where(seen[:, None], sc, -math.inf)
                w = torch.softmax(sc, -1)
                w = torch.where(seen[:, None], w, 0.0)
                # (a value that is not finite counts where it is seen, not as 0 x value)
                plain = torch.nan_to_num(v[:, h], nan=0.0, posinf=0.0, neginf=0.0)
                o = torch.einsum("tgj,jd->tgd", w, plain)
                odd = torch.where(torch.isfinite(v[:, h]), 0.0, v[:, h])
                hit = (odd != 0).any(1).nonzero().flatten().tolist()
                for x in hit:
                    o = o + torch.where(seen[:, x][:, None, None], odd[x], 0.0)
                out[cu : cu + n, : self.H * self.hd].view(n, self.H, self.hd)[:, h * g : (h + 1) * g] = o
                if len(j):
                    fin = torch.isfinite(k[:, h])
                    dS = abs(scale) * float(torch.einsum("tgd,jd->tgj", q[:, h].nan_to_num().abs(), torch.where(fin, k[:, h], 0.0).abs()).max()) * (2 ** -21 + self.hd / 8 * 2 ** -23)
                    worst = max(worst, float(plain.abs().max()) * (2 * dS + 2 ** -20 + len(j) / 8 * 2 ** -23))
        return out, worst


def check(be, b, window=0, scale=None, **kw):
    import torch

    want, tol = b.ref(window, scale)
    torch.cuda.synchronize()
    be.attention(b.op(be, window=window, **({} if scale is None else {"scale": scale}), **kw))
    be.sync()
    got = b.out.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    assert not off.isnan().any(), "NaN where there should be none, or the other way round"
    assert float(off.max()) <= tol, f"off by {float(off.max()):.3g}, allowed {tol:.3g}"
    return want


HEADS = [(8, 2, 64), (8, 1, 128), (16, 2, 256), (6, 2, 192), (3, 3, 80), (14, 2, 96), (16, 1, 128), (10, 2, 112), (4, 4, 16), (2, 1, 240)]


@pytest.mark.parametrize("H,K,hd", HEADS)
@pytest.mark.parametrize("path", [1, 2])
def test_single_tokens_over_pages(backend, H, K, hd, path):
    check(backend, Batch([1, 1, 1, 1, 1], [0, 1, 130, 700, 2047], H, K, hd, page=16, seed=hd), path=path)


@pytest.mark.parametrize("page", [16, 48, 64, 128, 256, 1024])
@pytest.mark.parametrize("path", [1, 2])
def test_page_sizes(backend, page, path):
    check(backend, Batch([1, 3, 5], [500, 63, 1200], 8, 2, 128, page=page, seed=page, spare=5), path=path)


@pytest.mark.parametrize("H,K,hd", HEADS)
@pytest.mark.parametrize("path", [1, 2])
def test_prompts_packed(backend, H, K, hd, path):
    check(backend, Batch([1, 17, 128, 0, 300, 2], [0] * 6, H, K, hd, seed=hd + 1), path=path)


@pytest.mark.parametrize("H,K,hd", HEADS)
@pytest.mark.parametrize("path", [1, 2])
def test_chunks_over_pages(backend, H, K, hd, path):
    check(backend, Batch([33, 1, 130, 5, 64], [100, 900, 257, 0, 127], H, K, hd, page=32, seed=hd + 2), path=path)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 500, 5000])
@pytest.mark.parametrize("path", [1, 2])
def test_windows(backend, window, path):
    check(backend, Batch([1, 40, 200, 1], [1000, 300, 0, 3], 8, 2, 128, page=64, seed=window), window=window, path=path)


@pytest.mark.parametrize("window", [1, 70, 300])
def test_windows_packed(backend, window):
    for path in (1, 2):
        check(backend, Batch([129, 1, 260], [0, 0, 0], 4, 2, 64, seed=window), window=window, path=path)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("page", [0, 16])
def test_rows_of_no_sequence_stay(backend, path, page):
    # 3 rows ahead of the first sequence, 5 behind the last, sequences without rows in between; padded strides
    b = Batch([0, 4, 0, 1, 0], [0] * 5 if not page else [9, 20, 0, 33, 50], 8, 2, 64, page=page, lead=3, tail=5, q_pad=12, out_pad=8, seed=3)
    check(backend, b, path=path)
    assert bool((b.out[:3] == 7.5).all()) and bool((b.out[-5:] == 7.5).all()) and bool((b.out[:, 512:] == 7.5).all())


@pytest.mark.parametrize("path", [1, 2])
def test_rows_that_see_nothing(backend, path):
    # fewer tokens in the cache than new rows: the rows in front have negative positions
    b = Batch([5, 3, 200], [-2, -3, -150], 8, 2, 128, page=16, seed=4)
    check(backend, b, path=path)
    assert bool((b.out[:2] == 0).all()) and bool((b.out[5:8] == 0).all()) and bool((b.out[8:158] == 0).all()) and bool((b.out[158:] != 0).any())


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("page", [0, 32])
@pytest.mark.parametrize("bits", [0x7E00, 0x7C00, 0xFC00])
def test_what_a_row_may_not_see_does_not_reach_it(backend, path, page, bits):
    # keys and values of later tokens of the same sequence that are not finite: the rows before them stay clean, the rows that see them do not
    import torch

    x = torch.tensor([bits], dtype=torch.int32, device="cuda").short().view(torch.float16)
    b = Batch([12, 140], [0, 0] if not page else [37, 200], 8, 2, 64, page=page, seed=5)
    for s, t in ((0, 7), (1, 100)):
        for cache, where in ((b.v, slice(10, 20)),):
            y = b.get(cache, s).clone()
            y[b.kv[s] - b.q_lens[s] + t, 1, where] = x
            b.put(cache, s, y)
    want = check(backend, b, path=path)
    assert not want[:7].isnan().any() and not want[:7].isinf().any()
    assert bool((~torch.isfinite(want[7:12].view(5, 8, 64)[:, 4:, 10:20])).all())
    # a key that is NaN: rows from it on are NaN in the heads that read it
    k = b.get(b.k, 1).clone()
    k[b.kv[1] - 140 + 100, 0, 5] = NAN
    b.put(b.k, 1, k)
    want = check(backend, b, path=path)
    assert bool(want[12 + 100 :].view(40, 8, 64)[:, :4].isnan().all()) and bool(torch.isfinite(want[12 : 12 + 100].view(100, 8, 64)[:, :4]).all())


@pytest.mark.parametrize("path", [1, 2])
def test_window_hides_bad_values_behind_it(backend, path):
    b = Batch([1, 30], [300, 300], 4, 1, 128, page=16, seed=6)
    for s in range(2):
        y = b.get(b.v, s).clone()
        y[:200] = NAN
        b.put(b.v, s, y)
        y = b.get(b.k, s).clone()
        y[:200] = float("inf")
        b.put(b.k, s, y)
    want = check(backend, b, window=64, path=path)
    assert bool(want.isfinite().all())


@pytest.mark.parametrize("path", [1, 2])
def test_queries_that_are_not_finite_keep_to_themselves(backend, path):
    b = Batch([6, 1], [50, 99], 8, 2, 64, page=16, seed=7)
    b.q[2, 64 * 3 + 5] = NAN
    want = check(backend, b, path=path)
    assert bool(want[2, 64 * 3 : 64 * 4].isnan().all()) and int(want.isnan().any(1).sum()) == 1


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 3e30])
def test_scales_of_q(backend, path, size):
    # q far outside f16's range, brought back by the scale
    b = Batch([1, 20], [200, 70], 8, 2, 128, page=16, seed=8, spread=size)
    check(backend, b, scale=1.0 / size / 11.0, path=path)


@pytest.mark.parametrize("path", [1, 2])
def test_sharp_and_growing_scores(backend, path):
    # the running maximum grows by far more than the slack again and again, and one key takes nearly all the weight
    b = Batch([1, 1, 150], [1500, 600, 600], 8, 2, 64, page=16, seed=9)
    for s in range(3):
        y = b.get(b.k, s)
        ramp = (1.0 + 5.0 * (y.new_tensor(range(b.kv[s])) / b.kv[s]))[:, None, None]
        b.put(b.k, s, (b.q[b.cu[s], :64] * ramp * 0.5).half().expand(b.kv[s], 2, 64) if s else y * ramp.half())
    check(backend, b, scale=1.0, path=path)


@pytest.mark.parametrize("path", [1, 2])
def test_same_bits_every_time_and_shared_pages(backend, path):
    # items cut between CTAs are joined in their order whoever finishes last; sequences share the pages of a common prefix
    import torch

    b = Batch([3, 3, 1], [6000, 5000, 4000], 16, 2, 128, page=64, seed=10)
    b.tables[1][:40] = b.tables[0][:40]
    b.tables[2] = list(b.tables[0][: len(b.tables[2])])
    b.table_t = torch.tensor([t + [-1] * (b.width - len(t)) for t in b.tables], dtype=torch.int32, device="cuda")
    check(backend, b, path=path)
    first = b.out.clone()
    op = b.op(backend, path=path)
    for _ in range(20):
        b.out.fill_(0)
        torch.cuda.synchronize()
        backend.attention(op)
        backend.sync()
        assert torch.equal(b.out.view(torch.int32), first.view(torch.int32))


def test_many_sequences(backend):
    r = random.Random(1)
    n = 1500
    check(backend, Batch([r.choice([0, 1, 1, 2]) for _ in range(n)], [r.randint(0, 60) for _ in range(n)], 4, 2, 64, page=16, seed=11))
    check(backend, Batch([r.choice([0, 1, 3, 9]) for _ in range(700)], [0] * 700, 4, 2, 64, seed=12))


@pytest.mark.parametrize("kv,hd,n,H", [(2000, 64, 9, 12), (140_000, 64, 9, 12), (7000, 128, 3, 40), (30_000, 128, 32, 4), (70_000, 192, 2, 20), (20_000, 256, 20, 6), (70_000, 16, 128, 1)])
def test_an_item_in_many_parts(backend, kv, hd, n, H):
    # one item, or two: its parts go up to as many as CTAs pay for, and past 32 for the longest caches
    check(backend, Batch([n], [kv], H, 1, hd, page=64, seed=hd + n), path=2)
    check(backend, Batch([n, 2], [kv, 300], H, 1, hd, page=64, seed=hd + n + 1), path=2)


@pytest.mark.parametrize("H,K", [(32, 1), (128, 1), (40, 2)])
def test_many_heads_to_a_kv_head(backend, H, K):
    check(backend, Batch([1, 3, 1], [300, 1000, 5], H, K, 64, page=16, seed=H))


def test_cache_past_32_bits(backend):
    """Pages whose values lie more than 2^32 bytes (and 2^31 values) into the cache."""
    import torch

    b = Batch([1, 40], [100, 70], 8, 2, 128, page=256, seed=13)
    per = 2 * 256 * 128
    far = (1 << 31) // per + 5
    n = far + b.n_pages
    small = b.k, b.v
    b.k, b.v = (torch.empty(n, 2, 256, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    for big, s in zip((b.k, b.v), small):
        big[far:] = s
    b.tables = [[far + i for i in t] for t in b.tables]
    b.table_t = torch.where(b.table_t >= 0, b.table_t + far, b.table_t)
    b.n_pages = n
    for path in (1, 2):
        check(backend, b, path=path)


def test_recorded_plan_follows_lengths_and_tables(backend):
    """A step recorded once and replayed while the sequences grow, in plans that share the context's workspace."""
    import torch

    be = backend
    b = Batch([1, 1, 1], [900, 1400, 40], 8, 2, 128, page=16, seed=14)
    c = Batch([60, 100], [500, 0], 8, 2, 128, page=16, seed=15)
    ops = [x.op(be) for x in (b, c)]
    for op in ops:
        be.attention(op)
    be.sync()
    plans = []
    for op in ops:
        be.graph_begin()
        be.attention(op)
        plans.append(be.graph_end())
    full = list(b.kv)
    for kv in (full, [901, 5, 41], [17, 1401, 1], [1, 1, 1]):
        b.kv = kv
        b.kv_t.copy_(torch.tensor(kv, dtype=torch.int32))
        want, tol = b.ref()
        want2, tol2 = c.ref()
        torch.cuda.synchronize()
        be.execute(plans[0])
        be.execute(plans[1])
        be.execute(plans[0])
        be.sync()
        assert float((b.out - want).abs().max()) <= tol and float((c.out - want2).abs().max()) <= tol2


def test_recorded_step_outlives_larger_calls(backend):
    """A decode step recorded by a fresh context, then a prompt of another kernel and size: the plan's workspace is still its own."""
    import torch

    from moe4all_b200 import BackendError, CudaBackend

    be = CudaBackend(0)
    b = Batch([1, 1], [3000, 5000], 8, 2, 128, page=16, seed=30)
    op = b.op(be)
    be.graph_begin()
    with pytest.raises(BackendError, match="un-recorded"):
        be.attention(op)
    be.graph_end()
    be.attention(op)
    be.sync()
    be.graph_begin()
    be.attention(op)
    plan = be.graph_end()
    c = Batch([700], [4000], 16, 2, 256, page=16, seed=31)
    check(be, c)
    keep = [torch.zeros(32 << 20, dtype=torch.uint8, device="cuda") for _ in range(4)]
    want, tol = b.ref()
    b.out.zero_()
    torch.cuda.synchronize()
    be.execute(plan)
    be.sync()
    assert float((b.out - want).abs().max()) <= tol
    assert not any(bool(x.any()) for x in keep)
    del plan, op
    be.close()


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
def test_scales_that_are_zero_negative_or_tiny(backend, path, scale):
    check(backend, Batch([1, 40, 200], [300, 20, 0], 8, 2, 64, page=16, seed=32), scale=scale, path=path)


def test_bound_that_is_too_small(backend):
    # max_q only picks the kernel: sequences longer than it says are served all the same
    check(backend, Batch([90, 1, 300], [10, 20, 0], 8, 2, 128, page=16, seed=33), max_q=1)
    check(backend, Batch([1, 1, 1], [10, 2000, 0], 8, 2, 128, page=16, seed=34), max_q=10 ** 6)


def test_on_the_callers_stream(backend):
    import torch

    be = backend
    s = torch.cuda.Stream()
    be.set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            b = Batch([1, 70], [333, 20], 8, 2, 128, page=16, seed=16)
            want, tol = b.ref()
            op = b.op(be)
            x = torch.randn(4096, 4096, device="cuda")
            for _ in range(5):
                x = x @ x * 1e-2  # the stream is busy when the call comes
            q = b.q.clone()
            b.q.zero_()
            b.q.copy_(q)
            be.attention(op)
            got = b.out.clone()
        s.synchronize()
        assert float((got - want).abs().max()) <= tol
    finally:
        be.sync()
        be.set_stream(None)


def test_bad_pages_and_lengths_are_reported(backend):
    from moe4all_b200 import BackendError

    import torch

    be = backend
    for path in (1, 2):
        for kind in ("page", "length", "rows"):
            b = Batch([1, 40], [100, 60], 8, 2, 64, page=16, seed=17)
            b.k.nan_to_num_()
            b.v.nan_to_num_()
            if kind == "page":
                b.table_t[1, 2] = b.n_pages
            elif kind == "length":
                b.kv_t[0] = 10 ** 6
            else:
                b.cu_t[2] = 1000
            torch.cuda.synchronize()
            be.attention(b.op(be, path=path))
            with pytest.raises(BackendError, match="attention kernel"):
                be.sync()
            b.table_t[1, 2] = b.tables[1][2]
            b.kv_t.copy_(torch.tensor(b.kv, dtype=torch.int32))
            b.cu_t.copy_(torch.tensor(b.cu, dtype=torch.int32))
            check(be, b, path=path)


def test_refusals(backend):
    from moe4all_b200 import BackendError, Unsupported

    be = backend
    b = Batch([1, 4], [20, 30], 8, 2, 64, page=16, seed=18)
    ok = b.op(be)
    be.attention(ok)
    be.sync()
    part = be.wrap(b.out.data_ptr(), 64)

    def refused(kind, **kw):
        with pytest.raises(kind) as e:
            be.attention(dataclasses.replace(ok, **kw))
        if kind is BackendError:
            assert not isinstance(e.value, Unsupported)

    for kw in (dict(n_head=9), dict(n_seq=0), dict(n_kv=0), dict(kv_len=None), dict(page_table=None), dict(page_table=None, kv_len=None), dict(page_size=0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(path=3), dict(q_stride=511), dict(q_stride=508), dict(q_stride=514), dict(out=part),
               dict(q=part), dict(k=part), dict(cu_q=part, n_seq=100), dict(out=ok.q), dict(n_pages=10 ** 6), dict(max_pages=10 ** 8), dict(window=1 << 31)):
        refused(BackendError, **kw)
    for kw in (dict(head_dim=72), dict(head_dim=272, n_head=1, n_kv=1), dict(page_size=24), dict(n_head=32, n_kv=1, head_dim=16, path=1), dict(n_seq=20000), dict(q_stride=(1 << 24) + 4)):
        refused(Unsupported, **kw)
    be.attention(dataclasses.replace(ok, rows=0))
    be.attention(ok)
    be.sync()


# ---- rope_kv ---------------------------------------------------------------------------------------


class Rope:
    def __init__(self, b, n_rot, interleaved, norm, factors, fused, seed=0, base=1e4, scale=1.0):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed + 100)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.b, self.n_rot, self.interleaved, self.fused, self.base, self.scale = b, n_rot, interleaved, fused, base, scale
        wide = (b.H + 2 * b.K) * b.hd
        self.qkv = r(b.rows, wide + (12 if fused else 0))
        self.parts = self.qkv[:, :wide].split([b.H * b.hd, b.K * b.hd, b.K * b.hd], 1)
        if not fused:
            self.parts = [x.contiguous() for x in self.parts]
        self.q_norm, self.k_norm = (1.0 + 0.2 * r(b.hd) if norm else None for _ in range(2))
        self.factors = 1.0 + r(n_rot // 2).abs() if factors else None
        self.q_out = torch.full((b.rows, b.H * b.hd), 7.5, device="cuda")

    def op(self, be, **kw):
        from moe4all_b200 import RopeKv

        b, w = self.b, lambda t: None if t is None else be.wrap_tensor(t)
        if self.fused:
            base, n = self.qkv.data_ptr(), self.qkv.numel()
            at = [0, b.H * b.hd, (b.H + b.K) * b.hd]
            q, k, v = (be.wrap(base + 4 * i, 4 * (n - i)) for i in at)
            st = dict.fromkeys(("q_stride", "k_stride", "v_stride"), self.qkv.shape[1])
        else:
            q, k, v = (w(x) for x in self.parts)
            st = {}
        f = dict(q=q, k=k, v=v, q_out=w(self.q_out), k_cache=w(b.k), v_cache=w(b.v), n_rot=self.n_rot, interleaved=self.interleaved, rope_base=self.base,
                 rope_scale=self.scale, q_norm=w(self.q_norm), k_norm=w(self.k_norm), norm_eps=1e-6, freq_factors=w(self.factors))
        return RopeKv(**{**f, **st, **b.fields(be), **kw})

    def ref(self):
        """q_out, k and v caches in 64 bits, and each value's pair magnitude."""
        import torch

        b = self.b
        out, kc, vc = self.q_out.double(), b.k.double(), b.v.double()
        mag = [torch.zeros_like(x) for x in (out, kc, vc)]
        half = self.n_rot // 2
        i = torch.arange(half, device="cuda")
        freq = float(self.base) ** (-2.0 * i.double() / max(1, self.n_rot)) * self.scale
        if self.factors is not None:
            freq = freq / self.factors.double()
        ia, ib = (2 * i, 2 * i + 1) if self.interleaved else (i, i + half)

        def rot(x, w, pos):
            if w is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
            y, m = x.clone(), x.abs().clone()
            ang = pos.double()[:, None, None] * freq
            y[..., ia] = x[..., ia] * ang.cos() - x[..., ib] * ang.sin()
            y[..., ib] = x[..., ia] * ang.sin() + x[..., ib] * ang.cos()
            m[..., ia] = m[..., ib] = x[..., ia].abs() + x[..., ib].abs()
            return y, m

        for s, n in enumerate(b.q_lens):
            skip = max(0, n - b.kv[s])
            rows = slice(b.cu[s] + skip, b.cu[s] + n)
            m = n - skip
            if m <= 0:
                continue
            pos = torch.arange(b.kv[s] - m, b.kv[s], device="cuda")
            q, k, v = (x[rows].double().view(m, -1, b.hd) for x in self.parts)
            (q, qm), (k, km) = rot(q, self.q_norm, pos), rot(k, self.k_norm, pos)
            out[rows], mag[0][rows] = q.reshape(m, -1), qm.reshape(m, -1)
            if b.page:
                at = tuple(x[b.kv[s] - m :] for x in b.at(s))
                kc[at[0], :, at[1]], vc[at[0], :, at[1]] = k, v
                mag[1][at[0], :, at[1]] = km
            else:
                kc[rows], vc[rows], mag[1][rows] = k, v, km
        return (out, kc, vc), mag


def rope_check(be, r, **kw):
    import torch

    want, mag = r.ref()
    torch.cuda.synchronize()
    op = r.op(be, **kw)
    be.rope_kv(op)
    be.sync()
    got_q = r.parts[0] if kw.get("q_out") is op.q else r.q_out
    for got, w, m, step in ((got_q, want[0], mag[0], 0.0), (r.b.k, want[1], mag[1], 2.0 ** -11), (r.b.v, want[2], mag[2], 2.0 ** -11)):
        got = got.double()
        same = (got == w) | (got.isnan() & w.isnan())
        off = torch.where(same, 0.0, (got - w).abs() - (2.0 ** -20 * m + step * w.abs() * (1 + 2 ** -9) + (2.0 ** -25 if step else 0.0)))
        assert not off.isnan().any() and float(off.max()) <= 0.0, float(off.max())


@pytest.mark.parametrize("H,K,hd,n_rot", [(8, 2, 64, 64), (32, 4, 128, 128), (16, 2, 256, 64), (16, 2, 256, 256), (3, 3, 80, 80), (14, 2, 96, 48), (4, 4, 16, 16), (4, 1, 112, 104), (2, 1, 192, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("page", [0, 16])
def test_rope_kv(backend, H, K, hd, n_rot, interleaved, page):
    b = Batch([1, 9, 0, 30], [0] * 4 if not page else [50, 0, 3, 1000], H, K, hd, page=page, lead=2, tail=3, seed=hd)
    rope_check(backend, Rope(b, n_rot, interleaved, norm=hd % 32 == 0, factors=hd == 128, fused=interleaved, seed=n_rot))


def test_rope_far_positions(backend):
    # frequencies near 1 at positions where f32 has no bits left for them
    b = Batch([1, 2], [1_000_000, 500_000], 2, 1, 128, page=1024, seed=20)
    rope_check(backend, Rope(b, 128, False, norm=False, factors=False, fused=False, base=1e6))
    rope_check(backend, Rope(b, 128, True, norm=False, factors=False, fused=False, base=1e4, scale=0.125))


def test_rope_in_place(backend):
    b = Batch([5, 40], [7, 100], 8, 2, 128, page=16, seed=21)
    r = Rope(b, 128, False, norm=True, factors=False, fused=False)
    want, mag = r.ref()
    q = backend.wrap_tensor(r.parts[0])
    backend.rope_kv(r.op(backend, q=q, q_out=q))
    backend.sync()
    assert float(((r.parts[0].double() - want[0]).abs() - 2.0 ** -20 * mag[0]).max()) <= 0


def test_rope_in_place_in_wide_rows(backend):
    from moe4all_b200 import BackendError

    b = Batch([5, 40], [7, 100], 8, 2, 128, page=16, seed=25)
    r = Rope(b, 128, True, norm=True, factors=False, fused=True)
    op = r.op(backend)
    op = dataclasses.replace(op, q_out=op.q, q_out_stride=op.q_stride)
    for kw in (dict(k=op.q), dict(v=op.q), dict(k_stride=op.k_stride - 12)):  # rows that the call would read and write
        with pytest.raises(BackendError, match="in place"):
            backend.rope_kv(dataclasses.replace(op, **kw))
    rest = r.qkv[:, 8 * 128 :].clone()
    want, mag = r.ref()
    backend.rope_kv(op)
    backend.sync()
    assert float(((r.parts[0].double() - want[0]).abs() - 2.0 ** -20 * mag[0]).max()) <= 0
    assert bool((r.qkv[:, 8 * 128 :] == rest).all())


def test_rope_negative_positions_and_bad_pages(backend):
    from moe4all_b200 import BackendError

    import torch

    b = Batch([5, 3], [-2, -3], 8, 2, 128, page=16, seed=22)
    r = Rope(b, 128, False, norm=False, factors=False, fused=False)
    rope_check(backend, r)
    assert bool((r.q_out[:2] == 7.5).all()) and bool((r.q_out[5:] == 7.5).all())
    b = Batch([5, 20], [30, 0], 8, 2, 128, page=16, seed=23)
    r = Rope(b, 128, False, norm=False, factors=False, fused=False)
    k = b.k.clone()
    b.table_t[1, 1] = -5
    torch.cuda.synchronize()
    backend.rope_kv(r.op(backend))
    with pytest.raises(BackendError, match="attention kernel"):
        backend.sync()
    lost = b.tables[1][1]
    assert torch.equal(b.k[lost].view(torch.int16), k[lost].view(torch.int16))  # the row whose page is not there wrote nowhere


def test_rope_refusals(backend):
    from moe4all_b200 import BackendError, Unsupported

    be = backend
    b = Batch([1, 4], [20, 30], 8, 2, 64, page=16, seed=24)
    r = Rope(b, 64, False, norm=True, factors=True, fused=False)
    ok = r.op(be)
    be.rope_kv(ok)
    be.sync()
    part = be.wrap(r.q_out.data_ptr(), 64)
    for kw in (dict(n_rot=60), dict(n_rot=72), dict(rope_base=0.0), dict(rope_base=-1.0), dict(rope_base=float("inf")), dict(rope_scale=NAN), dict(norm_eps=-1.0),
               dict(q_norm=part), dict(freq_factors=part), dict(q_stride=516 - 2), dict(k_stride=64), dict(q_out=part), dict(v=part), dict(v_cache=ok.k_cache),
               dict(q_out=ok.q, q_out_stride=516), dict(q_out=ok.k_cache), dict(k=ok.k_cache), dict(n_head=7), dict(kv_len=None)):
        with pytest.raises(BackendError) as e:
            be.rope_kv(dataclasses.replace(ok, **kw))
        assert not isinstance(e.value, Unsupported), kw
    with pytest.raises(Unsupported):
        be.rope_kv(dataclasses.replace(ok, head_dim=56, n_rot=56))
    be.rope_kv(dataclasses.replace(ok, rows=0))
    be.sync()


def test_rope_then_attention_step_by_step(backend):
    """A sequence written and read token by token through pages gives what the whole prompt gives packed."""
    import torch

    from moe4all_b200 import Attention, RopeKv

    be, n, H, K, hd, page = backend, 75, 8, 2, 128, 16
    whole = Batch([n], [0], H, K, hd, seed=25)
    r = Rope(whole, hd, False, norm=True, factors=False, fused=False, base=1e6)
    be.rope_kv(r.op(be))
    w = be.wrap_tensor
    full = torch.zeros(n, H * hd, device="cuda")
    be.attention(Attention(q=w(r.q_out), k=w(whole.k), v=w(whole.v), out=w(full), scale=hd ** -0.5, **whole.fields(be)))
    be.sync()
    paged = Batch([n], [0], H, K, hd, page=page, seed=26)
    paged.k.fill_(NAN), paged.v.fill_(NAN)
    out = torch.zeros(n, H * hd, device="cuda")
    at, steps = 0, [30, 1, 1, 1, 5, 1, 36]
    for m in steps:
        q, k, v = (x[at : at + m].contiguous() for x in r.parts)
        qo, o = torch.empty_like(q), torch.empty(m, H * hd, device="cuda")
        cu, kv = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, m], [at + m]))
        batch = dict(cu_q=w(cu), kv_len=w(kv), page_table=w(paged.table_t), rows=m, n_seq=1, n_head=H, n_kv=K, head_dim=hd, n_pages=paged.n_pages, page_size=page, max_pages=paged.width)
        torch.cuda.synchronize()
        be.rope_kv(RopeKv(q=w(q), k=w(k), v=w(v), q_out=w(qo), k_cache=w(paged.k), v_cache=w(paged.v), n_rot=hd, rope_base=1e6, q_norm=w(r.q_norm), k_norm=w(r.k_norm), **batch))
        be.attention(Attention(q=w(qo), k=w(paged.k), v=w(paged.v), out=w(o), scale=hd ** -0.5, max_q=m, **batch))
        be.sync()
        out[at : at + m] = o
        at += m
    assert torch.equal(paged.get(paged.k, 0), whole.get(whole.k, 0)) and torch.equal(paged.get(paged.v, 0), whole.get(whole.v, 0))
    # the same numbers by other orders of summation: twice the bound of one
    whole.q.copy_(r.q_out)
    want, tol = whole.ref()
    assert float((full - want).abs().max()) <= tol and float((out - want).abs().max()) <= tol
