"""GPU: pages of 8 bits through the C ABI - rows into them, out of them, attention over them - against the formulas in 64 bits.

Attention's tolerance is that of f16 pages (test_gpu_attention.py): the values that codes stand for are f16 numbers, and it is these that the 64-bit
reference reads.  A row on its way into the cache: 2^-20 of a pair's magnitude for the rotation, and half a step d of its 16 values, where d is the scale that
64 bits give, or the next one where the largest magnitude is that near to a border (2^-19 of it)."""
import dataclasses

import numpy as np
import pytest

from test_gpu_attention import HEADS, NAN, Batch, Rope, check

pytestmark = pytest.mark.gpu


def scale_value(s):
    """What a scale byte stands for, in 64 bits: 0xC0 and above are no numbers."""
    s = np.asarray(s).astype(np.int64)
    e, m = s >> 3, (s & 7).astype(np.float64)
    return np.where(s >= 0xC0, np.nan, np.where(e > 0, (8 + m) * 2.0 ** (e - 18.0), m * 2.0 ** -17))


SCALES = scale_value(np.arange(0xC0))


def least_scale(a):
    """The byte of the least scale of which 127 reach a; 0xFF where none does."""
    i = np.searchsorted(SCALES * 127.0, a, side="left")
    return np.where((i < 0xC0) & np.isfinite(a), i, 0xFF)


def values(codes, scales):
    """[.., hd] codes and [.., hd / 16] scale bytes (tensors on the GPU) as the numbers that they are, f64."""
    import torch

    d = torch.tensor(scale_value(np.arange(256)), device="cuda")[scales.long()]
    return (codes.double() - 128) * d.repeat_interleave(16, -1)


class Q8Batch(Batch):
    """A batch over pages of 8 bits.  `k` and `v` hold the values, for the reference; what no row may see is bytes that are no numbers."""

    def __init__(self, *args, **kw):
        import torch

        super().__init__(*args, **kw)
        assert self.page
        g = torch.Generator(device="cuda").manual_seed(kw.get("seed", 0) + 1000)
        self.codes, self.scales = {}, {}
        for name in "kv":
            x = getattr(self, name)
            c = torch.randint(0, 256, x.shape, generator=g, device="cuda", dtype=torch.uint8)
            s = torch.randint(0xC0, 256, (*x.shape[:3], self.hd // 16), generator=g, device="cuda", dtype=torch.uint8)
            own = ~x[..., ::16].isnan()
            # magnitudes from 2^-10 to 1 side by side
            s[own] = torch.randint(0x10, 0x60, (int(own.sum()),), generator=g, device="cuda", dtype=torch.uint8)
            self.codes[name], self.scales[name] = c, s
        self.take()

    def take(self):
        """The reference's values from the codes."""
        for name in "kv":
            setattr(self, name, values(self.codes[name], self.scales[name]).half())

    def q8_fields(self, be, **names):
        w = be.wrap_tensor
        return {names.get("k", "k"): w(self.codes["k"]), names.get("v", "v"): w(self.codes["v"]), "k_scale": w(self.scales["k"]), "v_scale": w(self.scales["v"])}

    def op(self, be, **kw):
        return super().op(be, **{**self.q8_fields(be), **kw})


def test_values_are_f16_numbers():
    import torch

    c = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(0xC0, 1)
    s = torch.arange(0xC0, device="cuda", dtype=torch.uint8)[:, None].repeat(1, 16)
    x = values(c, s)
    x[c == 0] = 0  # (the code that rope_kv never writes: -128 x 480 is one too, but 61440)
    assert torch.equal(x.half().double(), x)


@pytest.mark.parametrize("H,K,hd", HEADS)
@pytest.mark.parametrize("path", [1, 2])
def test_single_tokens(backend, H, K, hd, path):
    check(backend, Q8Batch([1, 1, 1, 1, 1], [0, 1, 130, 700, 2047], H, K, hd, page=16, seed=hd), path=path)


@pytest.mark.parametrize("page", [16, 48, 64, 128, 256, 1024])
@pytest.mark.parametrize("path", [1, 2])
def test_page_sizes(backend, page, path):
    check(backend, Q8Batch([1, 3, 5], [500, 63, 1200], 8, 2, 128, page=page, seed=page, spare=5), path=path)


@pytest.mark.parametrize("H,K,hd", HEADS)
@pytest.mark.parametrize("path", [1, 2])
def test_chunks(backend, H, K, hd, path):
    check(backend, Q8Batch([33, 1, 130, 5, 64], [100, 900, 257, 0, 127], H, K, hd, page=32, seed=hd + 2), path=path)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 500, 5000])
@pytest.mark.parametrize("path", [1, 2])
def test_windows(backend, window, path):
    check(backend, Q8Batch([1, 40, 200, 1], [1000, 300, 0, 3], 8, 2, 128, page=64, seed=window), window=window, path=path)


@pytest.mark.parametrize("path", [1, 2])
def test_rows_of_no_sequence_stay_and_rows_that_see_nothing(backend, path):
    b = Q8Batch([0, 4, 0, 1, 0], [9, 20, 0, 33, 50], 8, 2, 64, page=16, lead=3, tail=5, q_pad=12, out_pad=8, seed=3)
    check(backend, b, path=path)
    assert bool((b.out[:3] == 7.5).all()) and bool((b.out[-5:] == 7.5).all()) and bool((b.out[:, 512:] == 7.5).all())
    b = Q8Batch([5, 3, 200], [-2, -3, -150], 8, 2, 128, page=16, seed=4)
    check(backend, b, path=path)
    assert bool((b.out[:2] == 0).all()) and bool((b.out[5:8] == 0).all()) and bool((b.out[8:158] == 0).all()) and bool((b.out[158:] != 0).any())


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("H,K,hd", [(8, 2, 64), (8, 1, 128), (3, 3, 80), (16, 2, 256)])
@pytest.mark.parametrize("window", [0, 30])
def test_what_is_no_number_reaches_the_rows_that_see_it(backend, path, H, K, hd, window):
    # values of 16 columns of a late token, a key of another: rows before them, and rows whose window has left them behind, stay clean
    b = Q8Batch([4, 60, 1], [700, 40, 5000], H, K, hd, page=16, seed=hd + window)
    for s, token, name in ((0, 702, "v"), (0, 100, "v"), (1, 70, "v"), (1, 95, "k"), (2, 4990, "v"), (2, 17, "v")):
        page, at = b.tables[s][token // 16], token % 16
        b.scales[name][page, K - 1, at, (hd // 16) // 2 if name == "v" else 0] = 0xC0 + token % 64
    b.take()
    want = check(backend, b, window=window, path=path)
    assert bool(want[:, : H * hd].isnan().any()) and bool(want[0, : H * hd].isfinite().any())


@pytest.mark.parametrize("kv,hd,n,H", [(40000, 128, 1, 8), (20000, 64, 3, 4), (9000, 256, 2, 4), (12000, 192, 40, 2)])
def test_an_item_in_many_parts(backend, kv, hd, n, H):
    check(backend, Q8Batch([n], [kv], H, 1, hd, page=64, seed=kv))


def test_many_sequences(backend):
    import random

    r = random.Random(5)
    check(backend, Q8Batch([r.choice([0, 1, 1, 2]) for _ in range(700)], [r.randrange(0, 90) for _ in range(700)], 4, 1, 64, page=16, seed=40), max_q=2)


@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_tiles_give_what_they_give_over_f16_pages(backend, hd):
    """The same kernel over the same values: the same bits.  As many pages as the cache has, and fewer places than that."""
    import torch

    for spare in (2, 400):
        b = Q8Batch([70, 129], [300, 17], 8, 2, hd, page=16, seed=hd, spare=spare)
        backend.attention(b.op(backend, path=2))
        backend.sync()
        got = b.out.clone()
        f16 = Batch.op(b, backend, path=2, k=backend.wrap_tensor(b.k), v=backend.wrap_tensor(b.v))
        torch.cuda.synchronize()
        backend.attention(f16)
        backend.sync()
        assert torch.equal(got, b.out)


def test_recorded_plans_outlive_larger_calls():
    """A chunk and a step recorded by a fresh context, then a chunk over more pages: the plans' f16 pages are still their own."""
    import torch

    from moe4all_b200 import BackendError, CudaBackend

    be = CudaBackend(0)
    b, c = Q8Batch([1, 1], [3000, 5000], 8, 2, 128, page=16, seed=30), Q8Batch([60, 100], [500, 0], 8, 2, 128, page=16, seed=31)
    ops = [x.op(be) for x in (b, c)]
    be.attention(ops[0])
    be.sync()
    be.graph_begin()
    with pytest.raises(BackendError, match="un-recorded"):
        be.attention(ops[1])
    be.graph_end()
    plans = []
    for op in ops:
        be.attention(op)
        be.sync()
        be.graph_begin()
        be.attention(op)
        plans.append(be.graph_end())
    for seed, past in ((32, 9000), (33, 30000)):
        check(be, Q8Batch([300], [past], 8, 2, 128, page=16, seed=seed))
        keep = [torch.full((8 << 20,), 5, dtype=torch.uint8, device="cuda") for _ in range(4)]
        for x, plan in zip((b, c), plans):
            want, tol = x.ref()
            x.out.fill_(7.5)
            torch.cuda.synchronize()
            be.execute(plan)
            be.sync()
            assert float((x.out - want).abs().max()) <= tol
        assert all(bool((x == 5).all()) for x in keep)
    b.kv = [17, 1]
    b.kv_t.copy_(torch.tensor(b.kv, dtype=torch.int32))
    want, tol = b.ref()
    torch.cuda.synchronize()
    be.execute(plans[0])
    be.sync()
    assert float((b.out - want).abs().max()) <= tol
    del plans, ops, op, plan
    be.close()


def test_same_bits_every_time_and_on_another_stream(backend):
    import torch

    b = Q8Batch([1, 5, 200], [9000, 700, 300], 8, 2, 128, page=64, seed=12)
    for path in (1, 2):
        seen = []
        op = b.op(backend, path=path)
        for i in range(4):
            if i == 2:
                stream = torch.cuda.Stream()
                backend.set_stream(stream.cuda_stream)
            b.out.fill_(7.5)
            torch.cuda.synchronize()
            backend.attention(op)
            backend.sync()
            seen.append(b.out.clone())
        backend.set_stream(None)
        assert all(torch.equal(seen[0], x) for x in seen)


def test_cache_past_32_bits(backend):
    """Codes from 4 GB on, scales beside them."""
    import torch

    K, hd, page = 8, 128, 64
    n_pages = (1 << 32) // (K * hd * page) + 40
    b = Q8Batch([1, 30], [500, 300], 8, K, hd, page=page, seed=6)
    big = {n: torch.zeros(n_pages, K, page, hd, dtype=torch.uint8, device="cuda") for n in "kv"}
    scales = {n: torch.full((n_pages, K, page, hd // 16), 0xFF, dtype=torch.uint8, device="cuda") for n in "kv"}
    at = n_pages - b.n_pages
    for n in "kv":
        big[n][at:], scales[n][at:] = b.codes[n], b.scales[n]
    b.table_t = torch.where(b.table_t >= 0, b.table_t + at, b.table_t)
    w = backend.wrap_tensor
    for path in (1, 2):
        check(backend, b, path=path, k=w(big["k"]), v=w(big["v"]), k_scale=w(scales["k"]), v_scale=w(scales["v"]), n_pages=n_pages, page_table=w(b.table_t))


def test_bad_pages_and_lengths_are_reported(backend):
    import torch

    from moe4all_b200 import BackendError

    for path in (1, 2):
        for kind in ("page", "length", "rows"):
            b = Q8Batch([1, 40], [100, 60], 8, 2, 64, page=16, seed=17)
            if kind == "page":
                b.table_t[1, 2] = b.n_pages
            elif kind == "length":
                b.kv_t[0] = 10 ** 6
            else:
                b.cu_t[2] = 1000
            torch.cuda.synchronize()
            backend.attention(b.op(backend, path=path))
            with pytest.raises(BackendError, match="attention kernel"):
                backend.sync()


# ---- rows into the cache, and out of it

def read_op(be, b, f16=True, pad=0, q8=True, **kw):
    import torch

    from moe4all_b200 import KvRead

    w = be.wrap_tensor
    n = b.K * b.hd + pad
    out = [torch.full((b.rows, n), 7.5, device="cuda", dtype=torch.float16 if f16 else torch.float32) for _ in range(2)]
    f = {k: v for k, v in b.fields(be).items() if k != "n_head"}
    cache = b.q8_fields(be, k="k_cache", v="v_cache") if q8 else dict(k_cache=w(b.k), v_cache=w(b.v))
    return KvRead(**{**cache, **f, "k": w(out[0]), "v": w(out[1]), "f16": f16, "k_stride": n if pad else 0, "v_stride": n if pad else 0, **kw}), out


def read_want(b, name):
    """[rows, K * hd] f64, 7.5 where nothing is written."""
    import torch

    want = torch.full((b.rows, b.K * b.hd), 7.5, device="cuda", dtype=torch.float64)
    for s, n in enumerate(b.q_lens):
        m = min(n, b.kv[s])
        want[b.cu[s] : b.cu[s] + n - m] = 0
        if m:
            want[b.cu[s] + n - m : b.cu[s] + n] = b.get(getattr(b, name), s)[b.kv[s] - m :].double().reshape(m, -1)
    return want


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("H,K,hd,page", [(8, 2, 64, 16), (8, 1, 128, 64), (3, 3, 80, 48), (16, 2, 256, 32), (4, 4, 16, 16), (2, 1, 240, 128)])
def test_read(backend, H, K, hd, page, f16, q8):
    import torch

    b = Q8Batch([0, 1, 300, 7, 0, 40], [5, 0, 100, 33, 0, -11], H, K, hd, page=page, lead=2, tail=3, seed=hd)
    b.scales["k"][b.tables[3][0], 0, 3] = 0xFF  # (read by nobody: 33 tokens are behind)
    b.scales["v"][b.tables[2][390 // page], K - 1, 390 % page, hd // 16 - 1] = 0xC5
    b.take()
    for pad in (0, 8):
        op, out = read_op(backend, b, f16, pad, q8)
        torch.cuda.synchronize()
        backend.kv_read(op)
        backend.sync()
        for got, name in zip(out, "kv"):
            want = read_want(b, name)
            assert torch.equal(got[:, : K * hd].double().nan_to_num(nan=1e6), want.nan_to_num(nan=1e6)) and bool((got[:, K * hd :] == 7.5).all())
        assert bool(out[1].isnan().any()) and not bool(out[0].isnan().any())


def test_read_many_sequences(backend):
    import random

    import torch

    r = random.Random(9)
    n = 2000
    b = Q8Batch([r.choice([0, 1, 3, 30]) for _ in range(n)], [r.randrange(0, 20) for _ in range(n)], 2, 1, 64, page=16, seed=41)
    op, out = read_op(backend, b)
    torch.cuda.synchronize()
    backend.kv_read(op)
    backend.sync()
    assert torch.equal(out[0].double(), read_want(b, "k")) and torch.equal(out[1].double(), read_want(b, "v"))


class Q8Rope(Rope):
    def __init__(self, b, n_rot, interleaved, norm=False, factors=False, fused=False, seed=0):
        super().__init__(b, n_rot, interleaved, norm, factors, fused, seed=seed)

    def op(self, be, **kw):
        b = self.b
        return super().op(be, **{**b.q8_fields(be, k="k_cache", v="v_cache"), **kw})


def written(b, name, rows):
    """Codes and scales of the rows' tokens, by sequence: [(first row, codes [n, K, hd], scales [n, K, hd / 16])]."""
    out = []
    for s, n in enumerate(b.q_lens):
        m = min(n, b.kv[s])
        if m:
            at = tuple(x[b.kv[s] - m :] for x in b.at(s))
            out.append((at, b.codes[name][at[0], :, at[1]], b.scales[name][at[0], :, at[1]]))
    return out


def write_check(be, r, exact_v=True, **kw):
    import torch

    b = r.b
    (want_q, want_k, want_v), mag = r.ref()
    before = {n: (b.codes[n].clone(), b.scales[n].clone()) for n in "kv"}
    torch.cuda.synchronize()
    be.rope_kv(r.op(be, **kw))
    be.sync()
    off = (r.q_out.double() - want_q).abs()
    assert bool(((off <= 2.0 ** -20 * mag[0]) | (r.q_out.double() == want_q)).all())
    for name, want, slop in (("k", want_k, mag[1]), ("v", want_v, torch.zeros_like(want_v))):
        touched = torch.zeros(b.codes[name].shape[:3], dtype=torch.bool, device="cuda")
        for at, codes, scales in written(b, name, b.rows):
            touched[at[0], :, at[1]] = True
            x, err = want[at[0], :, at[1]], 2.0 ** -20 * slop[at[0], :, at[1]]
            blocks, e16 = x.unflatten(-1, (-1, 16)), err.unflatten(-1, (-1, 16)).amax(-1)
            big = blocks.abs().amax(-1)
            lo, hi = (torch.tensor(least_scale((big + f * (e16 + big * 2.0 ** -22)).clamp(min=0).cpu().numpy()), device="cuda") for f in (-1, 1))
            ok = (scales.long() >= lo) & (scales.long() <= hi)
            assert bool(ok.all()), f"{name}: {int((~ok).sum())} scales"
            d = torch.tensor(scale_value(np.arange(256)), device="cuda")[scales.long()].repeat_interleave(16, -1)
            got = values(codes, scales)
            fine = ~d.isnan()
            # (the code comes from a product with a rounded 1 / d: 127 x 2^-23 of a step)
            assert bool((((got - x).abs() <= d * (0.5 + 2.0 ** -15) + err) | ~fine).all())
            assert bool((codes[fine] >= 1).all())
            if name == "v" and exact_v:
                assert torch.equal(scales.long(), torch.tensor(least_scale(big.cpu().numpy()), device="cuda"))
        # nothing but the rows' tokens was written
        assert torch.equal(b.codes[name][~touched], before[name][0][~touched]) and torch.equal(b.scales[name][~touched], before[name][1][~touched])


@pytest.mark.parametrize("H,K,hd,n_rot", [(8, 2, 64, 64), (32, 4, 128, 128), (16, 2, 256, 64), (16, 2, 256, 256), (3, 3, 80, 80), (3, 3, 80, 24), (14, 2, 96, 48), (4, 4, 16, 16), (4, 1, 112, 104), (2, 1, 192, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_write(backend, H, K, hd, n_rot, interleaved):
    b = Q8Batch([1, 17, 0, 5, 70, 3], [40, 0, 9, 100, 3, -1], H, K, hd, page=16, lead=2, tail=1, seed=hd)
    write_check(backend, Q8Rope(b, n_rot, interleaved, norm=True, seed=n_rot))
    write_check(backend, Q8Rope(b, n_rot, interleaved, factors=n_rot > 0, fused=True, seed=n_rot + 1))


def test_write_of_values_of_any_size(backend):
    """Rows from 0 and f32's least numbers to past the range, borders of a scale among them, and what is no number."""
    import torch

    b = Q8Batch([64], [3], 2, 2, 64, page=16, seed=50)
    r = Q8Rope(b, 0, False, seed=3)
    big = torch.tensor([0.0, 1e-45, 1e-38, 2.0 ** -17 * 127, 2.0 ** -17 * 127.5, 2.0 ** -14 * 127, 2.0 ** -14 * 126.9, 127.0, 127.00001, 128.0, 0.875 * 127, 60960.0, 60959.9, 60961.0, 65504.0,
                        1e38, float("inf"), -float("inf"), NAN], device="cuda")
    v = r.parts[2].view(64, 2, 4, 16)
    v.uniform_(-1, 1)
    each = big[torch.arange(64, device="cuda") % len(big)]
    v[..., 5] = torch.where(torch.arange(64, device="cuda")[:, None, None] % 2 == 0, 1.0, -1.0) * each[:, None, None]
    v[..., :5] = v[..., :5].mul(each[:, None, None, None].nan_to_num(0, 0, 0)).clamp(-3e38, 3e38)
    v[..., 6:] = v[..., 6:].mul(each[:, None, None, None].nan_to_num(0, 0, 0)).clamp(-3e38, 3e38)
    (_, _, want), _ = r.ref()
    torch.cuda.synchronize()
    backend.rope_kv(r.op(backend))
    backend.sync()
    (at, codes, scales), = written(b, "v", 64)
    x = want[at[0], :, at[1]].unflatten(-1, (-1, 16))
    a = x.abs().amax(-1)
    odd = ~(a <= 60960)
    assert bool((scales[odd] == 0xFF).all()) and bool((codes.unflatten(-1, (-1, 16))[odd] == 128).all())
    near = (a * (1 - 2.0 ** -23)).cpu().numpy()
    lo, hi = (torch.tensor(least_scale(y), device="cuda") for y in (near, a.cpu().numpy()))
    assert bool(((scales.long() >= lo) & (scales.long() <= hi) | odd).all())
    d = torch.tensor(scale_value(np.arange(256)), device="cuda")[scales.long()][..., None]
    off = (values(codes, scales).unflatten(-1, (-1, 16)) - x).abs()
    assert bool(((off <= d * (0.5 + 2.0 ** -15)) | odd[..., None]).all())


def test_write_negative_positions_and_bad_pages(backend):
    import torch

    from moe4all_b200 import BackendError

    b = Q8Batch([6, 40], [-2, 30], 4, 2, 64, page=16, seed=51)
    r = Q8Rope(b, 64, False, seed=4)
    write_check(backend, r)
    page = b.tables[1][3]
    before = b.codes["k"].clone()
    b.table_t[1, 3] = -7
    torch.cuda.synchronize()
    backend.rope_kv(r.op(backend))
    with pytest.raises(BackendError, match="attention kernel"):
        backend.sync()
    assert torch.equal(b.codes["k"][page], before[page])
    op, _ = read_op(backend, b)
    backend.kv_read(op)
    with pytest.raises(BackendError, match="attention kernel"):
        backend.sync()


def test_write_then_attention_step_by_step(backend):
    """A prompt in chunks and then single tokens, through one cache: each step's attention is that over the values that are in it then."""
    import torch

    H, K, hd, page = 8, 2, 64, 16
    b = Q8Batch([90, 60], [0, 0], H, K, hd, page=page, seed=60)
    final = list(b.kv)
    for n in "kv":
        b.scales[n].fill_(0xEE)
    done = [0, 0]
    for step in ([50, 20], [30, 30], [1, 1], [1, 1], [8, 8]):
        done = [a + c for a, c in zip(done, step)]
        assert all(a <= f for a, f in zip(done, final))
        s = object.__new__(Q8Batch)
        s.__dict__.update(b.__dict__)
        s.q_lens, s.pasts, s.kv = step, [a - c for a, c in zip(done, step)], list(done)
        s.cu = [0, step[0], step[0] + step[1]]
        s.rows = s.cu[-1]
        s.q, s.out = torch.randn(s.rows, H * hd, device="cuda"), torch.full((s.rows, H * hd), 7.5, device="cuda")
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        s.cu_t, s.kv_t = i32(s.cu), i32(s.kv)
        r = Q8Rope(s, hd, False, seed=done[0])
        r.q_out = s.q
        torch.cuda.synchronize()
        backend.rope_kv(r.op(backend))
        backend.sync()
        s.take()
        check(backend, s)


def test_recorded_step_writes_reads_and_attends(backend):
    import torch

    b = Q8Batch([1, 1, 1], [40, 300, 7], 8, 2, 128, page=16, seed=70)
    r = Q8Rope(b, 128, False, norm=True, seed=5)
    r.q_out = b.q
    read, out = read_op(backend, b)
    ops = r.op(backend), b.op(backend), read

    def step():
        backend.rope_kv(ops[0])
        backend.attention(ops[1])
        backend.kv_read(ops[2])

    step()
    backend.sync()
    backend.graph_begin()
    step()
    plan = backend.graph_end()
    for kv in ([41, 301, 8], [30, 2, 1]):
        b.kv = kv
        b.kv_t.copy_(torch.tensor(kv, dtype=torch.int32))
        b.out.fill_(7.5)
        torch.cuda.synchronize()
        backend.execute(plan)
        backend.sync()
        b.take()
        want, tol = b.ref()
        assert float((b.out - want).abs().max()) <= tol
        assert torch.equal(out[0].double(), read_want(b, "k")) and torch.equal(out[1].double(), read_want(b, "v"))


def test_refusals(backend):
    from moe4all_b200 import BackendError, KvRead, RopeKv, Unsupported

    be = backend
    b = Q8Batch([1, 4], [20, 30], 8, 2, 64, page=16, seed=18)
    r = Q8Rope(b, 64, False, seed=2)
    rope, att, (read, out) = r.op(be), b.op(be), read_op(be, b, f16=False)
    small = be.wrap(b.out.data_ptr(), 4)
    inside = lambda t, n: be.wrap(t.data_ptr(), n)

    def refused(call, op, kind, **kw):
        with pytest.raises(kind) as e:
            call(dataclasses.replace(op, **kw))
        if kind is BackendError:
            assert not isinstance(e.value, Unsupported)

    for call, op in ((be.rope_kv, rope), (be.attention, att), (be.kv_read, read)):
        for n in ("k_scale", "v_scale", "cu_q", "kv_len", "page_table"):
            refused(call, op, BackendError, **{n: small})
        refused(call, op, Unsupported, page_size=8)
        refused(call, op, Unsupported, head_dim=24)
        refused(call, op, BackendError, n_pages=1 << 29)
        refused(call, op, BackendError, kv_len=None)
        if call != be.kv_read:
            with pytest.raises(ValueError):
                dataclasses.replace(op, v_scale=None)
        else:
            refused(call, op, BackendError, v_scale=None)
    refused(be.rope_kv, rope, Unsupported, kv_len=None, page_table=None, n_pages=0, page_size=0, max_pages=0)
    refused(be.attention, att, Unsupported, kv_len=None, page_table=None, n_pages=0, page_size=0, max_pages=0)
    refused(be.kv_read, read, Unsupported, kv_len=None, page_table=None, n_pages=0, page_size=0, max_pages=0)
    refused(be.kv_read, dataclasses.replace(read, k_scale=None, v_scale=None, k_cache=be.wrap_tensor(b.k), v_cache=be.wrap_tensor(b.v)), BackendError, kv_len=None, page_table=None,
            n_pages=0, page_size=0, max_pages=0)
    # parts of the cache over each other, over rows
    refused(be.rope_kv, rope, BackendError, k_scale=rope.v_scale)
    refused(be.rope_kv, rope, BackendError, k_scale=rope.k_cache)
    refused(be.rope_kv, rope, BackendError, k_scale=inside(r.q_out, b.scales["k"].numel()))
    refused(be.attention, att, BackendError, k_scale=inside(b.out, b.scales["k"].numel()))
    refused(be.kv_read, read, BackendError, k=read.v)
    refused(be.kv_read, read, BackendError, k=small)
    refused(be.kv_read, read, BackendError, k_stride=100)
    refused(be.kv_read, read, BackendError, k_stride=130)
    refused(be.kv_read, read, BackendError, v=inside(b.codes["k"], out[0].numel() * 4))
    refused(be.kv_read, read, Unsupported, k_stride=1 << 25)
    assert be._lib.infr_cuda_kv_read(be._ctx, None) == -1 and be._lib.infr_cuda_rope_kv_q8(be._ctx, rope._desc, None, None) == -1
    assert be._lib.infr_cuda_attention_q8(be._ctx, None, rope.k_scale.handle, rope.v_scale.handle) == -1
    # and the calls as they were go through; a call without rows does nothing
    for call, op in ((be.rope_kv, rope), (be.attention, att), (be.kv_read, read)):
        call(op)
        call(dataclasses.replace(op, rows=0))
    be.sync()


@pytest.mark.parametrize("H,K,hd", [(9, 1, 144), (16, 1, 256), (32, 2, 192), (17, 1, 64)])
def test_more_heads_than_the_few_rows_kernel_takes(backend, H, K, hd):
    """The choice by itself goes to the tiles; the few-rows kernel asked for by name is refused."""
    from moe4all_b200 import Unsupported

    b = Q8Batch([1, 3, 1], [70, 0, 400], H, K, hd, page=16, seed=H)
    check(backend, b)
    with pytest.raises(Unsupported):
        backend.attention(b.op(backend, path=1))


@pytest.mark.parametrize("n,K,rows", [(2, 4, 64), (2, 4, 65), (4, 4, 48), (4, 4, 49), (9, 4, 32), (9, 4, 33)])
def test_both_sides_of_the_choice(backend, n, K, rows):
    check(backend, Q8Batch([rows] + [1] * (n - 1), [100 + i for i in range(n)], 2 * K, K, 64, page=32, seed=rows))


def test_two_contexts_side_by_side(backend):
    """Two contexts over one cache, calls of both under way at once: each has f16 pages and partial sums of its own."""
    import torch

    from moe4all_b200 import CudaBackend

    b = Q8Batch([70, 1, 90], [300, 2000, 0], 8, 2, 128, page=64, seed=90)
    want, tol = b.ref()
    other = CudaBackend(0)
    try:
        outs = [torch.full_like(b.out, 7.5) for _ in range(2)]
        ops = [[b.op(be, out=be.wrap_tensor(o), path=path) for path in (2, 1)] for be, o in zip((backend, other), outs)]
        torch.cuda.synchronize()
        for path in range(2):
            for _ in range(5):
                for be, op in zip((backend, other), ops):
                    be.attention(op[path])
            backend.sync(), other.sync()
            for o in outs:
                assert float((o - want).abs().max()) <= tol
                o.fill_(7.5)
            torch.cuda.synchronize()
    finally:
        other.close()


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("size", [3.0e38, 1.0e-38, 1.0e-44])
def test_rows_of_any_size(backend, path, size):
    """q near both ends of f32, and a scale that brings the scores back (both powers of two but for rounding of the rows themselves)."""
    import torch

    b = Q8Batch([1, 2], [60, 200], 4, 2, 64, page=16, seed=95)
    q = b.q.clone()
    s = 2.0 ** np.floor(np.log2(size / float(q.abs().max())))
    scale = float(np.clip(64 ** -0.5 / s, 2e-38, 1e37))
    b.q.copy_((q.double() * s).float())
    torch.cuda.synchronize()
    got = b.out.clone()
    op = b.op(backend, path=path, scale=scale, out=backend.wrap_tensor(got))
    backend.attention(op)
    backend.sync()
    # the plain scale over rows that are the same numbers (those that f32 rounded near its lower end among them)
    b.q.copy_((b.q.double() * (scale / 64 ** -0.5)).float())
    want, tol = b.ref()
    assert bool(got.isfinite().all()) and float((got - want).abs().max()) <= tol
