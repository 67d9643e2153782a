"""GPU: rope_kv and attention at the ends of what their arguments may be, against the formulas in 64 bits (tolerances as in
test_gpu_attention.py unless a test derives its own)."""
import dataclasses
import math

import pytest

from test_gpu_attention import NAN, Batch, Rope, check

pytestmark = pytest.mark.gpu


def test_caches_past_64_bits_are_refused(backend):
    # pages x tokens x heads x values x 2 bytes are 2^69, 2^65 and 2^68: nothing in 64 bits
    from moe4all_b200 import BackendError

    b = Batch([1], [20], 16, 16, 16, page=16, seed=1)
    r = Rope(b, 16, False, norm=False, factors=False, fused=False)
    for kw in (dict(n_pages=1 << 30, page_size=1 << 30), dict(n_pages=1 << 30, page_size=1 << 30, n_head=1, n_kv=1), dict(n_pages=1 << 29, page_size=1 << 30)):
        for call, op in ((backend.attention, b.op(backend, max_pages=1)), (backend.rope_kv, r.op(backend, max_pages=1))):
            with pytest.raises(BackendError, match="cache buffer"):
                call(dataclasses.replace(op, **kw))
    backend.sync()


@pytest.mark.parametrize("path", [1, 2])
def test_sequences_out_of_order_are_reported(backend, path):
    # every second of 4096 sequences has all 64 rows of the call
    from moe4all_b200 import BackendError
    import torch

    b = Batch([1] * 64 + [0] * 4032, [0] * 4096, 8, 2, 64, seed=2)
    r = Rope(b, 64, False, norm=False, factors=False, fused=False)
    b.cu_t.copy_(torch.tensor([0, 64] * 2048 + [0], dtype=torch.int32))
    torch.cuda.synchronize()
    for call, op in ((backend.attention, b.op(backend, path=path)), (backend.rope_kv, r.op(backend))):
        call(op)
        with pytest.raises(BackendError, match="attention kernel"):
            backend.sync()
    b.cu_t.copy_(torch.tensor(b.cu, dtype=torch.int32))
    b = Batch([1, 5, 0, 58], [0] * 4, 8, 2, 64, seed=3)
    check(backend, b, path=path)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 640, 639, 3])
def test_widest_windows_where_rows_in_front_see_nothing(backend, path, window):
    # fewer tokens in the cache than new rows, and every window that hides nothing, or next to nothing
    b = Batch([10, 16, 200], [-4, -5, -150], 8, 2, 64, page=16, seed=4)
    want = check(backend, b, window=window, path=path)
    assert bool((want[:4] == 0).all()) and bool((want[4:10] != 0).any(1).all())
    check(backend, Batch([1, 40, 7], [600, 20, 0], 8, 2, 64, page=16, seed=5), window=window, path=path)
    check(backend, Batch([30, 1, 200], [0, 0, 0], 8, 2, 64, seed=6), window=window, path=path)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("hd", [48, 80, 128])
def test_values_rewritten_between_calls_that_put_odd_ones_together(backend, path, hd):
    # infinities in other rows and columns every time, no wait between the calls: each sees its own
    import torch
    from moe4all_b200 import RopeKv

    H, K, n, steps, w = 4, 2, [70, 9], 12, backend.wrap_tensor
    b = Batch(n, [0, 0], H, K, hd, page=16, seed=hd)
    g = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k = r(79, H * hd), r(79, K * hd)
    vs, outs, ropes, ops, wants = [], [torch.zeros_like(b.out) for _ in range(steps)], [], [], []
    for i in range(steps):
        v = r(79, K * hd)
        for row, col in ((i * 5 % 70, i * 7 % (K * hd)), (70 + i % 9, (i * 11 + 3) % (K * hd))):
            v[row, col] = float("inf") if i % 3 else float("-inf")
        vs.append(v)
        ropes.append(RopeKv(q=w(q), k=w(k), v=w(v), q_out=w(b.q), k_cache=w(b.k), v_cache=w(b.v), **b.fields(backend)))
        ops.append(b.op(backend, path=path, out=w(outs[i])))
        torch.cuda.synchronize()
        backend.rope_kv(ropes[i])
        backend.sync()
        wants.append(b.ref())
    torch.cuda.synchronize()
    for rope, op in zip(ropes, ops):
        backend.rope_kv(rope)
        backend.attention(op)
    backend.sync()
    for got, (want, tol) in zip(outs, wants):
        assert torch.equal(got.isfinite(), want.isfinite())
        assert float(torch.where(want.isfinite(), (got - want).abs(), 0.0).max()) <= tol and torch.equal(torch.where(want.isinf(), got.double(), 0.0), torch.where(want.isinf(), want, 0.0))


@pytest.mark.parametrize("path,K,n,kv", [(2, 8, 40, 16384), (1, 8, 40, 16384), (2, 1, 1, 300_000), (1, 1, 1, 300_000)])
def test_long_contexts_of_nothing_but_infinities_end_in_time(backend, path, K, n, kv):
    # every value is infinite, of one sign per column or of both: put together for two items and more to a CTA while its other warps wait
    import torch
    from moe4all_b200 import Attention

    hd, page, rows, w = 64, 256, 4, backend.wrap_tensor
    g = torch.Generator(device="cuda").manual_seed(9)
    pages = n * -(-kv // page)
    k = torch.randn(pages, K, page, hd, generator=g, device="cuda", dtype=torch.float16)
    v = torch.full_like(k, float("inf"))
    v[..., 1::2] = float("-inf")
    v[:, :, ::2, 10] = float("-inf")
    v[:, :, ::2, 11] = NAN
    q, out = torch.randn(n * rows, K * hd, generator=g, device="cuda"), torch.zeros(n * rows, K * hd, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu, lens, table = i32([i * rows for i in range(n + 1)]), i32([kv] * n), i32(list(range(pages))).view(n, -1)
    torch.cuda.synchronize()
    backend.attention(Attention(q=w(q), k=w(k), v=w(v), out=w(out), scale=0.125, cu_q=w(cu), kv_len=w(lens), page_table=w(table), rows=n * rows, n_seq=n, n_head=K, n_kv=K,
                                head_dim=hd, n_pages=pages, page_size=page, max_pages=pages // n, max_q=rows, path=path))
    backend.sync()
    want = torch.full((hd,), float("inf"), device="cuda")
    want[1::2] = float("-inf")
    want[10] = want[11] = NAN
    assert torch.equal(out.view(-1, hd).nan_to_num(nan=7.0), want.expand(n * rows * K, hd).nan_to_num(nan=7.0))


@pytest.mark.parametrize("H,K,hd,n", [(8, 2, 64, 1), (8, 1, 128, 2), (4, 1, 256, 1), (2, 1, 192, 5), (4, 1, 128, 100), (6, 2, 64, 30), (2, 1, 256, 40)])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("kv", [40, 9000])
def test_what_is_not_finite_reaches_its_row_whatever_its_weight(backend, path, H, K, hd, n, kv):
    # early keys hundreds of powers of two below the later ones: their parts' weights underflow where warps and CTAs join
    b = Batch([n, 1], [kv, kv // 2], H, K, hd, page=16, seed=hd + n)
    for s in range(2):
        k, v = b.get(b.k, s).clone(), b.get(b.v, s).clone()
        b.q[b.cu[s] : b.cu[s + 1], : H * hd] = b.q[b.cu[s] : b.cu[s + 1], : H * hd].abs() + 1.0
        k[:] = k.abs() * 0.25
        k[: kv // 3] -= 60.0
        for key, col, x in ((0, 3, "inf"), (1, 4, "nan"), (5, 6, "-inf"), (11, 6, "inf"), (kv // 4, hd - 1, "-inf")):
            v[key, :, col] = float(x)
        b.put(b.k, s, k)
        b.put(b.v, s, v)
    want = check(backend, b, path=path)[:, : H * hd].view(-1, H, hd)
    assert bool((want[:, :, 3] == float("inf")).all()) and bool(want[:, :, [4, 6]].isnan().all()) and bool((want[:, :, hd - 1] == float("-inf")).all())
    assert bool(want[:, :, [0, 1, 2, 5]].isfinite().all())
    # and a key without a score makes NaN of its rows, as early and as light as it is
    k = b.get(b.k, 0).clone()
    k[7, 0, 2] = NAN
    b.put(b.k, 0, k)
    want = check(backend, b, path=path)[:, : H * hd].view(-1, H, hd)
    assert bool(want[:n, : H // K].isnan().all()) and bool(want[:n, H // K :, 0].isfinite().all()) and bool(want[n:, :, 0].isfinite().all())


@pytest.mark.parametrize("H,K,hd,n", [(8, 2, 64, 1), (8, 1, 128, 2), (4, 1, 256, 1), (3, 3, 80, 9), (2, 1, 192, 7), (4, 1, 128, 200), (16, 1, 64, 30), (2, 1, 256, 140)])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("scale", [1, -1])
def test_infinite_keys_count_by_their_scores(backend, path, page, H, K, hd, n, scale):
    # a key with an infinite component has a score of -inf (and no weight) or +inf (and its row is NaN), by q's sign there: the formula's, not
    # that of q's pieces, the second of which may be zero or of the other sign
    import torch

    b = Batch([n, 3], [0, 0] if not page else [700, 40], H, K, hd, page=page, seed=hd + n)
    b.q[: n + 3, 2 : H * hd : hd] = b.q[: n + 3, 2 : H * hd : hd].abs() * scale
    b.q[: n + 3, 3 : H * hd : hd] = -b.q[: n + 3, 3 : H * hd : hd].abs() * scale
    b.q[: n + 3 : 2, 2 : H * hd : hd] = b.q[: n + 3 : 2, 2 : H * hd : hd].half().float()  # (no second piece, or next to none)
    inf = float("inf")
    for s in range(2):  # (the first key is finite: every row sees a score)
        k = b.get(b.k, s).clone()
        for i, key in enumerate({1, b.kv[s] // 2, b.kv[s] - 2} & set(range(1, b.kv[s]))):
            k[key, :, 2 if i % 2 else 3] = -inf if i % 2 else inf
            if i == 2:
                k[key, :, 2] = -inf  # two of them, of one sign
        b.put(b.k, s, k)
    want = check(backend, b, scale=scale * hd ** -0.5, path=path)
    assert bool(want[:, : H * hd].isfinite().all())
    # of the other sign, in one of the heads' keys: NaN from there on
    t = b.kv[0] - n + n // 2
    k = b.get(b.k, 0).clone()
    k[t, 0, 2] = inf
    b.put(b.k, 0, k)
    want = check(backend, b, scale=scale * hd ** -0.5, path=path)[:, : H * hd].view(-1, H, hd)
    assert bool(want[n // 2 : n, : H // K].isnan().all()) and (n // 2 < 3 or bool(want[2 : n // 2].isfinite().all()))


@pytest.mark.parametrize("H,K,hd,n,lens", [(4, 1, 64, 1, [4096] * 160), (4, 1, 64, 3, [131072]), (8, 1, 128, 1, [2500] * 150), (2, 1, 256, 1, [3000] * 150), (8, 2, 128, 40, [9000, 700]),
                                           (2, 2, 192, 100, [3000]), (4, 1, 64, 130, [20000])])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("above", [5, 20, 33, 45, 70])
def test_a_sink_leaves_the_others_their_accuracy(backend, path, H, K, hd, n, lens, above):
    # one key 2^above times as heavy as any other, of value zero: what is left are the others.  A weight is known to 2^-25 and at least 2^-5 where the
    # reference has fallen to its neighbours (2^-20 of it), the exponential to 2^-20; the sums have kv / 64 steps of the tensor cores in a warp, or of tiles, 2^-23
    # each.  The keys that share the sink's reference are known to 2^-25 of its weight, which is all but the whole: the other 127 of its tile, 2^15, or those of four
    # slices of 16 after which a warp looks down, 2^10; their values go up to 1.5.  (Otherwise all of a warp's or a part's keys were off by that.)
    b = Batch([n] * len(lens), [x - n for x in lens], H, K, hd, page=64, seed=above)
    b.q.zero_()
    b.q[:, 0 : H * hd : hd] = 1.0
    b.q[:, 1 : H * hd : hd] = 0.25
    for s, kv in enumerate(lens):
        k, v = b.get(b.k, s).clone(), b.get(b.v, s).clone()
        k[:, :, 0] = 0.0
        k[:, :, 1].clamp_(-2.0, 2.0)
        v[:] = 1.0 + v.abs().clamp_(max=2.0) * 0.25
        sink = (s * 37) % (kv - n)
        k[sink, :, 0], k[sink, :, 1], v[sink] = above, 0.0, 0.0
        b.put(b.k, s, k)
        b.put(b.v, s, v)
    want, _ = b.ref(scale=math.log(2.0))
    backend.attention(b.op(backend, scale=math.log(2.0), path=path))
    backend.sync()
    off = ((b.out.double() - want).abs() - want * (2.0 ** -19 + max(lens) / 64 * 2.0 ** -23))[:, : H * hd].max()
    assert float(off) <= 1.5 * (63 * 2.0 ** -35 if path == 1 else 127 * 2.0 ** -40), float(off)


@pytest.mark.parametrize("H,K,hd,n,kv", [(8, 2, 64, 1, 900), (8, 1, 128, 2, 5000), (4, 1, 256, 1, 300), (8, 2, 128, 100, 700), (2, 1, 192, 150, 300)])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("e", [12, 13, 14, 15, 17, 20, 25, 60])
@pytest.mark.parametrize("scale", [math.log(2.0), 0.37, -0.37])
def test_scores_of_any_size(backend, path, H, K, hd, n, kv, e, scale):
    # scores of 2047 x 2^e: keys that tie share the weight; those a step below have none, and where f32 still tells powers of two apart, theirs
    import torch

    b = Batch([n, 1], [kv, kv // 3], H, K, hd, page=16, seed=e)
    b.q.zero_()
    b.q[:, 0 : H * hd : hd] = 2.0 ** e
    near = e == 12 and scale == math.log(2.0)
    if near:
        b.q[:, 1 : H * hd : hd] = 1.0
    g = torch.Generator(device="cuda").manual_seed(3)
    for s in range(2):
        k = b.get(b.k, s).clone()
        pick = torch.randint(0, 7, (b.kv[s], K), generator=g, device="cuda")
        k[:, :, 0] = 2047.0 if near else torch.where(pick < 2, 2047.0, 2046.0 - pick).half()
        k[:, :, 1] = -pick.half()
        k[0, :, 0], k[0, :, 1] = 2047.0, 0.0
        if scale < 0:
            k[:, :, 0] *= -1
        b.put(b.k, s, k)
    want, _ = b.ref(scale=scale)
    backend.attention(b.op(backend, scale=scale, path=path))
    backend.sync()
    # weights to 2^-20 and two pieces, kv / 64 steps of sums
    off = (b.out.double() - want)[:, : H * hd].abs().max()
    assert float(off) <= float(b.v.nan_to_num().abs().max()) * (2.0 ** -18 + kv / 64 * 2.0 ** -23), float(off)


@pytest.mark.parametrize("kv,hd,n,H", [(2000, 64, 9, 12), (140_000, 64, 9, 12), (140_000, 64, 1, 4), (30_000, 128, 32, 4), (70_000, 192, 2, 20), (20_000, 256, 20, 6), (70_000, 16, 128, 1), (131_072, 128, 1, 8)])
@pytest.mark.parametrize("path", [1, 2])
def test_no_part_of_an_item_is_lost_or_weighed_wrong(backend, path, kv, hd, n, H):
    # keys of 128 by 128 count in a column of their own, in turn, with weights of 2^-2 .. 2^2 by the 128: all of it powers of two, whose sums f32 holds without
    # rounding within a part.  What is left: half a step at each of up to 160 parts' sums, the division, and the exponential's 2^-22 where they meet.
    import torch

    if path == 1 and H > 16:
        pytest.skip("more query heads to a kv head than the few-rows kernel takes")
    b = Batch([n], [kv - n], H, 1, hd, page=64, seed=hd)
    b.q.zero_()
    b.q[:, 0 : H * hd : hd] = 1.0
    i = torch.arange(kv, device="cuda") // 128
    level = (i * 7 + i // 5) % 5 - 2
    k, v = torch.zeros(kv, 1, hd, device="cuda", dtype=torch.float16), torch.zeros(kv, 1, hd, device="cuda", dtype=torch.float16)
    k[:, 0, 0] = level.half()
    v[torch.arange(kv, device="cuda"), 0, i % hd] = 1.0
    b.put(b.k, 0, k)
    b.put(b.v, 0, v)
    want, _ = b.ref(scale=math.log(2.0))
    backend.attention(b.op(backend, scale=math.log(2.0), path=path))
    backend.sync()
    rel = 160 * 2.0 ** -24 + 2.0 ** -20
    got, want = b.out.double()[:, : H * hd], want[:, : H * hd]
    assert bool(((got - want).abs() <= rel * want).all()), float(((got - want).abs() / want.clamp(min=1e-9)).max())
    # without any 128 of the keys: a hundred times the bound at least
    weight = torch.pow(2.0, level.double())
    column = torch.zeros(hd, dtype=torch.float64, device="cuda").index_add_(0, i % hd, weight)
    part = torch.zeros(int(i[-1]) + 1, dtype=torch.float64, device="cuda").index_add_(0, i, weight)
    assert float((part / column[torch.arange(len(part), device="cuda") % hd])[:-1].min()) > 100 * rel


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("K,n,rows,kv", [(8, 40, 4, 8192), (1, 1, 8, 100_000)])
def test_long_contexts_of_infinite_keys_end_in_time(backend, path, K, n, rows, kv):
    # one component of every key but the first has overflowed: by q's sign there a row is NaN, or sees the first key alone
    import torch
    from moe4all_b200 import Attention

    hd, page, w = 128, 256, backend.wrap_tensor
    g = torch.Generator(device="cuda").manual_seed(10)
    pages = n * -(-kv // page)
    k, v = (torch.randn(pages, K, page, hd, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    first = torch.arange(0, pages, pages // n, device="cuda")
    keep = k[first, :, 0, hd - 1].clone()
    k[..., hd - 1] = float("inf")
    k[first, :, 0, hd - 1] = keep
    q, out = torch.randn(n * rows, K * hd, generator=g, device="cuda"), torch.zeros(n * rows, K * hd, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu, lens, table = i32([i * rows for i in range(n + 1)]), i32([kv] * n), i32(list(range(pages))).view(n, -1)
    torch.cuda.synchronize()
    backend.attention(Attention(q=w(q), k=w(k), v=w(v), out=w(out), scale=0.09, cu_q=w(cu), kv_len=w(lens), page_table=w(table), rows=n * rows, n_seq=n, n_head=K, n_kv=K,
                                head_dim=hd, n_pages=pages, page_size=page, max_pages=pages // n, max_q=rows, path=path))
    backend.sync()
    plus = q.view(n, rows, K, hd)[..., hd - 1] > 0
    got = out.view(n, rows, K, hd)
    assert bool(got[plus].isnan().all())
    # (the one key's weight is the whole: its value, by two f16 pieces and a division)
    want = v[first, :, 0].float()[:, None].expand(n, rows, K, hd)
    assert float((got - want)[~plus].abs().max()) <= float(v[first, :, 0].float().abs().max()) * 2.0 ** -20


@pytest.mark.parametrize("H,K,hd,kv,n", [(8, 1, 128, 65536, 150), (16, 1, 64, 65536, 150), (4, 1, 256, 32768, 150), (8, 1, 192, 40000, 150), (2, 1, 128, 300_000, 1)])
@pytest.mark.parametrize("path", [1, 2])
def test_long_sums_of_one_sign(backend, path, H, K, hd, kv, n):
    # equal weights of values of one sign: whatever a step of the sums loses adds up.  A whole item's are kv / 128 additions in f32, half a step each, of slices or tiles
    # that the tensor cores sum in sixteen steps from zero; then pieces, division, joins.
    import torch
    from moe4all_b200 import Attention

    page, w = 256, backend.wrap_tensor
    g = torch.Generator(device="cuda").manual_seed(12)
    pages = -(-kv // page)
    k = torch.randn(pages, K, page, hd, generator=g, device="cuda", dtype=torch.float16)
    v = (1.0 + 0.25 * torch.rand(pages, K, page, hd, generator=g, device="cuda")).half()
    q, out = torch.zeros(n, H * hd, device="cuda"), torch.zeros(n, H * hd, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu, lens, table = i32(list(range(n + 1))), i32([kv] * n), i32(list(range(pages))).expand(n, -1).contiguous()  # (all of them read the same pages)
    torch.cuda.synchronize()
    backend.attention(Attention(q=w(q), k=w(k), v=w(v), out=w(out), scale=0.1, cu_q=w(cu), kv_len=w(lens), page_table=w(table), rows=n, n_seq=n, n_head=H, n_kv=K,
                                head_dim=hd, n_pages=pages, page_size=page, max_pages=pages, max_q=1, path=path))
    backend.sync()
    want = v.double().permute(0, 2, 1, 3).reshape(-1, K, hd)[:kv].mean(0).repeat_interleave(H // K, 0).view(-1)
    off = ((out.double() - want) / want).abs().max()
    assert float(off) <= kv / 128 * 2.0 ** -24 + 2.0 ** -19, float(off)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("n", [1, 3, 150])
def test_rows_whose_every_score_is_minus_infinity_get_zeros(backend, path, n):
    # a window of one key, and of every second row's key a component that has overflowed against q's sign there: there is no weight to divide by
    b = Batch([n, 2], [500, 9], 8, 2, 64, page=16, seed=n)
    b.q[:, 0 : 8 * 64 : 64] = b.q[:, 0 : 8 * 64 : 64].abs() + 0.01
    k = b.get(b.k, 0).clone()
    k[::2, :, 0] = float("-inf")
    b.put(b.k, 0, k)
    backend.attention(b.op(backend, window=1, path=path))
    backend.sync()
    own = b.get(b.v, 0).double()[b.kv[0] - n :].repeat_interleave(4, 1).view(n, -1)  # (of the other rows their own value)
    own[(b.kv[0] - n) % 2 :: 2] = 0.0
    assert float((b.out[:n].double() - own).abs().max()) <= float(own.abs().max()) * 2.0 ** -20
