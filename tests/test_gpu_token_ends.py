"""GPU: the two ends of a step through the C ABI - rows of a token table, tokens of rows of logits - against the formulas in 64 bits.

embed: a weight is A * (code - off) + B of f32 numbers and one product with the scale, 2^-22 of |A code| + |B| at most (Q4_K: codes up to 15 of steps that cancel
against the minimum).  sample: ids are equal; u and the settings are chosen at random or well apart from where a sum of 64 bits could decide otherwise."""
import dataclasses

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def tensors(be, **arrays):
    import torch

    out = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in arrays.items()}
    torch.cuda.synchronize()
    return out


# ---- embed

BLOCKS = [2, 3, 6, 7, 8, 10, 11, 12, 13, 14, 20, 23, 39, 40, 42, 17, 22, 18, 21]


@pytest.mark.parametrize("dtype", [0, 1, 30] + BLOCKS)
@pytest.mark.parametrize("ne,rows", [(256, 1), (512, 37), (2048 + 256, 5), (7168, 130)])
def test_embed(backend, dtype, ne, rows):
    import torch

    from moe4all_b200 import DType, Embed, synth
    from oracle import oracle as orc

    rng = np.random.default_rng(dtype * 1000 + ne)
    V, scale = 61, 3.25
    if dtype == 0:
        raw = rng.normal(size=(V, ne)).astype(np.float32)
        want = raw.astype(np.float64)
    elif dtype == 1:
        raw = rng.normal(size=(V, ne)).astype(np.float16)
        want = raw.astype(np.float64)
    elif dtype == 30:
        want = torch.randn(V, ne, generator=torch.Generator().manual_seed(ne)).bfloat16()
        raw, want = want.view(torch.int16).numpy(), want.double().numpy()
    else:
        if dtype in (17, 18, 21, 22):
            table = synth.codebook(dtype)
            backend.set_codebook(dtype, table)
            orc.set_codebook(dtype, table)
        raw = synth.random_blocks(rng, dtype, V * ne)
        want = orc.dequant(dtype, raw, V * ne).astype(np.float64).reshape(V, ne)
    ids = rng.integers(0, V, rows).astype(np.int32)
    ids[0], ids[-1] = 0, V - 1
    pad = 8
    t = tensors(backend, table=raw.view(np.uint8).reshape(-1), ids=ids, dst=np.full((rows + 1, ne + pad), 7.5, np.float32))
    w = backend.wrap_tensor
    backend.embed(Embed(table=w(t["table"]), dtype=DType(dtype), ids=w(t["ids"]), dst=w(t["dst"]), rows=rows, ne=ne, n_vocab=V, scale=scale, dst_stride=ne + pad))
    backend.sync()
    got = t["dst"].cpu().numpy()
    assert (got[rows] == 7.5).all() and (got[:, ne:] == 7.5).all()
    want = scale * want[ids]
    # the affine formats cancel: |A code| and |B| are up to the block's spread
    tol = 2.0 ** -21 * np.abs(want) + (2.0 ** -21 * np.abs(want).max() if dtype in (3, 7, 10, 12, 13) else 0.0)
    assert (np.abs(got[:rows, :ne] - want) <= tol).all()


def test_embed_reports_ids_outside(backend):
    from moe4all_b200 import BackendError, DType, Embed

    rng = np.random.default_rng(1)
    t = tensors(backend, table=rng.normal(size=(10, 64)).astype(np.float32), ids=np.array([3, 10, -1, 9, 2 ** 31 - 1], np.int32), dst=np.full((5, 64), 7.5, np.float32))
    w = backend.wrap_tensor
    backend.embed(Embed(table=w(t["table"]), ids=w(t["ids"]), dst=w(t["dst"]), rows=5, ne=64, n_vocab=10))
    with pytest.raises(BackendError, match="token id"):
        backend.sync()
    got, table = t["dst"].cpu().numpy(), t["table"].cpu().numpy()
    assert (got[[1, 2, 4]] == 0).all() and (got[[0, 3]] == table[[3, 9]]).all()
    backend.sync()  # reported once


def test_embed_table_past_32_bits(backend):
    import torch

    from moe4all_b200 import DType, Embed

    ne, V = 4096, (1 << 32) // 8192 + 100
    table = torch.zeros(V, ne, dtype=torch.float16, device="cuda")
    table[-1] = torch.arange(ne, device="cuda").half()
    ids, dst = torch.tensor([V - 1, V - 2], dtype=torch.int32, device="cuda"), torch.full((2, ne), 7.5, device="cuda")
    torch.cuda.synchronize()
    w = backend.wrap_tensor
    backend.embed(Embed(table=w(table), dtype=DType.F16, ids=w(ids), dst=w(dst), rows=2, ne=ne, n_vocab=V))
    backend.sync()
    assert torch.equal(dst[0], table[-1].float()) and bool((dst[1] == 0).all())


def test_embed_refusals(backend):
    from moe4all_b200 import BackendError, DType, Embed, Unsupported

    be = backend
    t = tensors(be, table=np.zeros(64 * 144, np.uint8), ids=np.zeros(4, np.int32), dst=np.zeros((4, 256), np.float32))
    w = be.wrap_tensor
    ok = Embed(table=w(t["table"]), dtype=DType.Q4K, ids=w(t["ids"]), dst=w(t["dst"]), rows=4, ne=256, n_vocab=64)

    def refused(kind, **kw):
        with pytest.raises(kind) as e:
            be.embed(dataclasses.replace(ok, **kw))
        if kind is BackendError:
            assert not isinstance(e.value, Unsupported)

    for kw in (dict(ne=0), dict(n_vocab=0), dict(n_vocab=65), dict(ne=128), dict(rows=5), dict(scale=NAN), dict(scale=INF), dict(dst_stride=255), dict(dst_stride=258),
               dict(ids=be.wrap(t["ids"].data_ptr(), 12)), dict(dst=ok.table), dict(dst=be.wrap(t["table"].data_ptr() + 4096, 4096))):
        refused(BackendError, **kw)
    for kw in (dict(dtype=5), dict(dtype=DType.F32, ne=24, n_vocab=4), dict(n_vocab=1 << 31), dict(dst_stride=(1 << 24) + 4)):
        refused(Unsupported, **kw)
    assert be._lib.infr_cuda_embed(be._ctx, None) == -1
    be.embed(dataclasses.replace(ok, rows=0))
    be.embed(ok)
    be.sync()


# ---- sample

def reference(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """A row's token and its share of the kept weight, in 64 bits, by a sort."""
    x = x.astype(np.float64) + 0.0
    if np.isnan(x).any() or x.max() == -INF:
        return -1, 0.0
    if not T > 0 or k == 1:
        return int(np.argmax(x)), 1.0
    top = x.max()
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -INF, 0.0, np.exp(np.where(x == -INF, 0.0, (x - top)) / np.float64(T))))
    if top == INF:
        w = (x == INF).astype(np.float64)
    order = np.lexsort((np.arange(x.size), -x))
    n = min(k, x.size) if k > 0 else x.size
    ws = w[order]
    if p < 1:
        c = np.cumsum(ws[:n])
        n = min(n, 1 + int((c < p * c[-1]).sum())) if p > 0 else 1
    keep = np.zeros(x.size, bool)
    keep[order[:n]] = True
    if m > 0:
        keep &= w >= min(m, 1.0)
    w = np.where(keep, w, 0.0)
    c = np.cumsum(w)
    u = min(max(0.0 if np.isnan(u) else u, 0.0), 1.0)
    i = min(int((c <= u * c[-1]).sum()), int(np.flatnonzero(w)[-1]))
    return i, w[i] / c[-1]


def run(be, x, stride=0, prob=True, **rows):
    """Samples rows x [n, V] with settings by row; (ids, prob)."""
    from moe4all_b200 import Sample

    n, V = x.shape
    flat = np.full((n, max(stride, V)), NAN, np.float32)
    flat[:, :V] = x
    flat = np.concatenate([flat.reshape(-1)[: (n - 1) * max(stride, V) + V]])
    kinds = dict(u=np.float32, temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    t = tensors(be, x=flat, ids=np.full(n, -5, np.int32), prob=np.full(n, 7.5, np.float32), **{k: np.broadcast_to(np.asarray(v, kinds[k]), (n,)) for k, v in rows.items()})
    w = be.wrap_tensor
    op = Sample(logits=w(t["x"]), ids=w(t["ids"]), prob=w(t["prob"]) if prob else None, rows=n, n_vocab=V, stride=stride, **{k: w(t[k]) for k in rows})
    be.sample(op)
    be.sync()
    return t["ids"].cpu().numpy(), t["prob"].cpu().numpy(), t, op


def compare(be, x, stride=0, **rows):
    got, prob, _, _ = run(be, x, stride, **rows)
    names = dict(u="u", temperature="T", top_k="k", top_p="p", min_p="m")
    kinds = dict(u=np.float32, temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    for i in range(x.shape[0]):
        kw = {}
        for n, v in rows.items():
            v = np.broadcast_to(np.asarray(v, kinds[n]), (x.shape[0],))[i]
            kw[names[n]] = int(v) if n == "top_k" else float(v)
        id, share = reference(x[i], **kw)
        assert got[i] == id, (i, kw, got[i], id)
        # (weights in 64 bits, the quotient rounded once)
        assert abs(prob[i] - share) <= share * 2.0 ** -23 + 1e-14, (i, kw, prob[i], share)
    return got


def logits(rng, n, V, spread=2.2):
    x = rng.normal(size=(n, V)) * spread
    for r in x:
        r[rng.integers(0, V, 20)] += rng.uniform(3, 12) * rng.uniform(0, 1, 20)
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 7, 31, 32, 33, 100, 1000, 4097, 32000, 50257, 150001])
def test_settings_by_row(backend, V):
    rng = np.random.default_rng(V)
    n = 40 if V > 40000 else 96
    x = logits(rng, n, V)
    pick = lambda *v: rng.choice(np.array(v), n)
    compare(backend, x, u=rng.random(n, dtype=np.float32), temperature=pick(0.0, 0.05, 0.6, 1.0, 1.0, 2.5), top_k=pick(0, 0, 1, 2, 20, 50, 700, 3000, V, V + 5, -1),
            top_p=pick(1.0, 1.0, 0.05, 0.5, 0.9, 0.99, 0.0), min_p=pick(0.0, 0.0, 0.01, 0.1, 0.9))


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.3), dict(top_k=5), dict(top_p=0.7), dict(min_p=0.05), dict(top_k=2500), dict(top_k=2500, top_p=0.6), dict(top_k=60000, top_p=0.95),
                                dict(temperature=30.0, top_p=0.5), dict(temperature=1e6, top_p=0.3, top_k=40000), dict(temperature=1e-3, top_p=0.5, top_k=7)])
@pytest.mark.parametrize("V,stride", [(70001, 0), (70001, 70007), (65536, 65540), (400003, 0)])
def test_each_setting_alone(backend, kw, V, stride):
    # (400003: more than shared memory holds of a row)
    rng = np.random.default_rng(V + len(kw))
    compare(backend, logits(rng, 6, V), stride, u=rng.random(6, dtype=np.float32), **kw)


@pytest.mark.parametrize("V", [5000, 150000])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=37), dict(top_k=4321), dict(top_p=0.37), dict(top_p=0.9), dict(top_k=4500, top_p=0.5), dict(min_p=0.5)])
def test_equal_logits(backend, V, kw):
    """Ties: of equal logits the lowest ids are kept, however many there are."""
    rng = np.random.default_rng(V)
    x = np.zeros((5, V), np.float32)
    x[1] = -0.0
    x[1, ::3] = 0.0
    x[2] = rng.integers(0, 2, V)
    x[3] = np.where(rng.random(V) < 0.001, 1.0, np.where(rng.random(V) < 0.5, np.float32(1.0) - np.float32(2.0 ** -24), -20.0))
    x[4] = -3.4028234663852886e38
    compare(backend, x, u=np.array([0.3, 0.77, 0.5, 0.123, 0.9], np.float32), **kw)


def test_values_close_together(backend):
    """Rows whose values are a few of f32's steps apart, around nothing and far from it: the bins have to be drawn finer and finer."""
    rng = np.random.default_rng(4)
    V = 60000
    rows = []
    for base in (0.0, 1.0, -7.25, 3e-39, 1e30):
        step = np.spacing(np.float32(max(abs(base), 1e-40)))
        rows.append((np.float64(base) + rng.integers(-9000, 9000, V) * np.float64(step)).astype(np.float32))
    x = np.stack(rows)
    for kw in (dict(top_k=3000), dict(top_k=20000), dict(top_p=0.4), dict(top_k=30000, top_p=0.7), dict(top_p=0.9, min_p=0.1)):
        compare(backend, x, u=np.float32(0.61), **kw)
    # and two heaps far apart with a few values in between
    x = np.where(rng.random((4, V)) < 0.5, np.float32(5.0), np.float32(4.5)) + (rng.integers(0, 300, (4, V)) * 2.0 ** -21).astype(np.float32)
    for kw in (dict(top_k=9000), dict(top_p=0.33), dict(top_p=0.62), dict(top_p=0.97)):
        compare(backend, x.astype(np.float32), u=np.float32(0.4), **kw)


def test_masks_and_what_is_not_finite(backend):
    rng = np.random.default_rng(5)
    V = 20000
    x = logits(rng, 12, V)
    low = np.float32(-3.4028234663852886e38)
    x[0, 100:] = -INF
    x[1] = -INF
    x[1, 777] = -3.0
    x[2] = -INF
    x[3, 5] = NAN
    x[4] = low
    x[4, 19999] = 1.0
    x[5, 30], x[5, 19000] = INF, INF
    x[6, 1:] = low
    x[7] = np.where(rng.random(V) < 0.9, -INF, x[7])
    x[8] = np.where(rng.random(V) < 0.9, low, x[8])
    x[9, 0] = -NAN
    x[10] = 3.4028234663852886e38
    x[10, ::2] = low
    x[11] = -INF
    x[11, 3] = INF
    u = rng.random(12, dtype=np.float32)
    for kw in (dict(), dict(temperature=0.0), dict(top_k=300), dict(top_p=0.9), dict(top_k=6000, top_p=0.8), dict(temperature=0.01), dict(temperature=INF), dict(min_p=0.2), dict(top_k=1)):
        ids = compare(backend, x, u=u, **kw)
        assert (ids[[2, 3, 9]] == -1).all() and ids[1] == 777 and ids[11] == 3 and ids[5] in (30, 19000)
        assert (ids[[0, 1, 4, 5, 6, 7, 8, 10, 11]] >= 0).all()


def test_settings_that_are_no_settings(backend):
    rng = np.random.default_rng(6)
    x = logits(rng, 12, 3001)
    u = np.array([0.0, 1.0, 2.0, -1.0, NAN, INF, -INF, 0.5, 1 - 2.0 ** -24, 1e-45, 0.25, 0.75], np.float32)
    compare(backend, x, u=u)
    compare(backend, x, u=u, top_p=0.9, top_k=50)
    for kw in (dict(temperature=NAN), dict(temperature=-1.0), dict(top_p=NAN), dict(top_p=-2.0), dict(top_p=5.0), dict(min_p=NAN), dict(min_p=-1.0), dict(min_p=3.0),
               dict(top_k=-2 ** 31), dict(top_k=2 ** 31 - 1), dict(temperature=1e-45), dict(temperature=3e38)):
        kw = {k: np.float32(v) if k != "top_k" else v for k, v in kw.items()}
        compare(backend, x, u=np.linspace(0.05, 0.95, 12, dtype=np.float32), **kw)


def test_draws_follow_the_weights(backend):
    """4096 rows of the same logits: u on a grid takes each token as often as its weight says, to one in the grid."""
    rng = np.random.default_rng(7)
    n, V = 4096, 257
    row = logits(rng, 1, V, spread=1.0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    ids, _, _, _ = run(backend, np.repeat(row, n, 0), u=u, top_k=40)
    order = np.argsort(-row[0], kind="stable")[:40]
    w = np.zeros(V)
    w[order] = np.exp(row[0, order].astype(np.float64) - row[0].max())
    share = np.bincount(ids, minlength=V) / n
    assert np.abs(share - w / w.sum()).max() <= 1.01 / n and (np.diff(ids) >= 0).all()


def test_rows_do_not_touch_each_other_and_repeat(backend):
    import torch

    rng = np.random.default_rng(8)
    x = logits(rng, 300, 5003)
    kw = dict(u=rng.random(300, dtype=np.float32), top_k=rng.choice([0, 30, 2600], 300), top_p=rng.choice([1.0, 0.9], 300).astype(np.float32))
    ids, prob, t, op = run(backend, x, **kw)
    alone = [run(backend, x[i : i + 1], **{k: v[i : i + 1] for k, v in kw.items()})[:2] for i in range(0, 300, 7)]
    assert [int(a[0][0]) for a in alone] == ids[::7].tolist() and [float(a[1][0]) for a in alone] == prob[::7].tolist()
    backend.graph_begin()
    backend.sample(op)
    plan = backend.graph_end()
    stream = torch.cuda.Stream()
    for s in (None, stream.cuda_stream):
        backend.set_stream(s)
        t["ids"].fill_(-9)
        torch.cuda.synchronize()
        backend.execute(plan)
        backend.sync()
        assert t["ids"].cpu().numpy().tolist() == ids.tolist()
    backend.set_stream(None)


def test_sample_refusals(backend):
    from moe4all_b200 import BackendError, Sample, Unsupported

    be = backend
    x = logits(np.random.default_rng(9), 4, 1000)
    _, _, t, ok = run(be, x, u=0.5, temperature=1.0, top_k=5, top_p=0.9, min_p=0.1)
    small = be.wrap(t["u"].data_ptr(), 8)

    def refused(kind, **kw):
        with pytest.raises(kind) as e:
            be.sample(dataclasses.replace(ok, **kw))
        if kind is BackendError:
            assert not isinstance(e.value, Unsupported)

    for kw in (dict(n_vocab=0), dict(n_vocab=1001), dict(rows=5), dict(stride=999), dict(stride=1001), dict(u=small), dict(ids=small), dict(temperature=small), dict(top_k=small),
               dict(top_p=small), dict(min_p=small), dict(prob=small), dict(ids=ok.logits), dict(prob=ok.ids), dict(ids=ok.u), dict(prob=ok.min_p), dict(ids=ok.top_k)):
        refused(BackendError, **kw)
    for kw in (dict(n_vocab=(1 << 24) + 1), dict(rows=(1 << 22) + 1)):
        refused(Unsupported, **kw)
    assert be._lib.infr_cuda_sample(be._ctx, None) == -1
    be.sample(dataclasses.replace(ok, rows=0))
    be.sample(dataclasses.replace(ok, prob=None, temperature=None, top_k=None, top_p=None, min_p=None))
    be.sync()


@pytest.mark.parametrize("k", [2, 63, 64, 65, 1023, 1024, 1025, 4096, 4097])
@pytest.mark.parametrize("order", ["up", "down", "one_part", "mixed"])
def test_where_the_largest_lie(backend, k, order):
    """Sorted logits, and the largest all in one stretch of the row: what a CTA or a thread finds of them is anything from none to all."""
    V = 60000
    x = np.sort(logits(np.random.default_rng(k), 1, V)[0])
    if order == "down":
        x = x[::-1]
    elif order == "one_part":
        x = np.concatenate([x[: V // 3], x[V - 5000 :], x[V // 3 : V - 5000]])
    elif order == "mixed":
        x = np.random.default_rng(k + 1).permutation(x)
    x = np.tile(x, (4, 1)).astype(np.float32)
    compare(backend, x, u=np.array([0.0, 0.31, 0.77, 0.999]), top_k=[k, k, k, k], top_p=[1.0, 0.9, 1.0, 0.5], temperature=[1.0, 1.0, 3.0, 30.0])


def test_samplers_of_two_contexts(backend):
    import torch

    from moe4all_b200 import CudaBackend

    rng = np.random.default_rng(77)
    x = logits(rng, 3, 90001)
    kw = dict(u=rng.random(3), top_k=[0, 50, 2000], top_p=[0.9, 1.0, 0.8])
    want, _, _, op = run(backend, x, **kw)
    other = CudaBackend(0)
    try:
        got, _, _, op2 = run(other, x, **kw)
        assert (got == want).all()
        for _ in range(10):
            backend.sample(op), other.sample(op2)
        backend.sync(), other.sync()
        torch.cuda.synchronize()
        assert (run(backend, x, **kw)[0] == want).all()
    finally:
        other.close()
