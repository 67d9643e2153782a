"""GPU: rope_kv and attention at the ends of what their arguments may be, against the formulas in 64 bits (tolerances as in
test_gpu_attention.py unless a test derives its own)."""
import dataclasses

import pytest

from test_gpu_attention import Batch, Rope, check

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
