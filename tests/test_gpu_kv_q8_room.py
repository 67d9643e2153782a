"""GPU: attention over pages of 8 bits where the device has no room for their f16 copy."""
import pytest

from test_gpu_kv_q8 import Q8Batch

pytestmark = pytest.mark.gpu


def room_for_codes():
    """Pages of codes whose f16 pages are more than the device has: [n_pages, 1, page, hd], of which the first pages are a batch's."""
    import torch

    total = torch.cuda.get_device_properties(0).total_memory
    page = 1 << 14
    return page, total // 4 // (page * 128) + 64  # K and V in f16 together: four times the codes, which are both


def test_f16_pages_that_do_not_fit(backend):
    """Calls of many rows take the few-rows kernel where the device has no room for the f16 pages, recorded ones too; what had room before still has it."""
    import torch

    from moe4all_b200 import BackendError, CudaBackend

    be = CudaBackend(0)
    page, n_pages = room_for_codes()
    small = Q8Batch([70], [200], 8, 1, 128, page=64, seed=3)
    b = Q8Batch([70, 129], [300, page + 17], 8, 1, 128, page=page, seed=4)
    codes = torch.zeros(n_pages, 1, page, 128, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_pages, 1, page, 8), 0x20, dtype=torch.uint8, device="cuda")
    codes[: b.n_pages], scales[: b.n_pages] = b.codes["k"], b.scales["k"]
    b.v, b.codes["v"], b.scales["v"] = b.k, b.codes["k"], b.scales["k"]
    wide = torch.full((2, n_pages), -1, dtype=torch.int32, device="cuda")
    wide[:, : b.width] = b.table_t
    torch.cuda.synchronize()
    w = be.wrap_tensor
    big = dict(k=w(codes), v=w(codes), k_scale=w(scales), v_scale=w(scales), page_table=w(wide), n_pages=n_pages, max_pages=n_pages)

    def right(x, call):
        want, tol = x.ref()
        x.out.fill_(7.5)
        torch.cuda.synchronize()
        call()
        be.sync()
        assert float((x.out - want).abs().max()) <= tol

    def recorded(op):
        be.graph_begin()
        be.attention(op)
        return be.graph_end()

    small_op, op = small.op(be), b.op(be, **big)
    right(small, lambda: be.attention(small_op))  # f16 pages of its own
    for _ in range(2):
        right(b, lambda: be.attention(op))
        plan = recorded(op)
        right(b, lambda: be.execute(plan))
        plan = recorded(small_op)  # (its f16 pages are still there)
        right(small, lambda: be.execute(plan))
        right(small, lambda: be.attention(small_op))
        right(b, lambda: be.attention(op))
    with pytest.raises(BackendError, match="f16 pages"):
        be.attention(b.op(be, **big, path=2))
    right(small, lambda: be.execute(plan))
    del plan, small_op, op, big, codes, scales
    be.close()
    torch.cuda.empty_cache()  # (tens of GB)
