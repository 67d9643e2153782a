"""GPU: what a context keeps on the device between launches is there for its first launch, on whatever stream that comes."""
import pytest

pytestmark = pytest.mark.gpu


def test_first_call_of_a_fresh_context_on_the_callers_stream():
    # join counters (attention of one long item by many CTAs) and the router's logit words, used by the first launch behind the context's making
    import torch
    from moe4all_b200 import CudaBackend
    from test_gpu_attention import Batch

    b = Batch([1], [9000], 8, 1, 128, page=64, seed=3)
    want, tol = b.ref()
    s = torch.cuda.Stream()
    for i in range(6):
        b.out.zero_()
        torch.cuda.synchronize()
        be = CudaBackend(0)
        be.set_stream(s.cuda_stream if i % 2 else None)
        op = b.op(be)
        for _ in range(3):
            be.attention(op)
        be.sync()
        assert float((b.out - want).abs().max()) <= tol
        del op
        be.close()
