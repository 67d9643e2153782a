"""GPU: the angles of rows on their way into pages of 8 bits."""
import pytest

from test_gpu_kv_q8 import Q8Batch, Q8Rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_rot", [128, 32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sines_and_cosines(backend, n_rot, interleaved):
    """Pairs (1, 0) turn into their angle's cosine and sine.  These are off by f32's sincospi, one unit in the last place (2^-24 below 1), and by the rounding of
    the part that an angle of f32 leaves, half of one."""
    import torch

    b = Q8Batch([2000, 3000], [0, 30000], 2, 1, 128, page=64, seed=1)
    r = Q8Rope(b, n_rot, interleaved)
    for x in r.parts:
        x.zero_()
    half = n_rot // 2
    r.parts[0].view(-1, 2, 128)[..., slice(0, n_rot, 2) if interleaved else slice(0, half)] = 1.0
    (want, _, _), _ = r.ref()
    torch.cuda.synchronize()
    backend.rope_kv(r.op(backend))
    backend.sync()
    assert float((r.q_out.double() - want).abs().max()) <= 1.5 * 2.0 ** -24 + 1e-10
