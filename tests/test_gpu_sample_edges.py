"""GPU: `sample` where a temperature is less than a step of the logits' numbers, and where u asks for what has next to no weight, against a sort in 64 bits."""
import numpy as np
import pytest

from test_gpu_token_ends import INF, compare, run

pytestmark = pytest.mark.gpu

# The largest logit of a row and its temperature: from a step of f32 at the largest being far more than 45 temperatures (what is below it has no weight) to a few of these
# (the neighbours have some), near both ends of f32 and around nothing.
EDGES = [(100.0, 1e-8), (12.0, 1e-9), (20.0, 2e-9), (1e10, 1.0), (1e5, 1e-6), (-7.5, 1e-10), (100.0, 1e-6), (100.0, 1.69e-7), (100.0, 1.72e-7), (100.0, 3e-7), (1e17, 1.0), (-3e38, 1e30),
         (3e38, 1e-3), (1e-39, 1e-41), (1e-39, 1e-45), (0.0, 1e-45), (0.0, 1e-41), (-2.99e38, 3e37), (1.0, 1e-7), (16.0, 2e-8)]


def rows(rng, V, crowd):
    """A row to each edge: the largest some times, its neighbours below in f32 (`crowd`: most of the row), what is well below them."""
    x = np.empty((len(EDGES), V), np.float32)
    for r, (top, _) in zip(x, EDGES):
        top = np.float32(top)
        below = [top]
        for _ in range(6):
            below.append(np.nextafter(below[-1], np.float32(-INF), dtype=np.float32))
        r[:] = np.minimum(top - np.abs(top) * rng.uniform(0.1, 0.5, V) - 1e-30, below[-1]).astype(np.float32)
        n = int(V * 0.8) if crowd else 40
        r[rng.choice(V, n, replace=False)] = rng.choice(np.array(below[1:]), n, p=[0.6, 0.2, 0.1, 0.05, 0.03, 0.02])
        r[rng.choice(V, 7, replace=False)] = top
    return x


@pytest.mark.parametrize("kw", [dict(), dict(top_k=5), dict(top_k=50), dict(top_k=1500), dict(top_p=0.37), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=30, top_p=0.8, min_p=0.01),
                                dict(top_k=3000, top_p=0.95)])
@pytest.mark.parametrize("V,crowd", [(1, False), (5001, False), (5000, True), (150001, False), (40000, True)])
def test_temperatures_below_a_step_of_the_logits(backend, V, crowd, kw):
    rng = np.random.default_rng(V + crowd)
    x = rows(rng, V, crowd) if V > 1 else np.array([[t] for t, _ in EDGES], np.float32)
    ids = compare(backend, x, u=rng.random(len(EDGES), dtype=np.float32), temperature=np.array([t for _, t in EDGES], np.float32), **kw)
    assert (ids >= 0).all()


@pytest.mark.parametrize("V", [3000, 150000])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(top_k=2500), dict(top_p=0.999999), dict(top_k=2500, top_p=0.999999)])
def test_u_of_nothing_takes_the_first_token_with_a_weight(backend, V, kw):
    """Weights end at e^-45: of the first tokens those further below count as none, though a sort in 64 bits would have them."""
    x = np.full((4, V), -3.0, np.float32)
    x[:, 0], x[:, 1], x[:, 2] = -48.0, -46.0, -44.0
    x[1, 2] = -45.5
    x[2:, 3] = 0.0
    x[:, V - 7] = 0.0
    x[3] *= 0.25
    t = np.array([1.0, 1.0, 1.0, 0.25], np.float32)
    ids, prob, _, _ = run(backend, x, u=np.zeros(4, np.float32), temperature=t, **kw)
    # (what is cut off leaves less: the first of the -3.0 ones, or of the largest)
    first = [3, 3, 3, 3] if kw else [2, 3, 2, 2]
    assert ids.tolist() == first and (prob > 0).all()
