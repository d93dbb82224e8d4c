"""Sampling over logits of the whole range of floats, against the 64-bit plain form."""
import numpy as np
import pytest

import i8_cases as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import gcu  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    gcu.init(0)
    yield
    gcu.check_device()


@pytest.mark.parametrize("n", [700, 6000, 300000])
@pytest.mark.parametrize("settings", [(3e38, 0, 0.3, 0.0), (1e38, 0, 0.95, 0.0), (2e38, 40, 1.0, 0.0),
                                      (3.4e38, 3000, 0.9, 0.2), (1e37, 500, 0.7, 0.0), (3e38, 0, 0.999, 0.0)])
def test_logits_further_apart_than_the_largest_float(n, settings):
    """Temperatures at which that distance counts."""
    rng = np.random.default_rng(n)
    x = (rng.uniform(-1, 1, (6, n)) * 3.4e38).astype(np.float32)
    x[1] = np.where(rng.random(n) < 0.01, 3.4e38, -3.4e38).astype(np.float32)
    x[2] = np.where(rng.random(n) < 0.6, np.finfo(np.float32).min, x[2])
    u = rng.random(6, dtype=np.float32)
    t, k, p, m = settings
    token, prob = torch.empty(6, dtype=torch.int32, device="cuda"), torch.empty(6, device="cuda")
    gcu.dev_sample(token, torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), t, k, p, m, prob=prob)
    want = [R.sample(row, v, t, k, p, m) for row, v in zip(x, u)]
    assert token.tolist() == [w[0] for w in want]
    # weights are good to 2^-39 of themselves, their sums are exact; the quotient is rounded to a float
    assert np.allclose(prob.cpu().numpy(), [w[1] for w in want], rtol=2.0 ** -23, atol=0)
