"""Sampling on the GPU against the 64-bit plain form: tokens equal, shares to fp32."""
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


def run(x, u, t=1.0, k=0, p=1.0, minp=0.0):
    x = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda() if not torch.is_tensor(x) else x
    token = torch.full((len(u),), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((len(u),), -7.0, device="cuda")
    gcu.dev_sample(token, x, torch.from_numpy(np.asarray(u, np.float32)).cuda(), t, k, p, minp, prob=prob)
    torch.cuda.synchronize()
    return token.cpu().numpy(), prob.cpu().numpy()


def check(x, u, t=1.0, k=0, p=1.0, minp=0.0):
    token, prob = run(x, u, t, k, p, minp)
    for i, row in enumerate(x):
        want, share = R.sample(row, u[i], t, k, p, minp)
        assert token[i] == want, (i, token[i], want)
        # a share of 64-bit sums, rounded once, of weights kept to 2^-43 of the largest at least
        assert abs(prob[i] - share) <= share * 2.0 ** -24 + 2.0 ** -40


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 1, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.3, 0, 0.5, 0.0), (1.0, 0, 0.9, 0.05),
            (2.0, 5000, 0.99, 0.0), (0.3, 7, 0.3, 0.2), (1.0, 0, 1.0, 0.01), (5.0, 0, 0.97, 0.0), (0.01, 0, 0.9, 0.0)]


@pytest.mark.parametrize("t,k,p,minp", SETTINGS)
@pytest.mark.parametrize("n", [1, 2, 31, 1000, 4097, 50001, 262144])
def test_random_rows(n, t, k, p, minp):
    rng = np.random.default_rng(n)
    m = 3 if n > 10000 else 6
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    check(x, rng.random(m, dtype=np.float32), t, k, p, minp)


@pytest.mark.parametrize("t,k,p,minp", SETTINGS)
def test_ties(t, k, p, minp):
    """Whole rows of few values: the cut falls among equal logits, by the lowest index."""
    rng = np.random.default_rng(12)
    x = rng.integers(0, 3, (6, 20000)).astype(np.float32)
    x[0] = 0
    x[1] = np.where(x[1] == 0, -0.0, 0.0)  # -0 and +0 are equal
    check(x, np.array([0.0, 0.2, 0.5, 0.7, 0.999, 0.31], np.float32), t, k, p, minp)


def test_greedy_and_odd_rows():
    rng = np.random.default_rng(13)
    x = rng.standard_normal((7, 1003)).astype(np.float32)
    x[0, [700, 12]] = 50  # a tie: the lower index
    x[1] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4, [5, 900]] = np.inf
    x[5] = -np.inf
    x[5, 77] = -3e38
    x[6] = -3.4028235e38  # the type's lowest value everywhere
    u = np.array([0.4, 0.4, 0.4, 0.4, 0.6, 0.4, 0.4], np.float32)
    for s in [(0.0, 0, 1.0, 0.0)] + SETTINGS:
        check(x, u, *s)
    assert run(x, u, 0.0)[0][0] == 12 and run(x, u)[0][1] == -1 and run(x, u)[0][4] == 900


def test_random_numbers_at_the_ends():
    x = np.zeros((5, 64), np.float32)
    token, _ = run(x, np.array([0.0, np.float32(1) - np.float32(2 ** -24), 1.0, -1.0, np.nan], np.float32))
    assert token.tolist() == [0, 63, 63, 0, 0]


def test_strided_rows_and_no_prob():
    rng = np.random.default_rng(14)
    x = torch.from_numpy(rng.standard_normal((5, 1100)).astype(np.float32)).cuda()
    v = x[:, 3:1040]  # odd offset, row stride 1100
    token = torch.empty(5, dtype=torch.int32, device="cuda")
    u = rng.random(5, dtype=np.float32)
    gcu.dev_sample(token, v, torch.from_numpy(u).cuda(), 0.9, 50, 0.9)
    for i, row in enumerate(v.cpu().numpy()):
        assert token[i].item() == R.sample(row, u[i], 0.9, 50, 0.9, 0.0)[0]


def test_the_draws_follow_the_weights():
    """Evenly spread random numbers hit each token as often as its share says, to one draw each."""
    x = np.log(np.array([[0.1, 0.2, 0.3, 0.4]], np.float32)).repeat(1000, 0)
    u = (np.arange(1000, dtype=np.float32) + 0.5) / 1000
    token, _ = run(x, u)
    assert np.all(np.abs(np.bincount(token, minlength=4) - [100, 200, 300, 400]) <= 1)


def test_same_answer_in_every_call_and_graph():
    rng = np.random.default_rng(15)
    x = torch.from_numpy((rng.standard_normal((4, 30000)) * 2).astype(np.float32)).cuda()
    u = torch.rand(4, device="cuda")
    token = torch.empty(4, dtype=torch.int32, device="cuda")
    gcu.dev_sample(token, x, u, 1.0, 0, 0.9)
    first = token.clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        gcu.dev_sample(token, x, u, 1.0, 0, 0.9)
    for _ in range(3):
        token.zero_()
        g.replay()
        assert torch.equal(token, first)
    u.fill_(0.0)
    g.replay()
    assert token.tolist() == [R.sample(r, 0.0, 1.0, 0, 0.9, 0.0)[0] for r in x.cpu().numpy()]


@pytest.mark.parametrize("t,k,p,minp", SETTINGS)
@pytest.mark.parametrize("n", [262145, 400001, 1 << 20])
def test_rows_longer_than_shared_memory(n, t, k, p, minp):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((3, n)) * 3).astype(np.float32)
    x[1] = rng.integers(0, 2, n)  # ties
    x[2, ::3] = np.nan
    x[2, [n - 5, 70]] = np.inf
    check(x, np.array([0.3, 0.6, 0.7], np.float32), t, k, p, minp)


@pytest.mark.parametrize("t", [1e-45, 1e-38, 1e-20, 1e20, 3e38])
@pytest.mark.parametrize("k,p,minp", [(0, 1.0, 0.0), (20, 1.0, 0.0), (0, 0.9, 0.0), (900, 0.4, 0.3)])
def test_extreme_temperatures(t, k, p, minp):
    rng = np.random.default_rng(16)
    x = rng.standard_normal((5, 3001)).astype(np.float32)
    x[1, 100:] = -np.inf
    x[2] = np.float32(1e-45) * rng.integers(0, 4, 3001).astype(np.float32)  # steps of the smallest float
    x[3] = np.where(rng.random(3001) < 0.5, -3.4028235e38, 3.4028235e38)
    x[4, 1::2] = np.nan
    check(x, np.array([0.2, 0.9, 0.5, 0.7, 0.999], np.float32), t, k, p, minp)


def test_many_rows():
    rng = np.random.default_rng(17)
    x, u = (rng.standard_normal((700, 517)) * 2).astype(np.float32), rng.random(700, dtype=np.float32)
    check(x, u, 0.8, 30, 0.9, 0.02)
    check(x, u)


def test_two_streams_at_once():
    rng = np.random.default_rng(18)
    x, u = (rng.standard_normal((40, 20001)) * 2).astype(np.float32), rng.random(40, dtype=np.float32)
    want = [R.sample(r, v, 0.9, 0, 0.9, 0.0)[0] for r, v in zip(x, u)]
    dx, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            token = torch.empty(40, dtype=torch.int32, device="cuda")
            gcu.dev_sample(token, dx, du, 0.9, 0, 0.9)
            outs.append(token)
    torch.cuda.synchronize()
    assert all(t.tolist() == want for t in outs)


@pytest.mark.parametrize("k", [2, 31, 32, 33, 255, 256, 257, 600, 1023, 1024, 1025])
def test_lists_of_every_length(k):
    """Cuts whose lists are sorted by counting, by exchanges, and not at all."""
    rng = np.random.default_rng(k)
    x = (rng.standard_normal((3, 30000)) * 2).astype(np.float32)
    x[1] = rng.integers(0, 200, 30000).astype(np.float32) / 8  # steps of many equal logits
    x[2, k:] = -np.inf  # no more than k to keep
    u = np.array([0.35, 0.77, 0.999], np.float32)
    check(x, u, 1.0, k)
    check(x, u, 3.0, k, 0.6, 0.01)
    check(x, u, 0.5, 0, 1 - 1 / k)
