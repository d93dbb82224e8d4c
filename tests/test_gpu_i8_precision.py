"""Precision of attention over the 8-bit cache where few keys dominate, relative to each output
element (i8_bounds derives the tolerances)."""
import math

import numpy as np
import pytest

import i8_bounds as B
import i8_cases as R
from test_gpu_prefill_i8 import forced

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import gcu  # noqa: E402

# steps of k_kt's weights, of the row's largest; k_tc's are two fp16 parts
UNIT = {"few rows": 2.0 ** -25, "many rows": 2.0 ** -35}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    gcu.init(0)
    yield
    gcu.check_device()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def handle(c):
    return gcu.KvCacheI8(*(dev(t) for t in c))


def one_key_over_many(n, hd, ratio, nkv):
    """A cache whose key 5 outweighs each of the others, all alike, by exp(ratio)."""
    c = gcu.KvCacheI8.empty(1, nkv, n, hd)
    c.k.fill_(127)
    c.ks.fill_(1.0 / 127)
    c.ks[:, :, 5] = (1.0 + ratio) / 127
    return c, torch.full((1, nkv, hd), 1.0 / hd, device="cuda")


@pytest.mark.parametrize("n", [1820, 3641, 16384])
@pytest.mark.parametrize("hd", [64, 256])
def test_many_small_weights_of_equal_values(n, hd):
    """Values that are all alike come out as they are: what the small weights lose in the sum of
    products they must not keep in the sum of weights.  More heads than SMs: a CTA takes all keys."""
    nkv = 150
    # The exponentials are the same in both sums.  fp32 sums as in i8_bounds, and the weights' steps:
    # less than one each, a standard deviation of a half, six times, against a largest weight of 1.
    tol = 2.0 ** -24 * (math.sqrt(n) + 64) + 3 * math.sqrt(n) * UNIT["few rows"]
    for ratio in (16.0, 17.4, 18.0, 20.0):
        c, q = one_key_over_many(n, hd, ratio, nkv)
        c.v.fill_(127)
        c.vs.fill_(1.0 / 127)
        xo = torch.empty_like(q)
        gcu.dev_attention_decode_i8(xo, q, c, None, n, 1.0)
        one = 127 * np.float64(np.float32(1.0 / 127))
        B.check(xo, np.full((1, nkv, hd), one), np.full((1, nkv, hd), tol))


@pytest.mark.parametrize("kernel", UNIT)
@pytest.mark.parametrize("ratio", [10.0, 17.4])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_key_and_many_small_weights(kernel, ratio, hd):
    """Random values; the heavy key's are small in half of the columns, which are the others' then."""
    rng = np.random.default_rng(41)
    n, ntok = 5000, 3
    k = rng.standard_normal((1, 1, n, hd), dtype=np.float32)
    v = rng.standard_normal((1, 1, n, hd), dtype=np.float32)
    v[..., 2000, ::2] *= 1e-6
    c = R.quantize_rows(k) + R.quantize_rows(v)
    c = [c[0], c[2], c[1], c[3]]
    xq = rng.standard_normal((2, ntok, hd), dtype=np.float32) * np.float32(1 / np.sqrt(hd))
    c[2][0, 0, 2000] = 0
    scores = np.einsum("htd,nd->htn", xq, c[0][0, 0].astype(np.float32) * c[2][0, 0, :, None])
    # the heavy key: along the mean query, its scale such that it outweighs the largest by `ratio` on average
    c[0][0, 0, 2000] = R.quantize_rows(xq.mean((0, 1)))[0]
    base = np.einsum("htd,d->ht", xq, c[0][0, 0, 2000].astype(np.float32)).mean()
    c[2][0, 0, 2000] = (scores.max() + ratio) / base
    got = forced(kernel, xq, handle(c), n - ntok).reshape(ntok, 2, hd)
    for i in range(ntok):
        m = n - ntok + i + 1
        for h in range(2):
            want, tol = B.attend(xq[h, i], c[0][0, 0, :m], c[2][0, 0, :m], c[1][0, 0, :m], c[3][0, 0, :m], 1.0,
                                 unit=UNIT[kernel], cut=kernel == "many rows")
            B.check(got[i, h], want, tol)


def with_zero_rows(rng, nkv, n, hd, size):
    """Value rows of a size, one in six of zeros as the writer leaves them (scale 1), 200 in a row too."""
    v = rng.standard_normal((1, nkv, n, hd), dtype=np.float32) * np.float32(size)
    v[0, :, rng.random(n) < 1 / 6] = 0
    v[0, :, 300:500] = 0
    k, ks = R.quantize_rows(rng.standard_normal((1, nkv, n, hd), dtype=np.float32))
    v, vs = R.quantize_rows(v)
    assert np.all(vs[0, :, 300:500] == 1)
    return k, v, ks, vs


SIZES = [1e-6, 1e-3, 0.01, 1.0, 1e4, 1e24]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kernel", UNIT)
def test_prefill_rows_of_zeros(kernel, hd, size):
    """They weigh in the sum of weights and leave the other rows their precision."""
    rng = np.random.default_rng(51)
    n, ntok = 900, 130
    c = with_zero_rows(rng, 1, n, hd, size)
    xq = rng.standard_normal((2, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    got = forced(kernel, xq, handle(c), n - ntok).reshape(ntok, 2, hd)
    for i in range(0, ntok, 7):
        m = n - ntok + i + 1
        for h in range(2):
            row = c[0][0, 0, :m], c[2][0, 0, :m], c[1][0, 0, :m], c[3][0, 0, :m]
            want, tol = B.attend(xq[h, i], *row, 1.0, unit=UNIT[kernel], cut=kernel == "many rows")
            B.check(got[i, h], want, tol)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("hd", [64, 256])
def test_decode_rows_of_zeros(size, shared, hd):
    """In the sequences' own caches and in a shared prefix; the heaviest key of one head among them."""
    rng = np.random.default_rng(52)
    nseq, nkv, G, n = 3, 2, 2, 1100
    pre = with_zero_rows(rng, nkv, n, hd, size)
    own = [np.repeat(t, nseq, 0) for t in with_zero_rows(rng, nkv, 600, hd, size)]
    pre[2][0, 1, 400] *= 8
    xq = rng.standard_normal((nseq, nkv * G, hd), dtype=np.float32) * np.float32(1.5)
    lens = [600, 450, 290]
    xo = torch.empty(xq.shape, device="cuda")
    gcu.dev_attention_decode_i8(xo, dev(xq), handle(own), dev(np.asarray(lens, np.int32)), 600, hd ** -0.5,
                                prefix=handle(pre) if shared else None, plen=n if shared else 0)
    got = xo.cpu().numpy()
    for b in range(nseq):
        for h in range(nkv * G):
            j = h // G
            row = [own[t][b, j, :lens[b]] for t in (0, 2, 1, 3)]
            if shared:
                row = [np.concatenate([pre[t][0, j], r]) for t, r in zip((0, 2, 1, 3), row)]
            want, tol = B.attend(xq[b, h], *row, hd ** -0.5, unit=UNIT["few rows"])
            B.check(got[b, h], want, tol)


def test_only_rows_of_zeros():
    """Zeros come out, also when a chunk sees nothing else."""
    hd = 128
    c = gcu.KvCacheI8.empty(2, 1, 4000, hd)
    c.k.fill_(3)
    q, xo = torch.ones((2, 4, hd), device="cuda"), torch.full((2, 4, hd), 9.0, device="cuda")
    gcu.dev_attention_decode_i8(xo, q, c, None, 4000, 1.0)
    assert not xo.any()
    c.v[0, 0, 3999] = 127  # one row of 127 among 4000 equal weights
    gcu.dev_attention_decode_i8(xo, q, c, None, 4000, 1.0)
    B.check(xo[0], np.full((4, hd), 127 / 4000), np.full((4, hd), 127 / 4000 * 2.0 ** -24 * (math.sqrt(4000) + 64)))
    assert not xo[1].any()
    rows, xq = torch.full((30, 4 * hd), 9.0, device="cuda"), torch.ones((4, 30, hd), device="cuda")
    gcu.dev_attention_prefill_i8(rows, xq, c.seq(1), 3900)
    assert not rows.any()


SCORES = [1e3, 3e5, 4e7, 3e8, 6e8, 1e10, 1e26, -1e3, -3e8, -6e8, -1e10, -1e20, -1e29,
          1e32, -1e32]


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("hd", [64, 256])
def test_scores_of_any_size(score, hd):
    """One key wins by half of its score (3e8: past 2^28 in log2 units, whose neighbours are 32
    apart): its values come out.  Two such keys, alike: their mean."""
    rng = np.random.default_rng(61)
    n, at, twin = 700, 513, 77
    v, vs = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32))
    vs[0, 0, twin] = vs[0, 0, at]
    k = np.full((1, 1, n, hd), 127 if score > 0 else -127, np.int8)
    ks = np.full((1, 1, n), abs(score) / 127 * (0.5 if score > 0 else 2), np.float32)
    row = lambda t: v[0, 0, t] * np.float64(vs[0, 0, t])
    xq = np.full((1, 2, hd), 1 / hd, np.float32)
    for winners in ((at,), (twin, at)):
        ks[0, 0, list(winners)] = abs(score) / 127
        want = np.mean([row(t) for t in winners], 0)
        size = np.mean([np.abs(row(t)) for t in winners], 0)
        # a step of the weight or, of two fp16 parts, its 2^-22, the digits' sums, the division
        tol = np.broadcast_to(size * 2.0 ** -21, (2, hd))
        kv = handle((k, v, ks, vs))
        xo = torch.empty((1, 2, hd), device="cuda")
        gcu.dev_attention_decode_i8(xo, dev(xq), kv, None, n, 1.0)
        B.check(xo[0], np.broadcast_to(want, (2, hd)), tol)
        for kernel in UNIT:
            got = forced(kernel, np.repeat(xq.transpose(1, 0, 2), 90, 1), kv, n - 90).reshape(90, 2, hd)
            for i in (-1, -8):
                B.check(got[i], np.broadcast_to(want, (2, hd)), tol)


@pytest.mark.parametrize("kernel", UNIT)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("key,query", [(1e30, 1e-30), (1e33, 1e-33), (1e-30, 1e30)])
def test_large_keys_and_small_queries(kernel, cap, key, query):
    """And the other way round: their scores are ordinary ones."""
    rng = np.random.default_rng(71)
    n, ntok, hd = 300, 40, 256
    k, ks = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32) * np.float32(key))
    v, vs = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32))
    xq = (rng.standard_normal((2, ntok, hd)) * (query / 16)).astype(np.float32)
    got = forced(kernel, xq, handle((k, v, ks, vs)), n - ntok, cap=cap).reshape(ntok, 2, hd)
    for i in range(0, ntok, 5):
        m = n - ntok + i + 1
        for h in range(2):
            want, tol = B.attend(xq[h, i], k[0, 0, :m], ks[0, 0, :m], v[0, 0, :m], vs[0, 0, :m], 1.0, cap,
                                 unit=UNIT[kernel], cut=kernel == "many rows")
            B.check(got[i, h], want, tol)


@pytest.mark.parametrize("kernel", UNIT)
@pytest.mark.parametrize("outlier", [27.0, 270.0, 2700.0])
def test_outlier_query_channels(kernel, outlier):
    """A query channel far above the others over a key channel that is small: the others' bits are
    what the largest leaves them, as stated."""
    rng = np.random.default_rng(81)
    n, ntok, hd = 600, 24, 128
    k = rng.standard_normal((1, 1, n, hd), dtype=np.float32)
    k[..., 9] *= np.float32(1 / outlier)
    k, ks = R.quantize_rows(k)
    v, vs = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32))
    xq = rng.standard_normal((2, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    xq[..., 9] *= np.float32(outlier)
    got = forced(kernel, xq, handle((k, v, ks, vs)), n - ntok).reshape(ntok, 2, hd)
    for i in range(ntok):
        m = n - ntok + i + 1
        for h in range(2):
            want, tol = B.attend(xq[h, i], k[0, 0, :m], ks[0, 0, :m], v[0, 0, :m], vs[0, 0, :m], 1.0,
                                 unit=UNIT[kernel], cut=kernel == "many rows")
            B.check(got[i, h], want, tol)


@pytest.mark.parametrize("kernel", UNIT)
def test_queries_keep_24_bits(kernel):
    """Elements of three steps of the largest one's 2^-23, over keys that are zero where that one is:
    the scores are theirs alone, and nothing of them is rounded."""
    rng = np.random.default_rng(91)
    n, ntok, hd = 500, 20, 128
    k, _ = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32))
    k[..., 0] = 0
    ks = rng.uniform(600, 1200, (1, 1, n)).astype(np.float32)
    v, vs = R.quantize_rows(rng.standard_normal((1, 1, n, hd), dtype=np.float32))
    small = (rng.choice([-3, -1, 1, 3], (2, ntok, hd)) / 8355000).astype(np.float32)
    xq = small.copy()
    xq[..., 0] = 1
    small[..., 0] = 0
    got = forced(kernel, xq, handle((k, v, ks, vs)), n - ntok).reshape(ntok, 2, hd)
    for i in range(ntok):
        m = n - ntok + i + 1
        for h in range(2):
            want, tol = B.attend(small[h, i], k[0, 0, :m], ks[0, 0, :m], v[0, 0, :m], vs[0, 0, :m], 1.0,
                                 unit=UNIT[kernel], cut=kernel == "many rows")
            B.check(got[i, h], want, tol)
