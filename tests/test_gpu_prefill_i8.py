"""Both kernels of prefill attention over the 8-bit cache, each forced, against the 64-bit
plain form (tolerance derived in i8_cases.tolerance), and the public call at sizes
where either is taken."""
import numpy as np
import pytest

import i8_cases as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import gcu  # noqa: E402

KERNELS = {"few rows": 1, "many rows": 2}


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


def forced(kernel, xq, kv, spos, slide=0, cap=0.0, mask=True, extra=0):
    nh, ntok, hd = xq.shape
    xo, q = torch.full((ntok, nh * hd + extra), 9.0, device="cuda"), dev(xq)
    work = torch.full((64 << 18,), float("nan"), device="cuda")  # 64 MB that nothing may be read from unwritten
    rc = gcu.lib().gcu_dev_attention_prefill_i8_tuned(xo.data_ptr(), nh * hd + extra, q.data_ptr(), kv.ref, nh, spos, ntok,
                                                      slide, cap, int(mask), work.data_ptr(), work.numel() * 4,
                                                      KERNELS[kernel], torch.cuda.current_stream().cuda_stream)
    assert rc == 0, gcu.lib().gcu_last_error().decode()
    torch.cuda.synchronize()
    got = xo.cpu().numpy()
    assert np.all(got[:, nh * hd:] == 9.0)
    return got[:, :nh * hd]


def check(got, want, tol):
    assert np.all(np.isfinite(got))
    err = np.max(np.abs(got - want))
    assert err <= tol, f"max error {err:.3g}, allowed {tol:.3g}"


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 256), (8, 4, 256), (4, 2, 128), (6, 4, 64), (8, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("spos,ntok,slide,cap,mask", [
    (0, 1, 0, 0.0, True), (0, 33, 0, 0.0, True), (63, 65, 0, 0.0, True), (5, 130, 0, 0.0, True),
    (100, 70, 20, 0.0, True), (0, 129, 64, 0.0, True), (0, 150, 1, 0.0, True), (7, 60, 0, 4.0, True),
    (13, 67, 0, 0.0, False), (200, 9, 0, 0.0, True), (900, 40, 0, 0.0, True), (500, 100, 333, 0.0, True)])
def test_sizes_and_masks(kernel, nh, nkv, hd, spos, ntok, slide, cap, mask):
    rng = np.random.default_rng(spos + ntok)
    c = R.cache(rng, 1, nkv, spos + ntok + 1, hd)
    c[2][0, :, -1], c[3][0, :, -1] = np.nan, np.nan  # behind the chunk
    xq = rng.standard_normal((nh, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    want, tol = R.prefill(xq, tuple(t[:, :, :spos + ntok] for t in c), spos, slide, cap, mask)
    check(forced(kernel, xq, handle(c), spos, slide, cap, mask, extra=4), want, tol)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_growing_scores(kernel, hd):
    """Each later key scores far above the ones before it: the reference point moves all the time."""
    rng = np.random.default_rng(2)
    c = list(R.cache(rng, 1, 1, 600, hd))
    xq = np.abs(rng.standard_normal((1, 200, hd), dtype=np.float32)) * np.float32(12.8 / hd)
    k = np.tile(np.linspace(0.1, 40, 600, dtype=np.float32)[None, None, :, None], (1, 1, 1, hd))
    c[0], c[2] = R.quantize_rows(k)
    for _ in range(2):
        want, tol = R.prefill(xq, tuple(c), 400, 0, 0.0, True)
        check(forced(kernel, xq, handle(c), 400), want, tol)
        c[0] = -c[0]  # and far below


@pytest.mark.parametrize("kernel", KERNELS)
def test_odd_scales(kernel):
    """Value rows of very different sizes, rows of zeros, and scales of zero."""
    rng = np.random.default_rng(3)
    c = list(R.cache(rng, 1, 2, 400, 128))
    c[3] = (c[3] * 10.0 ** rng.integers(-6, 4, c[3].shape)).astype(np.float32)
    c[0][0, 0, 50:60] = 0
    c[1][0, 1, 70:200] = 0
    c[2][0, 0, 5] = 0
    xq = rng.standard_normal((4, 90, 128), dtype=np.float32) * np.float32(1.5 / np.sqrt(128))
    want, tol = R.prefill(xq, tuple(c), 310, 0, 0.0, True)
    check(forced(kernel, xq, handle(c), 310), want, tol)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("which,bad", [(2, np.nan), (3, np.nan), (2, np.inf)])
@pytest.mark.parametrize("hd", [64, 256])
def test_what_a_row_does_not_see_may_hold_anything(kernel, which, bad, hd):
    """A scale that is no number: the rows before it in the same tile, and those whose window has
    left it behind, are as without it."""
    rng = np.random.default_rng(23)
    c = R.cache(rng, 1, 1, 300, hd)
    xq = rng.standard_normal((2, 200, hd), dtype=np.float32) * np.float32(1 / np.sqrt(hd))
    want, tol = R.prefill(xq, c, 100, 50, 0.0, True)
    for at in (170, 255, 299):
        broken = [t.copy() for t in c]
        broken[which][0, 0, at] = bad
        got = forced(kernel, xq, handle(broken), 100, 50)
        sees = np.array([at <= 100 + i < at + 50 for i in range(200)])
        check(got[~sees], want[~sees], tol)
        if np.isnan(bad):
            assert np.all(np.isnan(got[sees]))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("vs", [1e-18, 1e28])
def test_value_scales(kernel, vs):
    rng = np.random.default_rng(22)
    c = R.cache(rng, 1, 2, 900, 128)
    c[3][:] = vs * rng.uniform(0.5, 2, c[3].shape).astype(np.float32)
    xq = rng.standard_normal((4, 140, 128), dtype=np.float32) * np.float32(0.1)
    want, tol = R.prefill(xq, c, 760, 0, 0.0, True)
    check(forced(kernel, xq, handle(c), 760), want, tol)


@pytest.mark.parametrize("nh,nkv,hd,spos,ntok,slide,cap", [
    (16, 8, 128, 0, 1025, 0, 0.0), (16, 8, 256, 100, 1900, 0, 0.0), (8, 4, 64, 0, 2051, 0, 30.0),
    (8, 4, 256, 0, 2048, 512, 0.0), (6, 4, 128, 7, 2500, 300, 0.0), (8, 1, 256, 2000, 700, 0, 0.0)])
def test_large_chunks(nh, nkv, hd, spos, ntok, slide, cap):
    """The public call; some rows of each head against the plain form."""
    rng = np.random.default_rng(ntok)
    c = R.cache(rng, 1, nkv, spos + ntok, hd)
    xq = rng.standard_normal((nh, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    kv, xo = handle(c), torch.empty((ntok, nh * hd), device="cuda")
    gcu.dev_attention_prefill_i8(xo, dev(xq), kv, spos, slide, cap)
    got = xo.cpu().numpy().reshape(ntok, nh, hd)
    assert np.all(np.isfinite(got))
    both = [forced(k, xq, kv, spos, slide, cap).reshape(ntok, nh, hd) for k in KERNELS]
    vmax = np.max(np.abs(c[1]) * c[3][..., None])
    for h in range(nh):
        for i in {0, 1, 127, 128, ntok // 2 + h, ntok - 2, ntok - 1}:
            hi = spos + i + 1
            lo = max(0, hi - slide) if slide else 0
            k, v = R.rows_of(c, 0, h * nkv // nh, lo, hi)
            want, big = R.attend(xq[h, i], k, v, 1.0, cap)
            tol = R.tolerance(big, hi - lo, vmax)
            for o in (got, *both):
                check(o[i, h], want, tol)
    # every row: the two kernels agree
    assert np.max(np.abs(both[0] - both[1])) <= 2 * R.tolerance(R_SCORE, spos + ntok, vmax)


R_SCORE = 12.0  # above any score of these inputs: |q . k| of 1.5 standard deviations by 4000 keys


@pytest.mark.parametrize("nh,nkv,hd,spos,ntok,cap", [
    (16, 8, 128, 777, 1023, 50.0), (8, 4, 128, 0, 2000, 0.0), (16, 8, 256, 3, 1001, 0.0), (5, 2, 64, 0, 4001, 0.0),
    (4, 1, 64, 50, 4096, 0.0)])
def test_chunks_of_different_lengths(nh, nkv, hd, spos, ntok, cap):
    """Sizes whose long rows are split in two and whose short ones are not: every row of a head
    against the few-row kernel, some against the plain form."""
    rng = np.random.default_rng(ntok)
    c = R.cache(rng, 1, nkv, spos + ntok, hd)
    xq = rng.standard_normal((nh, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    kv = handle(c)
    few, many = (forced(k, xq, kv, spos, 0, cap, extra=8).reshape(ntok, nh, hd) for k in KERNELS)
    xo = torch.full((ntok, nh * hd), 9.0, device="cuda")
    gcu.dev_attention_prefill_i8(xo, dev(xq), kv, spos, 0, cap)
    got = xo.cpu().numpy().reshape(ntok, nh, hd)
    vmax = np.max(np.abs(c[1]) * c[3][..., None])
    tol = R.tolerance(R_SCORE, spos + ntok, vmax)
    assert np.max(np.abs(few - many)) <= 2 * tol and np.max(np.abs(few - got)) <= 2 * tol
    for i in rng.integers(0, ntok, 40):
        h = int(rng.integers(0, nh))
        k, v = R.rows_of(c, 0, h * nkv // nh, 0, spos + i + 1)
        want, big = R.attend(xq[h, i], k, v, 1.0, cap)
        for o in (few, many, got):
            check(o[i, h], want, R.tolerance(big, spos + i + 1, vmax))


def test_the_public_call_is_capturable():
    rng = np.random.default_rng(5)
    c = R.cache(rng, 1, 2, 700, 128)
    for spos, ntok in ((650, 40), (0, 700)):
        xq = rng.standard_normal((4, ntok, 128), dtype=np.float32) * np.float32(0.1)
        kv, q, xo = handle(c), dev(xq), torch.zeros((ntok, 512), device="cuda")
        gcu.dev_attention_prefill_i8(xo, q, kv, spos)
        first = xo.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gcu.dev_attention_prefill_i8(xo, q, kv, spos)
        xo.zero_()
        g.replay()
        assert torch.equal(xo, first)
        want, tol = R.prefill(xq, tuple(t[:, :, :spos + ntok] for t in c), spos, 0, 0.0, True)
        check(first.cpu().numpy(), want, tol)
