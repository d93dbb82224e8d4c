"""Attention over the 8-bit KV cache against the 64-bit plain form (tolerance
derived in i8_cases.tolerance), at the lengths, masks and layouts where it can go
wrong."""
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


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def handle(c):
    return gcu.KvCacheI8(*(dev(t) for t in c))


def check(got, want, tol):
    got = got.cpu().numpy() if torch.is_tensor(got) else got
    assert np.all(np.isfinite(got))
    err = np.max(np.abs(got - want))
    assert err <= tol, f"max error {err:.3g}, allowed {tol:.3g}"


def run_decode(xq, kv, lens, max_len, cap=0.0, slide=0, prefix=None, plen=0):
    xo = torch.full(xq.shape, 9.0, device="cuda")
    n = dev(np.asarray(lens, np.int32)) if lens is not None else None
    gcu.dev_attention_decode_i8(xo, dev(xq), kv, n, max_len, xq.shape[-1] ** -0.5, cap, slide, prefix, plen)
    torch.cuda.synchronize()
    return xo


@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 256), (8, 4, 256), (16, 8, 128), (8, 1, 64), (8, 1, 256), (6, 4, 128),
                                       (3, 3, 64), (5, 2, 256)])
@pytest.mark.parametrize("n", [1, 2, 31, 33, 65, 700])
def test_decode_one_sequence(nh, nkv, hd, n):
    rng = np.random.default_rng(n)
    c = R.cache(rng, 1, nkv, n + 3, hd)
    xq = rng.standard_normal((1, nh, hd), dtype=np.float32) * 1.5
    want, tol = R.decode(xq, c, [n], hd ** -0.5, 0.0, 0)
    check(run_decode(xq, handle(c), None, n), want, tol)


@pytest.mark.parametrize("slide,cap", [(0, 0.0), (1, 0.0), (64, 0.0), (100, 20.0), (5000, 0.0), (0, 5.0)])
def test_decode_windows_and_cap(slide, cap):
    rng = np.random.default_rng(slide + 7)
    c = R.cache(rng, 1, 2, 2500, 128)
    xq = rng.standard_normal((1, 8, 128), dtype=np.float32) * 2
    want, tol = R.decode(xq, c, [2497], 128 ** -0.5, cap, slide)
    check(run_decode(xq, handle(c), [2497], 2500, cap, slide), want, tol)


@pytest.mark.parametrize("nh,nkv,hd,plen,slide,cap", [
    (4, 1, 256, 1, 0, 0.0), (8, 4, 256, 130, 0, 0.0), (16, 8, 64, 64, 0, 30.0), (8, 1, 128, 777, 50, 0.0),
    (6, 4, 256, 63, 0, 0.0), (8, 4, 128, 500, 505, 0.0), (4, 4, 64, 129, 100, 0.0), (8, 1, 256, 300, 0, 0.0)])
@pytest.mark.parametrize("nseq", [1, 2, 5, 19])
def test_decode_shared_prefix(nh, nkv, hd, plen, slide, cap, nseq):
    rng = np.random.default_rng(plen + nseq)
    lens = [(0, 17, 1, -1, 40, 33, 64, 65)[b % 8] for b in range(nseq)]
    pre, own = R.cache(rng, 1, nkv, plen + 2, hd), R.cache(rng, nseq, nkv, 70, hd)
    xq = rng.standard_normal((nseq, nh, hd), dtype=np.float32) * 1.5
    want, tol = R.decode(xq, own, lens, hd ** -0.5, cap, slide, pre, plen)
    got = run_decode(xq, handle(own), lens, 70, cap, slide, handle(pre), plen).cpu().numpy()
    live = np.asarray(lens) >= 0
    assert np.all(got[~live] == 9.0)  # skipped rows are left as they were
    check(got[live], want[live], tol)


def test_decode_many_rows_of_one_prefix():
    """More (sequence, head) rows than one query tile holds, and a prefix cut into many chunks."""
    rng = np.random.default_rng(11)
    pre, own = R.cache(rng, 1, 2, 1500, 64), R.cache(rng, 40, 2, 9, 64)
    lens = [b % 10 for b in range(40)]
    xq = rng.standard_normal((40, 16, 64), dtype=np.float32)
    want, tol = R.decode(xq, own, lens, 0.125, 0.0, 0, pre, 1500)
    check(run_decode(xq, handle(own), lens, 9, prefix=handle(pre), plen=1500), want, tol)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("plen", [63, 129, 700, 705])
def test_decode_long_chunks(hd, plen):
    """More query tiles than SMs: each walks the whole prefix; scores grow along it in half the rows."""
    rng = np.random.default_rng(plen)
    nseq = 150 * 128 // 8
    pre = list(R.cache(rng, 1, 1, plen, hd))
    pre[2][0, 0] *= np.linspace(0.5, 6, plen, dtype=np.float32)
    xq = rng.standard_normal((nseq, 8, hd), dtype=np.float32)
    xq[::2] *= np.float32(3)
    own = gcu.KvCacheI8.empty(nseq, 1, 1, hd)
    lens = dev(np.zeros(nseq, np.int32))
    xo = torch.full(xq.shape, 9.0, device="cuda")
    gcu.dev_attention_decode_i8(xo, dev(xq), own, lens, 1, hd ** -0.5, 0.0, 0, handle(pre), plen)
    some = np.r_[0:40, 1000:1016, nseq - 24:nseq]
    want, tol = R.decode(xq[some], tuple(np.zeros((len(some), 1, 1, hd), np.int8) if i < 2 else
                                         np.ones((len(some), 1, 1), np.float32) for i in range(4)),
                         [0] * len(some), hd ** -0.5, 0.0, 0, tuple(pre), plen)
    check(xo[torch.from_numpy(some).cuda()], want, tol)


def test_decode_sees_nothing():
    rng = np.random.default_rng(3)
    own = R.cache(rng, 3, 1, 8, 64)
    xq = rng.standard_normal((3, 2, 64), dtype=np.float32)
    got = run_decode(xq, handle(own), [0, -1, 2], 8).cpu().numpy()
    assert not got[0].any() and np.all(got[1] == 9.0) and got[2].any()
    assert not run_decode(xq, handle(own), None, 0).cpu().numpy().any()


def test_decode_masked_places_may_hold_anything():
    """NaN and infinite scales outside a window, and past the last position, do not show."""
    rng = np.random.default_rng(4)
    pre, own = R.cache(rng, 1, 2, 200, 128), R.cache(rng, 3, 2, 80, 128)
    lens, slide = [5, 70, 64], 100
    xq = rng.standard_normal((3, 4, 128), dtype=np.float32)
    want, tol = R.decode(xq, own, lens, 128 ** -0.5, 0.0, slide, pre, 190)
    for b, n in enumerate(lens):
        own[2][b, :, n:], own[3][b, :, n:] = np.nan, np.inf
    pre[2][:, :, 190:], pre[3][:, :, 190:] = np.inf, np.nan
    pre[2][:, :, :95], pre[3][:, :, :95] = np.nan, -np.inf  # before every window
    check(run_decode(xq, handle(own), lens, 80, 0.0, slide, handle(pre), 190), want, tol)


def test_decode_nan_shows_where_it_is_seen():
    rng = np.random.default_rng(5)
    own = R.cache(rng, 2, 1, 64, 64)
    own[2][1, 0, 3] = np.nan
    xq = rng.standard_normal((2, 2, 64), dtype=np.float32)
    got = run_decode(xq, handle(own), [64, 64], 64).cpu().numpy()
    assert np.all(np.isfinite(got[0])) and np.all(np.isnan(got[1]))


def test_decode_extreme_scales():
    """Value rows of very different size, and scores far apart."""
    rng = np.random.default_rng(6)
    own = R.cache(rng, 1, 1, 300, 128)
    own[3][0, 0] *= (10.0 ** rng.uniform(-15, 15, 300)).astype(np.float32)
    own[2][0, 0, ::7] *= 30
    xq = rng.standard_normal((1, 4, 128), dtype=np.float32)
    want, tol = R.decode(xq, own, [300], 128 ** -0.5, 0.0, 0)
    check(run_decode(xq, handle(own), None, 300), want, tol)
    xq[:] = 0  # all scores equal
    want, tol = R.decode(xq, own, [300], 128 ** -0.5, 0.0, 0)
    check(run_decode(xq, handle(own), None, 300), want, tol)


def test_decode_length_past_the_cache_is_reported():
    rng = np.random.default_rng(7)
    own = R.cache(rng, 2, 1, 8, 64)
    xq = rng.standard_normal((2, 1, 64), dtype=np.float32)
    got = run_decode(xq, handle(own), [9, 8], 8).cpu().numpy()
    with pytest.raises(gcu.GcuError, match="length outside"):
        gcu.check_device()
    want, tol = R.decode(xq, own, [-1, 8], 0.125, 0.0, 0)
    assert np.all(got[0] == 9.0)
    check(got[1], want[1], tol)


def run_prefill(xq, kv, spos, slide=0, cap=0.0, mask=True, extra=0):
    nh, ntok, hd = xq.shape
    xo = torch.full((ntok, nh * hd + extra), 9.0, device="cuda")
    gcu.dev_attention_prefill_i8(xo, dev(xq), kv, spos, slide, cap, mask)
    torch.cuda.synchronize()
    got = xo.cpu().numpy()
    assert np.all(got[:, nh * hd:] == 9.0)
    return got[:, :nh * hd]


@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 256), (8, 4, 256), (4, 2, 128), (6, 4, 64), (8, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("spos,ntok,slide,cap,mask", [
    (0, 1, 0, 0.0, True), (0, 2, 0, 0.0, True), (0, 33, 0, 0.0, True), (63, 65, 0, 0.0, True), (5, 130, 0, 0.0, True),
    (100, 70, 20, 0.0, True), (0, 129, 64, 0.0, True), (0, 150, 1, 0.0, True), (7, 60, 0, 4.0, True),
    (13, 67, 0, 0.0, False), (200, 9, 0, 0.0, True)])
def test_prefill(nh, nkv, hd, spos, ntok, slide, cap, mask):
    rng = np.random.default_rng(spos + ntok)
    c = R.cache(rng, 1, nkv, spos + ntok + 1, hd)
    c[2][0, :, -1], c[3][0, :, -1] = np.nan, np.nan  # behind the chunk
    xq = rng.standard_normal((nh, ntok, hd), dtype=np.float32) * np.float32(1.5 / np.sqrt(hd))
    want, tol = R.prefill(xq, tuple(t[:, :, :spos + ntok] for t in c), spos, slide, cap, mask)
    check(run_prefill(xq, handle(c), spos, slide, cap, mask, extra=4), want, tol)


def test_prefill_long_and_sliding():
    rng = np.random.default_rng(1)
    c = R.cache(rng, 1, 1, 1300, 128)
    xq = rng.standard_normal((2, 500, 128), dtype=np.float32) * np.float32(2 / np.sqrt(128))
    for slide in (0, 256, 700):
        want, tol = R.prefill(xq, c, 800, slide, 0.0, True)
        check(run_prefill(xq, handle(c), 800, slide), want, tol)


def test_prefill_growing_scores():
    """Each later key scores far above the ones before it: the running maximum moves all the time."""
    rng = np.random.default_rng(2)
    c = list(R.cache(rng, 1, 1, 400, 64))
    xq = np.abs(rng.standard_normal((1, 200, 64), dtype=np.float32)) * np.float32(0.2)
    k = np.tile(np.linspace(0.1, 40, 400, dtype=np.float32)[None, None, :, None], (1, 1, 1, 64))
    c[0], c[2] = R.quantize_rows(k)
    want, tol = R.prefill(xq, tuple(c), 200, 0, 0.0, True)
    check(run_prefill(xq, handle(c), 200), want, tol)
    c[0] = -c[0]  # and far below
    want, tol = R.prefill(xq, tuple(c), 200, 0, 0.0, True)
    check(run_prefill(xq, handle(c), 200), want, tol)


def test_prefill_rows_equal_decode():
    """A chunk's last token attends as one decode step does."""
    rng = np.random.default_rng(8)
    c = R.cache(rng, 1, 4, 900, 256)
    xq = rng.standard_normal((8, 40, 256), dtype=np.float32) / np.float32(16)
    kv = handle(c)
    a = run_prefill(xq, kv, 860)[-1].reshape(8, 256)
    b = run_decode(xq[None, :, -1] * np.float32(16), kv, None, 900).cpu().numpy()[0]
    _, tol = R.decode(xq[None, :, -1] * np.float32(16), c, [900], 1 / 16, 0.0, 0)
    check(a, b, 2 * tol)


def test_graph_replay_and_two_graphs():
    """Captured calls own their scratch: two graphs replayed in turn, lengths changed between."""
    rng = np.random.default_rng(9)
    own, pre = R.cache(rng, 4, 2, 64, 128), R.cache(rng, 1, 2, 500, 128)
    kv, pkv = handle(own), handle(pre)
    xq = rng.standard_normal((4, 8, 128), dtype=np.float32)
    q = dev(xq)
    outs, graphs, lens = [], [], []
    for i in range(2):
        xo, n = torch.empty_like(q), dev(np.array([1, 2, 3, 4], np.int32))
        outs.append(xo)
        lens.append(n)
        call = lambda: gcu.dev_attention_decode_i8(xo, q, kv, n, 64, 128 ** -0.5, 0.0, 0, pkv, 500 - 100 * i)
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for round_ in range(3):
        for i in range(2):
            lens[i].copy_(torch.tensor([10 * round_ + 1, 5, 0, 64], dtype=torch.int32))
            graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        want, tol = R.decode(xq, own, [21, 5, 0, 64], 128 ** -0.5, 0.0, 0, pre, 500 - 100 * i)
        check(outs[i], want, tol)


def test_side_stream():
    rng = np.random.default_rng(10)
    c = R.cache(rng, 1, 1, 3000, 64)
    kv, xq = handle(c), rng.standard_normal((1, 4, 64), dtype=np.float32)
    q, xo, s = dev(xq), torch.empty((1, 4, 64), device="cuda"), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        gcu.dev_attention_decode_i8(xo, q, kv, None, 3000, 0.125, stream=s)
        torch.empty(1 << 20, device="cuda").fill_(3.0)  # the call's scratch is not reused under it
    s.synchronize()
    want, tol = R.decode(xq, c, [3000], 0.125, 0.0, 0)
    check(xo, want, tol)


def same_rows(nseq, nkv, clen, hd):
    """A cache whose rows are all alike, codes at 127, but for a first key a little larger: every
    other weight is 0.997 of the largest, so that its leading byte is 255."""
    c = gcu.KvCacheI8.empty(nseq, nkv, clen, hd, "cuda")
    c.k.fill_(127)
    c.v.fill_(127)
    c.ks.fill_(1.5 / 127)
    c.ks[:, :, 0] = 1.503 / 127
    c.vs.fill_(0.5)
    return c


@pytest.mark.parametrize("shared", [False, True])
def test_decode_sums_of_very_long_ranges(shared):
    """More rows than there are SMs, so that one CTA could take a whole range, over a cache
    longer than a 32-bit sum of byte products holds (66,312 keys of 255*127)."""
    hd, n = 64, 70001
    if shared:
        nseq, nh, nkv = 592, 8, 1
        pre, own = same_rows(1, nkv, n, hd), same_rows(nseq, nkv, 4, hd)
        length = torch.zeros(nseq, dtype=torch.int32, device="cuda")
    else:
        nseq, nh, nkv = 149, 1, 1
        pre, own, length = None, same_rows(nseq, nkv, n, hd), torch.full((nseq,), n, dtype=torch.int32, device="cuda")
    xq = torch.full((nseq, nh, hd), 1.0 / hd, device="cuda")
    xo = torch.empty_like(xq)
    gcu.dev_attention_decode_i8(xo, xq, own, length, own.k.shape[2], 1.0, 0.0, 0, pre, n if shared else 0)
    # The mean of equal rows.  fp32 sums of at most 128 equal weights in a row, each step off by half a
    # step of the sum so far: 64 * 2^-24 of the total; 20 for the few sums that join them and the division.
    check(xo, np.full(xq.shape, 63.5), 63.5 * 84 * 2.0 ** -24)


def test_two_streams_at_once():
    """Decode and prefill of two streams, each with scratch of its own."""
    rng = np.random.default_rng(12)
    c = R.cache(rng, 2, 2, 5000, 128)
    xq = rng.standard_normal((2, 8, 128), dtype=np.float32)
    xp = rng.standard_normal((8, 40, 128), dtype=np.float32)
    kv, q, p = handle(c), dev(xq), dev(xp)
    want, tol = R.decode(xq, c, [4999, 3000], 128 ** -0.5, 0.0, 0)
    wantp, tolp = R.prefill(xp, [t[:1] for t in c], 4960, 0, 0.0, True)
    length = dev(np.asarray([4999, 3000], np.int32))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                xo, po = torch.empty_like(q), torch.empty((40, 8 * 128), device="cuda")
                gcu.dev_attention_decode_i8(xo, q, kv, length, 5000, 128 ** -0.5)
                gcu.dev_attention_prefill_i8(po, p, kv.seq(0), 4960)
                outs.append((xo, po))
    torch.cuda.synchronize()
    for xo, po in outs:
        check(xo, want, tol)
        check(po, wantp, tolp)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 256), (6, 4, 64), (4, 2, 128)])
@pytest.mark.parametrize("max_len", [130, 513, 900, 1024])
def test_decode_few_chunks(nh, nkv, hd, max_len):
    """Two to eight chunks, joined in the launch that makes them: lengths that end in the first
    chunk, between chunks, and in the last; skipped sequences; empty ones."""
    rng = np.random.default_rng(max_len)
    lens = [max_len, 0, -1, 1, 128, 129, max_len - 1, 7]
    c = R.cache(rng, len(lens), nkv, max_len, hd)
    xq = rng.standard_normal((len(lens), nh, hd), dtype=np.float32)
    live = np.asarray(lens) >= 0
    for slide, cap in ((0, 0.0), (140, 0.0), (0, 8.0)):
        want, tol = R.decode(xq, c, lens, hd ** -0.5, cap, slide)
        got = run_decode(xq, handle(c), lens, max_len, cap, slide).cpu().numpy()
        assert np.all(got[~live] == 9.0) and np.all(got[np.asarray(lens) == 0] == 0.0)
        check(got[live], want[live], tol)


@pytest.mark.parametrize("vs", [1e-18, 1e-12, 1e12, 1e28])
def test_all_value_scales_small_or_large(vs):
    rng = np.random.default_rng(21)
    own = R.cache(rng, 1, 2, 3000, 128)
    own[3][:] = vs * rng.uniform(0.5, 2, own[3].shape).astype(np.float32)
    xq = rng.standard_normal((1, 4, 128), dtype=np.float32)
    want, tol = R.decode(xq, own, [3000], 128 ** -0.5, 0.0, 0)
    check(run_decode(xq, handle(own), None, 3000), want, tol)
    xp = rng.standard_normal((4, 50, 128), dtype=np.float32) * np.float32(0.1)
    want, tol = R.prefill(xp, own, 2950, 0, 0.0, True)
    check(run_prefill(xp, handle(own), 2950), want, tol)
