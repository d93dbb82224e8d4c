"""The 8-bit KV cache on the GPU: codes, scales and rows bit for bit against the
plain form, rows outside the call left as they were, refusals."""
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


def filled(nseq, nkv, clen, hd, strided=False):
    """A cache of code 77, scale 7; strided: views into larger buffers."""
    pad = 3 if strided else 0
    codes = torch.full((2, nseq, nkv + pad, clen + pad, hd), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((2, nseq, nkv + pad, clen + pad + 1), 7.0, device="cuda")
    c, s = codes[:, :, :nkv, :clen], scales[:, :, :nkv, :clen]
    return gcu.KvCacheI8(c[0], c[1], s[0], s[1]), codes, scales


CASES = [(4, 1, 256, 1, 5), (8, 4, 256, 33, 0), (16, 8, 128, 7, 100), (6, 4, 64, 19, 2), (1, 1, 64, 1, 0)]


@pytest.mark.parametrize("nh,nkv,hd,ntok,spos", CASES)
@pytest.mark.parametrize("norm", [True, False])
def test_chunk_is_bit_exact(nh, nkv, hd, ntok, spos, norm):
    rng = np.random.default_rng(nh * 100 + ntok)
    ld = (nh + 2 * nkv) * hd + 12  # rows longer than the projection
    x = rng.standard_normal((ntok, ld), dtype=np.float32)
    x[ntok // 2, (nh + nkv) * hd:(nh + nkv + 1) * hd] = 0  # a value row of zeros
    nq, nk = ((rng.standard_normal(hd) * 0.1).astype(np.float32) for _ in range(2)) if norm else (None, None)
    fr, qs = R.tables(np.arange(spos, spos + ntok), hd), float(np.float32(1 / np.sqrt(hd)))
    kv, codes, scales = filled(1, nkv, spos + ntok + 4, hd, strided=True)
    before = codes.clone(), scales.clone()
    xq = torch.full((nh, ntok, hd), 9.0, device="cuda")
    w = lambda a: dev(a) if a is not None else None
    gcu.dev_qkv_norm_rope_cache_i8(xq, dev(x), kv, dev(fr), spos, qs, w(nq), w(nk), 1e-6)
    rows = x[:, :(nh + 2 * nkv) * hd].reshape(ntok, -1, hd)
    f = fr[:, None]
    assert np.array_equal(xq.cpu().numpy(), R.norm_rope(rows[:, :nh], nq, 1e-6, f, qs).transpose(1, 0, 2))
    k, ks = R.quantize_rows(R.norm_rope(rows[:, nh:nh + nkv], nk, 1e-6, f, 1.0))
    v, vs = R.quantize_rows(rows[:, nh + nkv:])
    at = (0, slice(None), slice(spos, spos + ntok))
    for got, want in ((kv.k, k), (kv.v, v), (kv.ks, ks), (kv.vs, vs)):
        assert np.array_equal(got[at].cpu().numpy(), np.moveaxis(want, 0, 1))
    assert vs[ntok // 2, 0] == 1
    # everything else in the buffers is as it was
    for t in (kv.k, kv.v, kv.ks, kv.vs):
        t[at] = 77 if t.dtype == torch.int8 else 7.0
    assert torch.equal(codes, before[0]) and torch.equal(scales, before[1])


@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 256), (4, 1, 128), (6, 4, 64)])
def test_sequences_are_bit_exact(nh, nkv, hd):
    rng = np.random.default_rng(nh)
    clen, lens = 21, np.array([1, 21, 7, 0, -3, 20], np.int32)
    n = len(lens)
    x = rng.standard_normal((n, (nh + 2 * nkv) * hd), dtype=np.float32)
    nq, nk = ((rng.standard_normal(hd) * 0.1).astype(np.float32) for _ in range(2))
    fr = R.tables(1000 + np.maximum(lens, 0), hd)
    kv, codes, scales = filled(n, nkv, clen, hd)
    xq = torch.full((n, nh, hd), 9.0, device="cuda")
    gcu.dev_qkv_norm_rope_cache_i8_seqs(xq, dev(x), kv, dev(lens), dev(fr), 1.0, dev(nq), dev(nk), 1e-6)
    rows, f = x.reshape(n, -1, hd), fr[:, None]
    q = R.norm_rope(rows[:, :nh], nq, 1e-6, f, 1.0)
    k, ks = R.quantize_rows(R.norm_rope(rows[:, nh:nh + nkv], nk, 1e-6, f, 1.0))
    v, vs = R.quantize_rows(rows[:, nh + nkv:])
    q[lens < 1] = 9.0  # skipped rows
    assert np.array_equal(xq.cpu().numpy(), q)
    want = {"k": np.full((n, nkv, clen, hd), 77, np.int8), "ks": np.full((n, nkv, clen), 7, np.float32)}
    want["v"], want["vs"] = want["k"].copy(), want["ks"].copy()
    for b, m in enumerate(lens):
        if m > 0:
            want["k"][b, :, m - 1], want["ks"][b, :, m - 1] = k[b], ks[b]
            want["v"][b, :, m - 1], want["vs"][b, :, m - 1] = v[b], vs[b]
    for name, t in want.items():
        assert np.array_equal(getattr(kv, name).cpu().numpy(), t), name


def test_length_past_the_cache_is_reported():
    kv, codes, scales = filled(2, 1, 8, 64)
    x, fr = torch.randn((2, 3 * 64), device="cuda"), torch.ones((2, 64), device="cuda")
    xq = torch.full((2, 1, 64), 9.0, device="cuda")
    gcu.dev_qkv_norm_rope_cache_i8_seqs(xq, x, kv, torch.tensor([9, 8], dtype=torch.int32, device="cuda"), fr)
    with pytest.raises(gcu.GcuError, match="length outside"):
        gcu.check_device()
    gcu.check_device()  # reported once
    assert bool((kv.k[0] == 77).all()) and bool((xq[0] == 9).all())
    assert bool((kv.k[1, :, 7] != 77).any()) and bool((kv.k[1, :, :7] == 77).all())


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_read_back(hd):
    rng = np.random.default_rng(hd)
    c = R.cache(rng, 3, 2, 40, hd)
    kv = gcu.KvCacheI8(*map(dev, (c[0], c[1], c[2], c[3])))
    # into the middle of an fp32 cache
    k = torch.full((3, 2, 64, hd), 5.0, device="cuda")
    v = k.clone()
    gcu.dev_cache_i8_read(k[:, :, 10:33], v[:, :, 10:33], kv, 17)
    for got, q, s in ((k, c[0], c[2]), (v, c[1], c[3])):
        want = np.full(got.shape, 5.0, np.float32)
        want[:, :, 10:33] = q[:, :, 17:].astype(np.float32) * s[:, :, 17:, None]
        assert np.array_equal(got.cpu().numpy(), want)


def test_capture_and_other_stream():
    """A captured write replays with new lengths; a call on a side stream is ordered by it."""
    kv, _, _ = filled(2, 1, 8, 64)
    x, fr = torch.randn((2, 3 * 64), device="cuda"), torch.from_numpy(R.tables([3, 4], 64)).cuda()
    xq, n = torch.zeros((2, 1, 64), device="cuda"), torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    gcu.dev_qkv_norm_rope_cache_i8_seqs(xq, x, kv, n, fr)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gcu.dev_qkv_norm_rope_cache_i8_seqs(xq, x, kv, n, fr)
        n.add_(1)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for b, (lo, hi) in enumerate([(0, 3), (1, 4)]):
        for t in range(lo, hi):
            assert torch.equal(kv.k[b, :, t], kv.k[b, :, lo])
        assert bool((kv.k[b, :, hi:] == 77).all())
    s = torch.cuda.Stream()
    out = torch.empty((2, 1, 8, 64), device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    gcu.dev_cache_i8_read(out, torch.empty_like(out), kv, 0, stream=s)
    s.synchronize()
    assert torch.equal(out, kv.k.float() * kv.ks.unsqueeze(-1))


def test_odd_strides_of_single_rows():
    """A stride along a dimension of one is never taken, whatever it is."""
    rng = np.random.default_rng(31)
    x = rng.standard_normal((6 * 64,), dtype=np.float32)
    kv = gcu.KvCacheI8.empty(1, 1, 5, 64)
    qkv = torch.as_strided(dev(x), (1, 6 * 64), (7, 1))
    xq, fr = torch.empty((4, 1, 64), device="cuda"), R.tables([3], 64)
    gcu.dev_qkv_norm_rope_cache_i8(xq, qkv, kv, dev(fr), 3)
    k, ks = R.quantize_rows(R.norm_rope(x.reshape(6, 64)[4:5], None, 1e-6, fr, 1.0))
    assert np.array_equal(kv.k[0, :, 3].cpu().numpy(), k) and np.array_equal(kv.ks[0, :, 3].cpu().numpy(), ks)
    out = torch.zeros((2, 1 * 64), device="cuda")
    rk, rv = (torch.as_strided(o, (1, 1, 1, 64), (5, 3, 64, 1)) for o in out)
    gcu.dev_cache_i8_read(rk, rv, kv, 3)
    assert np.array_equal(out[0].cpu().numpy(), k[0] * ks[0])
    xo = torch.as_strided(torch.zeros(4 * 64, device="cuda"), (1, 4 * 64), (1, 1))
    gcu.dev_attention_prefill_i8(xo, xq, kv, 3, slide=1)
    v, vs = R.quantize_rows(x.reshape(6, 64)[5])
    assert np.allclose(xo.cpu().numpy().reshape(4, 64), v * vs, rtol=2.0 ** -20, atol=0)


def test_offsets_past_32_bits():
    """The last head of a cache whose heads begin 4.8 GB in: write, read back, and both kinds of
    attention over a window at its end."""
    nkv, clen, hd, nh, n = 3, 9_400_003, 256, 3, 40
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("24 GB of device memory needed")
    rng = np.random.default_rng(32)
    codes = torch.empty((2, 1, nkv, clen, hd), dtype=torch.int8, device="cuda")
    scales = torch.empty((2, 1, nkv, clen), device="cuda")
    kv = gcu.KvCacheI8(codes[0], codes[1], scales[0], scales[1])
    spos = clen - n
    x = rng.standard_normal((n, (nh + 2 * nkv) * hd), dtype=np.float32)
    fr = R.tables(np.arange(n), hd)  # angles small enough to be exact
    xq = torch.empty((nh, n, hd), device="cuda")
    gcu.dev_qkv_norm_rope_cache_i8(xq, dev(x), kv, dev(fr), spos, hd ** -0.5)
    rows = x.reshape(n, -1, hd)
    k, ks = R.quantize_rows(R.norm_rope(rows[:, nh:nh + nkv], None, 1e-6, fr[:, None], 1.0))
    v, vs = R.quantize_rows(rows[:, nh + nkv:])
    small = tuple(np.moveaxis(t, 0, 1)[None] for t in (k, v, ks, vs))
    assert np.array_equal(kv.k[0, :, spos:].cpu().numpy(), small[0][0])
    rk, rv = (torch.empty((1, nkv, n, hd), device="cuda") for _ in range(2))
    gcu.dev_cache_i8_read(rk, rv, kv, spos)
    assert np.array_equal(rv.cpu().numpy(), small[1] * small[3][..., None])
    q = xq.cpu().numpy()
    xo = torch.empty((n, nh * hd), device="cuda")
    gcu.dev_attention_prefill_i8(xo, xq, kv, spos, slide=8)
    want, tol = R.prefill(q[:, 8:], small, 8, 8, 0.0, True)
    assert np.max(np.abs(xo.cpu().numpy()[8:] - want)) <= tol
    one = torch.empty((1, nh, hd), device="cuda")
    gcu.dev_attention_decode_i8(one, xq[:, -1][None].contiguous(), kv, None, clen, 1.0, 0.0, n)
    want, tol = R.decode(q[None, :, -1], small, [n], 1.0, 0.0, 0)
    assert np.max(np.abs(one.cpu().numpy() - want)) <= tol
