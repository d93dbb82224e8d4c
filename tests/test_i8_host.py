"""The 8-bit cache, its attention and sampling without a GPU: argument checks run
before any CUDA call, and the plain forms agree with hand-made cases."""
import ctypes

import numpy as np
import pytest

import gcu
import i8_cases as R

torch = pytest.importorskip("torch")


def kv_struct(nseq=1, nkv=2, clen=16, hdim=64, **over):
    n = nseq * nkv * clen
    codes = torch.zeros(n * hdim + 64, dtype=torch.int8)
    base = (codes.data_ptr() + 15) // 16 * 16
    scales = torch.ones(n + 8)
    c = gcu._KvI8(base, base, scales.data_ptr(), scales.data_ptr(), nkv * clen * hdim, clen * hdim, nkv * clen, clen,
                  nseq, nkv, clen, hdim)
    for k, v in over.items():
        setattr(c, k, v)
    c.keep = (codes, scales)
    return c


def refused(rc, *words):
    assert rc == 1
    msg = gcu.lib().gcu_last_error().decode()
    for w in words:
        assert w in msg, msg


BUF = torch.zeros(4096)
P = (BUF.data_ptr() + 15) // 16 * 16


def write(kv, ld=64 * 8, nh=4, spos=0, ntok=1, xq=P, qkv=P, freqs=P):
    return gcu.lib().gcu_dev_qkv_norm_rope_cache_i8(xq, qkv, ld, ctypes.byref(kv) if kv else None, None, None, 1e-6,
                                                    freqs, 1.0, nh, spos, ntok, None)


@pytest.mark.parametrize("over,words", [
    (dict(hdim=96), ["head size 96"]), (dict(nkv=0), ["0 kv heads"]), (dict(k=None), ["null cache"]),
    (dict(ks=None), ["null cache"]), (dict(kv_stride=24), ["multiples of 16"]), (dict(kv_stride=16), ["overlap"]),
    (dict(sc_stride=3), ["overlap"]), (dict(clen=0), ["0 positions"]), (dict(nseq=2, seq_stride=16), ["overlap"])])
def test_bad_caches_are_refused(over, words):
    kv = kv_struct(**{k: v for k, v in over.items()})
    lib = gcu.lib()
    refused(write(kv), *words)
    refused(lib.gcu_dev_cache_i8_read(P, P, 1 << 20, 1 << 16, ctypes.byref(kv), 0, 1, None), *words)
    refused(lib.gcu_dev_attention_decode_i8(P, P, None, 0, ctypes.byref(kv), None, 1, 4, 0, 1.0, 0.0, None, 0, None),
            *words)


def test_bad_writes_are_refused():
    kv = kv_struct()
    refused(write(None), "null cache")
    refused(write(kv, xq=None), "null pointer")
    refused(write(kv, qkv=P + 4), "16-byte aligned")
    refused(write(kv, ld=64 * 8 + 2), "row stride")
    refused(write(kv, ld=64 * 7), "row stride")
    refused(write(kv, nh=1), "query heads")
    refused(write(kv, spos=16), "outside a cache of 16")
    refused(write(kv, spos=-1), "outside")
    refused(write(kv, ntok=2**31 - 1), "outside")
    refused(write(kv_struct(nseq=2)), "one sequence")
    assert write(kv, ntok=0) == 0
    refused(gcu.lib().gcu_dev_qkv_norm_rope_cache_i8_seqs(P, P, 512, ctypes.byref(kv), None, None, None, 1e-6, P, 1.0, 4,
                                                          None), "null pointer")


def test_bad_reads_are_refused():
    kv = kv_struct()
    read = lambda k, ss, s, spos, n: gcu.lib().gcu_dev_cache_i8_read(k, P, ss, s, ctypes.byref(kv), spos, n, None)
    refused(read(None, 0, 1024, 0, 1), "null pointer")
    refused(read(P, 0, 1024, 10, 7), "outside a cache of 16")
    refused(read(P, 0, 1022, 0, 1), "multiples of 4")
    refused(read(P, 0, 64, 0, 2), "overlap")
    assert read(P, 0, 1024, 0, 0) == 0


def test_bad_decodes_are_refused():
    kv, other = kv_struct(), kv_struct(nkv=1)
    ref = ctypes.byref

    def run(xo=P, xq=P, prefix=None, plen=0, max_len=4, nh=4, slide=0, work=None, nbytes=0):
        return gcu.lib().gcu_dev_attention_decode_i8(xo, xq, ref(prefix) if prefix else None, plen, ref(kv), None,
                                                     max_len, nh, slide, 1.0, 0.0, work, nbytes, None)
    refused(run(xo=None), "null pointer")
    refused(run(xq=P + 4), "16-byte aligned")
    refused(run(max_len=17), "own positions")
    refused(run(max_len=-1), "own positions")
    refused(run(slide=-1), "window")
    refused(run(nh=17), "query heads")
    refused(run(nh=1), "query heads")
    refused(run(plen=3), "null cache")
    refused(run(prefix=other, plen=3), "a prefix of 3")
    refused(run(prefix=kv_struct(), plen=17), "a prefix of 17")
    refused(run(prefix=kv_struct(nseq=2), plen=3), "2 sequences")
    # two key ranges need scratch
    refused(run(prefix=kv_struct(), plen=3), "scratch needed")
    refused(run(prefix=kv_struct(), plen=3, work=P + 4, nbytes=1 << 30), "scratch needed")


def test_bad_prefills_are_refused():
    kv = kv_struct()

    def run(xo=P, xostr=0, xq=P, nh=4, spos=0, ntok=4, slide=0, c=kv):
        return gcu.lib().gcu_dev_attention_prefill_i8(xo, xostr, xq, ctypes.byref(c), nh, spos, ntok, slide, 0.0, 1,
                                                      None, 0, None)
    refused(run(xq=None), "null pointer")
    refused(run(xostr=250), "xostr")
    refused(run(xostr=252), "xostr")
    refused(run(spos=13), "outside a cache of 16")
    refused(run(slide=-2), "window")
    refused(run(nh=20), "query heads")
    refused(run(c=kv_struct(nseq=2)), "2 sequences")
    assert run(ntok=0) == 0


def test_bad_samples_are_refused():
    def run(token=P, logits=P, ld=0, u=P, t=1.0, k=0, p=1.0, minp=0.0, m=1, n=8):
        return gcu.lib().gcu_dev_sample(token, None, logits, ld, u, t, k, p, minp, m, n, None)
    refused(run(token=None), "null pointer")
    refused(run(u=None), "null pointer")
    refused(run(n=0), "logits")
    refused(run(n=(1 << 20) + 1), "logits")
    refused(run(ld=7), "stride 7")
    refused(run(m=-1), "-1 rows")
    for bad in (dict(t=-1.0), dict(t=float("nan")), dict(t=float("inf")), dict(k=-1), dict(p=0.0), dict(p=float("nan")),
                dict(minp=-0.1), dict(minp=1.5), dict(minp=float("nan"))):
        refused(run(**bad), "temperature")
    assert run(m=0) == 0


def test_binding_refuses_wrong_tensors():
    k = torch.zeros((1, 2, 16, 64), dtype=torch.int8)
    s = torch.ones((1, 2, 16))
    gcu.KvCacheI8(k, k, s, s)
    with pytest.raises(gcu.GcuError, match="alike"):
        gcu.KvCacheI8(k, k.float(), s, s)
    with pytest.raises(gcu.GcuError, match="scales"):
        gcu.KvCacheI8(k, k, s[:, :1], s[:, :1])
    with pytest.raises(gcu.GcuError, match="contiguous"):
        t = torch.zeros((1, 16, 2, 64), dtype=torch.int8).transpose(1, 2)
        gcu.KvCacheI8(t, t, s, s)
    kv = gcu.KvCacheI8.empty(3, 2, 8, 64, device="cpu")
    assert kv.seq(1).nseq == 1
    # tensors that are on no CUDA device, or not on the current one, never reach the library
    x = torch.zeros((3, 4, 64))
    with pytest.raises(gcu.GcuError, match="device"):
        gcu.dev_attention_decode_i8(x, x, kv, None, 8, 1.0)
    with pytest.raises(gcu.GcuError, match="device"):
        gcu.dev_attention_prefill_i8(torch.zeros((4, 256)), torch.zeros((4, 4, 64)), kv.seq(0), 0)
    with pytest.raises(gcu.GcuError, match="device"):
        gcu.dev_cache_i8_read(torch.zeros((3, 2, 4, 64)), torch.zeros((3, 2, 4, 64)), kv, 0)
    with pytest.raises(gcu.GcuError, match="device"):
        gcu.dev_sample(torch.zeros(1, dtype=torch.int32), torch.zeros((1, 8)), torch.zeros(1))
    with pytest.raises(gcu.GcuError, match="device"):
        gcu.dev_qkv_norm_rope_cache_i8(torch.zeros((4, 1, 64)), torch.zeros((1, 512)), kv.seq(0), torch.zeros((1, 64)), 0)


def test_plain_forms():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 64), dtype=np.float32)
    x[1] = 0
    q, s = R.quantize_rows(x)
    assert np.max(np.abs(q)) == 127 and s[1] == 1 and not q[1].any()
    assert np.all(np.abs(q * s[:, None] - x) <= s[:, None] * 0.5001)
    # softmax over equal scores is the mean of the values; an empty row is zero
    c = R.cache(rng, 1, 1, 8, 64)
    out, _ = R.decode(np.zeros((1, 1, 64), np.float32), c, [5], 1.0, 0.0, 0)
    assert np.allclose(out[0, 0], R.rows_of(c, 0, 0, 0, 5)[1].mean(0))
    out, _ = R.decode(np.zeros((1, 1, 64), np.float32), c, [0], 1.0, 0.0, 0)
    assert not out.any()
    # a window of 3 over a prefix of 4 and 2 own positions: one of the prefix, two own
    out, _ = R.decode(np.zeros((1, 1, 64), np.float32), c, [2], 1.0, 0.0, 3, c, 4)
    v = R.rows_of(c, 0, 0, 0, 8)[1]
    assert np.allclose(out[0, 0], (v[3] + v[0] + v[1]) / 3)
    # sampling: index order, ties to the lowest index
    assert R.sample([1, 3, 3, 0], 0.0, 1.0, 1, 1.0, 0.0)[0] == 1
    assert R.sample([0, 0, 0, 0], 0.49, 1.0, 2, 1.0, 0.0) == (0, 0.5)
    assert R.sample([0, 0, 0, 0], 0.5, 1.0, 2, 1.0, 0.0) == (1, 0.5)
    assert R.sample([np.nan, -np.inf], 0.3, 1.0, 0, 1.0, 0.0) == (-1, 0.0)


def test_scratch_of_unusable_caches_is_zero():
    """The scratch queries answer 0 for what the calls refuse; they never divide by a count of zero."""
    lib, ref = gcu.lib(), ctypes.byref
    for over in (dict(nseq=0), dict(nkv=0), dict(nseq=-3), dict(nkv=-1)):
        bad = kv_struct()
        for k, v in over.items():
            setattr(bad, k, v)
        assert lib.gcu_attention_decode_i8_work(None, 0, ref(bad), 16, 4, 0) == 0
        assert lib.gcu_attention_decode_i8_work(ref(bad), 8, ref(bad), 16, 4, 0) == 0
        if "nkv" in over:
            assert lib.gcu_attention_prefill_i8_work(ref(bad), 4, 0, 4, 0, 0.0, 1) == 0
    kv = kv_struct()
    assert lib.gcu_attention_decode_i8_work(None, 0, None, 16, 4, 0) == 0
    assert lib.gcu_attention_decode_i8_work(None, 0, ref(kv), 16, 0, 0) == 0
    assert lib.gcu_attention_decode_i8_work(None, -5, ref(kv), -7, 4, -1) == 0
    assert lib.gcu_attention_prefill_i8_work(ref(kv), 0, 0, 4, 0, 0.0, 1) == 0
    assert lib.gcu_attention_prefill_i8_work(ref(kv), 4, -1, 4, 0, 0.0, 1) == 0
    assert lib.gcu_attention_prefill_i8_work(ref(kv), 4, 0, 0, 0, 0.0, 1) == 0


def test_outputs_over_their_inputs_are_refused():
    """Rows are read by several CTAs while others are written."""
    kv = kv_struct()
    lib, ref = gcu.lib(), ctypes.byref
    refused(write(kv, xq=P + 64), "overlap")
    for xo, xq in ((P, P), (P, P + 4 * 64 * 4 - 16), (P + 16, P)):
        refused(lib.gcu_dev_attention_decode_i8(xo, xq, None, 0, ref(kv), None, 4, 4, 0, 1.0, 0.0, None, 0, None), "overlap")
    refused(lib.gcu_dev_attention_prefill_i8(P, 0, P + 64, ref(kv), 4, 0, 3, 0, 0.0, 1, None, 0, None), "overlap")
    refused(lib.gcu_dev_cache_i8_read(P, P, 0, 1024, ref(kv), 0, 1, None), "overlap")
