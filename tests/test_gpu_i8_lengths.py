"""Sequences that run past their 8-bit caches: who is told, and what is left alone."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import gcu  # noqa: E402
import oracle  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    gcu.init(0)
    yield
    gcu.check_device()


def too_long(op):
    """One of two sequences is a position too long for its cache of 8."""
    kv = gcu.KvCacheI8.empty(2, 1, 8, 64)
    n = torch.tensor([9, 3], dtype=torch.int32, device="cuda")
    if op == "write":
        gcu.dev_qkv_norm_rope_cache_i8_seqs(torch.empty((2, 1, 64), device="cuda"), torch.randn((2, 3 * 64), device="cuda"),
                                            kv, n, torch.ones((2, 64), device="cuda"))
    else:
        gcu.dev_attention_decode_i8(torch.empty((2, 1, 64), device="cuda"), torch.randn((2, 1, 64), device="cuda"), kv, n,
                                    8, 0.125)
    torch.cuda.synchronize()


@pytest.mark.parametrize("op", ["write", "decode"])
def test_a_length_error_is_not_the_next_matmuls(op):
    """Host calls report their own waits; the length waits for gcu_check_device."""
    rng = np.random.default_rng(8)
    w, x = rng.integers(-127, 128, (48, 64)).astype(np.int8), rng.integers(-127, 128, (16, 64)).astype(np.int8)
    ws, xs = rng.random(48).astype(np.float32), rng.random(16).astype(np.float32)
    want = oracle.gemm_int8(w, ws, x, xs)
    too_long(op)
    assert np.array_equal(gcu.gemm_int8(w, ws, x, xs), want)  # 16 rows: the GEMM kernel
    assert np.array_equal(gcu.gemv_int8(w, ws, x[0], xs[0]), want[0])
    with pytest.raises(gcu.GcuError, match="length outside"):
        gcu.check_device()
    gcu.check_device()  # reported once


@pytest.mark.parametrize("first", ["length", "wait"])
def test_a_length_error_does_not_hide_a_wait(first):
    if first == "length":
        too_long("decode")
    gcu.selftest_bounded_wait(0, 100)
    if first == "wait":
        too_long("write")
    with pytest.raises(gcu.GcuError, match="wait gave up.*length outside"):
        gcu.check_device()
    gcu.check_device()


def test_decoder_stops_at_its_tail():
    """The steps that fit, from replays too, and then a refusal on the host or the device's report."""
    import synth
    import test_gpu_decode_i8 as D
    name = next(iter(D.META["cases"]))
    cfg, emb, dec = D.model(name, 8, 8)
    D.prefill(cfg, dec, synth.normal(cfg["tid"] + 777, (4, cfg["dim"])))

    def start():
        dec.fork(2, 4, 3)
        dec.set_seq_freqs(*D.tables(cfg, [4] * 2))
        dec.sx.copy_(torch.from_numpy(synth.normal(93, (2, cfg["dim"]))))
    start()
    for _ in range(3):
        dec.step_seqs()
    with pytest.raises(ValueError, match="3 tokens"):
        dec.step_seqs()
    assert dec.slen.tolist() == [3, 3]
    gcu.check_device()
    start()
    dec.step_seqs()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step_seqs()
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    gcu.check_device()
    assert dec.slen.tolist() == [3, 3]
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(gcu.GcuError, match="length outside"):
        gcu.check_device()
