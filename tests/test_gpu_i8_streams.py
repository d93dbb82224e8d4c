"""The 8-bit cache's attention and sampling on several streams of one thread, nothing waited for
between the calls: each call's result is, bit for bit, that of the same call alone."""
import pytest

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


@pytest.mark.parametrize("side_first", [False, True])
def test_scratch_of_calls_on_two_streams(side_first):
    """Calls with the same scratch size, at once on the current stream and on another: about 100 us
    of work each, several times what a call takes its caller."""
    g = torch.Generator(device="cuda").manual_seed(31)
    n = 262144
    codes = torch.randint(-127, 128, (2, 1, 8, n, 128), generator=g, dtype=torch.int8, device="cuda")
    scales = torch.rand((2, 1, 8, n), generator=g, device="cuda") * 0.02 + 0.01
    kv = gcu.KvCacheI8(codes[0], codes[1], scales[0], scales[1])
    q = [torch.randn((1, 16, 128), generator=g, device="cuda") for _ in range(2)]
    p = [torch.randn((16, 700, 128), generator=g, device="cuda") * 0.1 for _ in range(2)]
    assert gcu.lib().gcu_attention_decode_i8_work(None, 0, kv.ref, n, 16, 0) > 0
    assert gcu.lib().gcu_attention_prefill_i8_work(kv.ref, 16, 1000, 700, 0, 0.0, 1) > 0

    def decode(i, xo, stream=None):
        gcu.dev_attention_decode_i8(xo, q[i], kv, None, n, 128 ** -0.5, stream=stream)

    def prefill(i, xo, stream=None):
        gcu.dev_attention_prefill_i8(xo, p[i], kv, 1000, stream=stream)

    side = torch.cuda.Stream()
    for call, like in ((decode, q[0]), (prefill, torch.empty((700, 16 * 128), device="cuda"))):
        alone = [torch.empty_like(like) for _ in range(2)]
        for i in range(2):
            call(i, alone[i])
            torch.cuda.synchronize()
        for _ in range(10):
            outs = [torch.full_like(like, 7.0) for _ in range(4)]
            torch.cuda.synchronize()
            for j, out in enumerate(outs):
                call(j % 2, out, side if (j % 2 == 1) != side_first else None)
            torch.cuda.synchronize()
            for j, out in enumerate(outs):
                assert torch.equal(out, alone[j % 2])


def test_tokens_sampled_on_another_stream():
    """Tokens of a side stream beside work of the current stream that drops blocks of their size."""
    import decode
    dec = object.__new__(decode.Decoder)
    g = torch.Generator(device="cuda").manual_seed(32)
    dec.torch, dec.dev, dec.slogits = torch, "cuda", torch.randn((5, 50000), generator=g, device="cuda")
    u, big = torch.rand(5, generator=g, device="cuda"), torch.zeros(1 << 28, device="cuda")
    want = dec.sample(u, 0.9, 50, seqs=True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        big.add_(1)  # some 300 us
        torch.zeros(5, dtype=torch.int32, device="cuda")  # written after that, dropped now
        token = dec.sample(u, 0.9, 50, seqs=True, stream=side)
        side.synchronize()
        early = token.tolist()
        torch.cuda.synchronize()
        assert early == token.tolist() == want.tolist()


def test_forked_sequences_on_another_stream():
    """fork, tables, steps and samples on a side stream while the current one is busy, twice over:
    as on the current stream."""
    import synth
    import test_gpu_decode_i8 as D
    name = next(iter(D.META["cases"]))
    cfg, emb, _ = D.model(name, 8, 12)
    x = synth.normal(cfg["tid"] + 777, (6, cfg["dim"]))
    u = torch.rand((3, 4), generator=torch.Generator().manual_seed(5)).cuda()
    start = torch.from_numpy(synth.normal(92, (4, cfg["dim"]))).cuda()
    big = torch.zeros(1 << 28, device="cuda")
    side = torch.cuda.Stream()
    results = []
    for stream in (None, side):
        dec = D.model(name, 8, 12)[2]
        D.prefill(cfg, dec, x)
        torch.cuda.synchronize()
        got = []
        for turn in range(2):
            big.add_(1)
            dec.fork(4, 6, 3, stream=stream)
            for r in range(3):
                dec.set_seq_freqs(*D.tables(cfg, [6 + r] * 4), stream=stream)
                with torch.cuda.stream(stream) if stream is not None else torch.no_grad():
                    dec.sx.copy_(start)
                dec.step_seqs(stream=stream)
                t = dec.sample(u[r], 0.9, 20, seqs=True, stream=stream)
                with torch.cuda.stream(stream) if stream is not None else torch.no_grad():
                    got.append((t.clone(), dec.slogits.clone(), dec.slen.clone()))
        torch.cuda.synchronize()
        results.append([[v.cpu() for v in g] for g in got])
    for a, b in zip(*results):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
