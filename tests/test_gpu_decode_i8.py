"""The 8-bit KV cache, its attention and sampling together, as a decoder runs them.

An fp32 value a few ulps from a rounding boundary can take the neighbouring int8
code, in an activation or in the cache, which moves that product by one code
step; the bound is the one of the fp32-cache decoder's chain (max difference
2e-3 of the largest value, median 1e-5 of it)."""
import json
import os

import numpy as np
import pytest

import i8_cases as R
import synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decode  # noqa: E402
import gcu  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
META = json.loads(str(np.load(os.path.join(HERE, "golden", "decode.npz"))["meta"]))


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    gcu.init(0)
    yield
    gcu.check_device()


def close(got, want):
    err = np.abs(got - want)
    scale = float(np.max(np.abs(want)))
    assert err.max() <= 2e-3 * scale and np.median(err) <= 1e-5 * scale, (err.max() / scale, np.median(err) / scale)


def model(name, kv_bits, clen):
    cfg = META["cases"][name]
    layers, emb, fnorm = synth.decoder_model(cfg["tid"], cfg)
    return cfg, emb, decode.Decoder(cfg, layers, emb, fnorm, clen=clen, kv_bits=kv_bits)


def tables(cfg, pos):
    return [np.stack(t) for t in zip(*(decode.rope_tables(cfg["hdim"], cfg["theta_l"], cfg["theta_g"], p) for p in pos))]


def embed(cfg, emb, token):
    """gemma.c:5466-5490: the embedding's row, dequantized, times sqrt(dim)."""
    return (emb[0][token].astype(np.float32) * emb[1][token] * np.float32(np.sqrt(np.float32(cfg["dim"]))))


def prefill(cfg, dec, x, spos=0):
    dec.set_prefill_freqs(*tables(cfg, range(spos, spos + len(x))))
    dec.px[:len(x)].copy_(torch.from_numpy(x))
    dec.prefill(spos, len(x))


def step(cfg, dec, pos, x):
    dec.set_freqs(*(t[0] for t in tables(cfg, [pos])))
    dec.x.copy_(torch.from_numpy(x[None]))
    dec.step(pos)


@pytest.mark.parametrize("name", list(META["cases"]))
def test_prefill_and_step_agree(name):
    """A prompt in two chunks and then one token, against one token at a time."""
    cfg, emb, a = model(name, 8, 20)
    b = model(name, 8, 20)[2]
    x = synth.normal(cfg["tid"] + 777, (18, cfg["dim"]))
    prefill(cfg, a, x[:6])
    prefill(cfg, a, x[6:17], 6)
    step(cfg, a, 17, x[17])
    for p in range(18):
        step(cfg, b, p, x[p])
    torch.cuda.synchronize()
    close(a.logits.cpu().numpy()[0], b.logits.cpu().numpy()[0])
    for l in range(cfg["nl"]):  # the caches hold the same codes but for flips at boundaries
        d = (a.kv8[l].k[0, :, :18].int() - b.kv8[l].k[0, :, :18].int()).abs()
        assert int(d.max()) <= 1 and float((d > 0).float().mean()) <= 0.01


@pytest.mark.parametrize("name", list(META["cases"]))
def test_cache_holds_the_fp32_caches_rows(name):
    """The first layer's keys and values, read back, are the fp32 cache's to half a code step."""
    cfg, emb, a = model(name, 8, 16)
    b = model(name, 32, 16)[2]
    x = synth.normal(cfg["tid"] + 777, (13, cfg["dim"]))
    prefill(cfg, a, x)
    prefill(cfg, b, x)
    k = torch.empty((1, cfg["nkv"], 13, cfg["hdim"]), device="cuda")
    v = torch.empty_like(k)
    gcu.dev_cache_i8_read(k, v, a.kv8[0], 0)
    for got, want, s in ((k[0], b.kv[0, 0, :, :13], a.kv8[0].ks), (v[0], b.kv[0, 1, :, :13], a.kv8[0].vs)):
        # half a step of the row, and what the two norms' fp32 arithmetic differs by
        assert bool(((got - want).abs() <= s[0, :, :13, None] * 0.5001 + 1e-5 * want.abs().max()).all())


@pytest.mark.parametrize("name,nseq", [(n, 3) for n in META["cases"]] + [(next(iter(META["cases"])), 11)])
def test_sequences_share_a_prompt_and_sample(name, nseq):
    """Prompt, fork, and a few rounds of sample -> embed -> step of all sequences, against each
    sequence decoded alone over one cache with the same tokens."""
    cfg, emb, dec = model(name, 8, 16)
    plen, rounds = 9, 3
    x = synth.normal(cfg["tid"] + 777, (plen, cfg["dim"]))
    prefill(cfg, dec, x)
    first = dec.logits.expand(nseq, -1).contiguous()
    rng = np.random.default_rng(3)
    u = rng.random((rounds, nseq), dtype=np.float32)
    settings = (0.9, 50, 0.95, 0.01)
    token = torch.empty(nseq, dtype=torch.int32, device="cuda")
    gcu.dev_sample(token, first, torch.from_numpy(u[0]).cuda(), *settings)
    row = first[0].cpu().numpy()
    assert token.tolist() == [R.sample(row, v, *settings)[0] for v in u[0]]
    dec.fork(nseq, plen, rounds)
    tokens, logits = [token.tolist()], []
    for r in range(rounds):
        dec.set_seq_freqs(*tables(cfg, [plen + r] * nseq))
        dec.sx.copy_(torch.from_numpy(np.stack([embed(cfg, emb, t) for t in tokens[-1]])))
        dec.step_seqs()
        logits.append(dec.slogits.cpu().numpy())
        assert dec.slen.tolist() == [r + 1] * nseq
        if r + 1 < rounds:
            t = dec.sample(torch.from_numpy(u[r + 1]).cuda(), *settings, seqs=True)
            assert t.tolist() == [R.sample(lg, v, *settings)[0] for lg, v in zip(logits[-1], u[r + 1])]
            tokens.append(t.tolist())
    for b in range(min(nseq, 3)):
        alone = model(name, 8, 16)[2]
        prefill(cfg, alone, x)
        for r in range(rounds):
            step(cfg, alone, plen + r, embed(cfg, emb, tokens[r][b]))
            close(logits[r][b], alone.logits.cpu().numpy()[0])


def test_a_finished_sequence_stands_still():
    name = next(iter(META["cases"]))
    cfg, emb, dec = model(name, 8, 8)
    x = synth.normal(cfg["tid"] + 777, (5, cfg["dim"]))
    prefill(cfg, dec, x)
    dec.fork(2, 5, 4)
    for r in range(2):
        if r == 1:
            dec.slen[1] = -1
            kept = [o.k[1].clone() for o in dec.own8]
        dec.set_seq_freqs(*tables(cfg, [5 + r] * 2))
        dec.sx.copy_(torch.from_numpy(synth.normal(55 + r, (2, cfg["dim"]))))
        dec.step_seqs()
    assert dec.slen.tolist() == [2, -1]
    assert all(torch.equal(k, o.k[1]) for k, o in zip(kept, dec.own8))


def test_steps_are_capturable():
    """A captured step of all sequences and its sampling replay: lengths and caches move on."""
    name = next(iter(META["cases"]))
    cfg, emb, _ = model(name, 8, 8)
    outs = []
    for graph in (False, True):
        dec = model(name, 8, 8)[2]
        prefill(cfg, dec, synth.normal(cfg["tid"] + 777, (6, cfg["dim"])))
        dec.fork(3, 6, 4)
        dec.set_seq_freqs(*tables(cfg, [6] * 3))
        u, x = torch.tensor([0.1, 0.5, 0.9], device="cuda"), torch.from_numpy(synth.normal(91, (3, cfg["dim"]))).cuda()
        token = torch.empty(3, dtype=torch.int32, device="cuda")

        def one():
            dec.sx.copy_(x)
            dec.step_seqs()
            gcu.dev_sample(token, dec.slogits, u, 1.0, 20)
        one()  # also warms the library up
        if graph:
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                one()
            one = g.replay
        one()
        one()
        torch.cuda.synchronize()
        outs.append((dec.slogits.cpu().numpy(), token.tolist(), dec.slen.tolist(), dec.own8[0].k.cpu().numpy()))
    assert outs[0][1] == outs[1][1] and outs[0][2] == outs[1][2] == [3, 3, 3]
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][3], outs[1][3])


def test_refusals():
    name = next(iter(META["cases"]))
    cfg, emb, dec = model(name, 32, 8)
    with pytest.raises(ValueError, match="8-bit"):
        dec.fork(2, 4, 4)
    with pytest.raises(ValueError, match="8 or 32"):
        model(name, 16, 8)
    dec = model(name, 8, 8)[2]
    with pytest.raises(ValueError, match="fork first"):
        dec.step_seqs()
    for bad in ((0, 4, 4), (2, 9, 4), (2, 4, 0)):
        with pytest.raises(ValueError, match="fork of"):
            dec.fork(*bad)
