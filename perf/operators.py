"""The 8-bit KV cache, attention over it, and sampling: cases, plain forms and calls.

Cases are dicts with an "op":

  write    rows of a fused q|k|v projection are normed, rotated and written to an
           8-bit cache (per-row scales), and the written rows are read back;
  decode   one token of each of nseq sequences attends to a prefix that all of
           them share and to the sequence's own 8-bit cache;
  prefill  a chunk of a prompt attends to the 8-bit cache, causally;
  sample   next tokens from logits, given one random number per row.

Head counts and sizes are those of the Gemma 3 decoders this repository runs
(4/1/256, 8/4/256, 16/8/256) and the other head sizes its attention takes.
"""
import math
import os
import sys

import torch

own = False

_gcu = None


def _lib():
    """The framework's binding, ready on device 0 (only where `own` is true)."""
    global _gcu
    if _gcu is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "gemma.c_b200"))
        import gcu
        gcu.init(0)
        _gcu = gcu
    return _gcu


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _write(nh, nkv, hd, rows, pos, seqs=False, norm=True, **more):
    return dict(op="write", nh=nh, nkv=nkv, hd=hd, rows=rows, pos=pos, seqs=seqs, norm=norm, **more)


def _decode(nh, nkv, hd, nseq, plen, tail, slide=0, cap=0.0, **more):
    return dict(op="decode", nh=nh, nkv=nkv, hd=hd, nseq=nseq, plen=plen, tail=tail, slide=slide, cap=cap, **more)


def _prefill(nh, nkv, hd, spos, ntok, slide=0, cap=0.0, mask=True, **more):
    return dict(op="prefill", nh=nh, nkv=nkv, hd=hd, spos=spos, ntok=ntok, slide=slide, cap=cap, mask=mask, **more)


def _sample(rows, nvocab, temp, top_k, top_p, min_p, **more):
    return dict(op="sample", rows=rows, nvocab=nvocab, temp=temp, top_k=top_k, top_p=top_p, min_p=min_p, **more)


def listed():
    return [
        # one token's keys and values of a small decoder: a launch's latency
        _write(4, 1, 256, 1, 1023, name="write 1 token"),
        # one token for each of eight answers to a prompt, each to its own cache
        _write(8, 4, 256, 8, 60, seqs=True, name="write 8 sequences"),
        # a whole prompt of a large decoder
        _write(16, 8, 256, 4096, 0, name="write 4096 tokens"),
        # a sliding layer of a small decoder past its window: the smallest attention call
        _decode(4, 1, 256, 1, 0, 1024, slide=512, name="decode 512 window"),
        # a global layer of a large decoder, one sequence at a long context
        _decode(16, 8, 256, 1, 0, 32768, name="decode 32k"),
        # eight answers to one prompt, tails of different lengths
        _decode(8, 4, 256, 8, 2049, 97, name="decode 8 share 2k"),
        # many answers to one long document
        _decode(16, 8, 256, 32, 32768, 255, name="decode 32 share 32k"),
        # the first chunk of a prompt on a sliding layer
        _prefill(4, 1, 256, 0, 512, slide=512, name="prefill 512"),
        # an odd later chunk, capped scores, the smaller head size
        _prefill(16, 8, 128, 777, 1023, cap=50.0, name="prefill 1023 at 777"),
        # a long prompt in one chunk on a global layer
        _prefill(16, 8, 256, 0, 8192, name="prefill 8192"),
        # one sequence's next token, the usual settings
        _sample(1, 262144, 0.8, 64, 0.95, 0.0, name="sample 1"),
        # a batch over the whole vocabulary, nucleus and min-p
        _sample(32, 262144, 1.0, 0, 0.9, 0.02, name="sample 32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd ones too."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "prefill", "prefill", "sample"])
    nh, nkv = rng.choice([(4, 1), (8, 4), (16, 8), (8, 2), (8, 1), (6, 4), (4, 4)])
    hd = rng.choice([64, 128, 256, 256])
    if op == "write":
        seqs = rng.random() < 0.4
        rows = _log(rng, 1, 64) if seqs else _log(rng, 1, 4096)
        return _write(nh, nkv, hd, rows, rng.randint(0, 500), seqs, rng.random() < 0.7)
    if op == "decode":
        cap = rng.choice([0.0, 0.0, 50.0])
        if rng.random() < 0.4:
            tail = _log(rng, 1, 32768)
            return _decode(nh, nkv, hd, 1, 0, tail, rng.choice([0, 0, 512, 1024]), cap)
        nseq, plen = _log(rng, 1, 32), _log(rng, 1, 16384)
        return _decode(nh, nkv, hd, nseq, plen, _log(rng, 1, 300), rng.choice([0, 0, 1024]), cap)
    if op == "prefill":
        spos, ntok = rng.choice([0, _log(rng, 1, 4096)]), _log(rng, 9, 4096)
        return _prefill(nh, nkv, hd, spos, ntok, rng.choice([0, 0, 512, 1024]), rng.choice([0.0, 0.0, 50.0]),
                        rng.random() < 0.85)
    return _sample(_log(rng, 1, 32), rng.choice([262144, _log(rng, 1000, 262144)]), rng.uniform(0.3, 1.5),
                   rng.choice([0, 1, _log(rng, 2, 1000)]), rng.choice([1.0, rng.uniform(0.3, 0.99)]),
                   rng.choice([0.0, rng.uniform(0.001, 0.2)]))


def _lens(c):
    """Own positions of each sequence, the new token's among them: ragged when several share a prefix."""
    return [max(1, c["tail"] - (37 * b) % c["tail"]) for b in range(c["nseq"])]


def _windows(c):
    """Sum over sequences of visible positions, and the prefix and own positions that any of them sees."""
    total, first, seen_own = 0, c["plen"], 0
    for n in _lens(c):
        lo = max(0, c["plen"] + n - c["slide"]) if c["slide"] else 0
        total += c["plen"] + n - lo
        first = min(first, lo)
        seen_own += n - max(0, lo - c["plen"])
    return total, c["plen"] - first, seen_own


def work(c):
    if c["op"] == "write":
        nh, nkv, hd, n = c["nh"], c["nkv"], c["hd"], c["rows"]
        # q|k|v rows and tables in; rotated queries, codes and scales, and the rows read back, out
        return {"bytes": n * (4 * (nh + 2 * nkv) * hd + 4 * hd + 4 * nh * hd + nkv * (2 * hd + 8) + 8 * nkv * hd),
                "flops": n * (nh + 2 * nkv) * hd * 8}
    if c["op"] == "decode":
        total, pre, mine = _windows(c)
        return {"bytes": c["nkv"] * (2 * c["hd"] + 8) * (pre + mine) + 8 * c["nseq"] * c["nh"] * c["hd"],
                "flops": 4 * c["hd"] * c["nh"] * total}
    if c["op"] == "prefill":
        end, pairs = c["spos"] + c["ntok"], 0
        for i in range(c["spos"], end):
            pairs += (min(i + 1, c["slide"]) if c["slide"] else i + 1) if c["mask"] else end
        first = max(0, c["spos"] + 1 - c["slide"]) if c["mask"] and c["slide"] else 0
        return {"bytes": c["nkv"] * (2 * c["hd"] + 8) * (end - first) + 8 * c["ntok"] * c["nh"] * c["hd"],
                "flops": 4 * c["hd"] * c["nh"] * pairs}
    return {"bytes": 4 * c["rows"] * c["nvocab"] + 12 * c["rows"], "flops": 4 * c["rows"] * c["nvocab"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _codes(x):
    """Per-row int8 codes and scales of x (..., hd), as an 8-bit cache holds them."""
    amax = x.abs().amax(-1)
    live = amax > 0
    scale = torch.where(live, amax * torch.tensor(1.0 / 127.0, device=x.device), torch.ones_like(amax))
    inv = torch.where(live, torch.full_like(amax, 127.0) / amax, torch.ones_like(amax))
    t = x * inv.unsqueeze(-1)
    q = torch.trunc(t + torch.copysign(torch.full_like(t, 0.5), t)).clamp(-127, 127)
    return q.to(torch.int8), scale


def _cache(g, nseq, nkv, clen, hd):
    k, ks = _codes(torch.randn((nseq, nkv, clen, hd), generator=g, device="cuda"))
    v, vs = _codes(torch.randn((nseq, nkv, clen, hd), generator=g, device="cuda"))
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def _handle(cache):
    """The framework's description of a cache's buffers, which a program keeps beside them."""
    return _lib().KvCacheI8(cache["k"], cache["v"], cache["ks"], cache["vs"])


def _tables(pos, hd):
    """RoPE (cos, sin) interleaved per frequency for each position, from angles in 64 bits."""
    f = 10000.0 ** (torch.arange(hd // 2, dtype=torch.float64, device="cuda") * (-2.0 / hd))
    a = pos.to(torch.float64).unsqueeze(-1) * f
    return torch.stack([torch.cos(a), torch.sin(a)], -1).reshape(len(pos), hd).float()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    if c["op"] == "write":
        nh, nkv, hd, n = c["nh"], c["nkv"], c["hd"], c["rows"]
        nseq, clen = (n, c["pos"] + 8) if c["seqs"] else (1, c["pos"] + n + 8)
        cache = {"k": torch.zeros((nseq, nkv, clen, hd), dtype=torch.int8, **dev),
                 "v": torch.zeros((nseq, nkv, clen, hd), dtype=torch.int8, **dev),
                 "ks": torch.ones((nseq, nkv, clen), **dev), "vs": torch.ones((nseq, nkv, clen), **dev)}
        s = {"c": c, "cache": cache, "qkv": torch.randn((n, (nh + 2 * nkv) * hd), generator=g, **dev),
             "nq": torch.randn(hd, generator=g, **dev) * 0.1 if c["norm"] else None,
             "nk": torch.randn(hd, generator=g, **dev) * 0.1 if c["norm"] else None,
             "freqs": _tables(torch.full((n,), c["pos"], **dev) if c["seqs"]
                              else torch.arange(c["pos"], c["pos"] + n, **dev), hd),
             "q_scale": 1.0 if c["seqs"] else 1.0 / math.sqrt(hd),
             "len": torch.full((n,), c["pos"] + 1, dtype=torch.int32, **dev),
             "xq": torch.empty((n, nh, hd) if c["seqs"] else (nh, n, hd), **dev),
             "rk": torch.empty((nseq, nkv, 1 if c["seqs"] else n, hd), **dev),
             "rv": torch.empty((nseq, nkv, 1 if c["seqs"] else n, hd), **dev)}
        if own:
            s["kv"] = _handle(cache)
        return s
    if c["op"] == "decode":
        lens = _lens(c)
        s = {"c": c, "own": _cache(g, c["nseq"], c["nkv"], c["tail"] + 5, c["hd"]),
             "prefix": _cache(g, 1, c["nkv"], c["plen"], c["hd"]) if c["plen"] else None,
             "xq": torch.randn((c["nseq"], c["nh"], c["hd"]), generator=g, **dev) * 1.5,
             "xo": torch.empty((c["nseq"], c["nh"], c["hd"]), **dev),
             "len": torch.tensor(lens, dtype=torch.int32, **dev), "asc": 1.0 / math.sqrt(c["hd"])}
        if own:
            s["kv"] = _handle(s["own"])
            s["pkv"] = _handle(s["prefix"]) if s["prefix"] else None
        return s
    if c["op"] == "prefill":
        s = {"c": c, "own": _cache(g, 1, c["nkv"], c["spos"] + c["ntok"], c["hd"]),
             "xq": torch.randn((c["nh"], c["ntok"], c["hd"]), generator=g, **dev) * (1.5 / math.sqrt(c["hd"])),
             "xo": torch.empty((c["ntok"], c["nh"] * c["hd"]), **dev)}
        if own:
            s["kv"] = _handle(s["own"])
        return s
    # logits as a decoder gives them: most of a vocabulary far below a few likely tokens
    x = torch.randn((c["rows"], c["nvocab"]), generator=g, **dev) * 2.5
    x += 6.0 * torch.rand((c["rows"], c["nvocab"]), generator=g, **dev).pow(400)
    return {"c": c, "logits": x, "u": torch.rand(c["rows"], generator=g, **dev),
            "token": torch.empty(c["rows"], dtype=torch.int32, **dev), "prob": torch.empty(c["rows"], **dev)}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _head_of(nh, nkv):
    """The kv head of each query head."""
    return torch.arange(nh, device="cuda") * nkv // nh


def _norm_rope(x, w, eps, freqs, scale):
    """Head rows x (n, heads, hd) at the n positions of freqs; every fp32 step rounded by itself."""
    hd = x.shape[-1]
    if w is not None:
        mean = x.double().square().sum(-1, keepdim=True) / hd
        x = x * (1.0 / torch.sqrt(mean + float(torch.tensor(eps, dtype=torch.float32)))).float() * (w + 1.0)
    cos, sin = freqs[:, None, 0::2], freqs[:, None, 1::2]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([(a * cos - b * sin) * scale, (a * sin + b * cos) * scale], -1)


def _plain_write(s):
    c, cache = s["c"], s["cache"]
    nh, nkv, hd, n = c["nh"], c["nkv"], c["hd"], c["rows"]
    x = s["qkv"].view(n, nh + 2 * nkv, hd)
    q_scale = torch.tensor(s["q_scale"], dtype=torch.float32, device="cuda")
    one = torch.ones((), device="cuda")
    q = _norm_rope(x[:, :nh], s["nq"], 1e-6, s["freqs"], q_scale)
    k, ks = _codes(_norm_rope(x[:, nh:nh + nkv], s["nk"], 1e-6, s["freqs"], one))
    v, vs = _codes(x[:, nh + nkv:])
    if c["seqs"]:  # row b to position pos of sequence b's cache
        at = (slice(None), slice(None), slice(c["pos"], c["pos"] + 1))
        put = lambda t: t.unsqueeze(2)
    else:
        at = (slice(0, 1), slice(None), slice(c["pos"], c["pos"] + n))
        put = lambda t: t.transpose(0, 1).unsqueeze(0)
    for name, t in (("k", k), ("ks", ks), ("v", v), ("vs", vs)):
        cache[name][at] = put(t)
    s["xq"].copy_(q if c["seqs"] else q.transpose(0, 1))
    s["rk"].copy_(cache["k"][at].float() * cache["ks"][at].unsqueeze(-1))
    s["rv"].copy_(cache["v"][at].float() * cache["vs"][at].unsqueeze(-1))
    return {"xq": s["xq"], "k": s["rk"], "v": s["rv"]}


def _softmax_values(score, cap, seen, values):
    """Capped, masked softmax of score (..., n) and its weighted sum of values (..., n, hd); an empty row gives zeros."""
    if cap:
        score = torch.tanh(score / cap) * cap
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return (p @ values) / torch.where(total > 0, total, torch.ones_like(total))


def _wide(cache, what, kind):
    return cache[what].to(kind) * cache[what + "s"].to(kind).unsqueeze(-1)


def _attend_decode(s, kind):
    c, own_c, pre = s["c"], s["own"], s["prefix"]
    nh, nkv, nseq, tail = c["nh"], c["nkv"], c["nseq"], c["tail"]
    hk = _head_of(nh, nkv)
    q = s["xq"].to(kind)
    k, v = _wide(own_c, "k", kind)[:, :, :tail], _wide(own_c, "v", kind)[:, :, :tail]
    score = (k[:, hk] @ q.unsqueeze(-1)).squeeze(-1)
    values = v[:, hk]
    if pre:
        pk, pv = _wide(pre, "k", kind)[0][hk], _wide(pre, "v", kind)[0][hk]
        score = torch.cat([(q.transpose(0, 1) @ pk.transpose(1, 2)).transpose(0, 1), score], -1)
    n = c["plen"] + s["len"].long()
    t = torch.arange(c["plen"] + tail, device="cuda")
    lo = (n - c["slide"]).clamp(min=0) if c["slide"] else torch.zeros_like(n)
    seen = (t < n[:, None]) & (t >= lo[:, None])
    score = score * torch.tensor(s["asc"], dtype=kind, device="cuda")
    if c["cap"]:
        score = torch.tanh(score / c["cap"]) * c["cap"]
    score = score.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p[..., c["plen"]:].unsqueeze(2) @ values).squeeze(2)
    if pre:
        out = out + (p[..., :c["plen"]].transpose(0, 1) @ pv).transpose(0, 1)
    return out / p.sum(-1, keepdim=True)


def _attend_prefill(s, kind, heads):
    c = s["c"]
    hk = _head_of(c["nh"], c["nkv"])[heads]
    k, v = _wide(s["own"], "k", kind)[0][hk], _wide(s["own"], "v", kind)[0][hk]
    score = s["xq"][heads].to(kind) @ k.transpose(1, 2)
    pos = torch.arange(c["spos"], c["spos"] + c["ntok"], device="cuda")[:, None]
    t = torch.arange(c["spos"] + c["ntok"], device="cuda")[None]
    seen = torch.ones((c["ntok"], c["spos"] + c["ntok"]), dtype=torch.bool, device="cuda")
    if c["mask"]:
        seen = t <= pos
        if c["slide"]:
            seen = seen & (t > pos - c["slide"])
    return _softmax_values(score, c["cap"], seen, v)


def _plain_sample(s):
    c, x, u = s["c"], s["logits"], s["u"]
    n = x.shape[1]
    top, order = torch.sort(x, dim=1, descending=True, stable=True)  # of equals the lowest index first
    w = torch.exp((top.double() - top[:, :1].double()) / float(torch.tensor(c["temp"], dtype=torch.float32)))
    rank = torch.arange(n, device="cuda")
    keep = rank[None] < (c["top_k"] or n)
    kept = torch.where(keep, w, torch.zeros_like(w))
    if c["top_p"] < 1.0:
        before = torch.cumsum(kept, 1) - kept
        keep = keep & (before < float(torch.tensor(c["top_p"], dtype=torch.float32)) * kept.sum(1, keepdim=True))
    keep = keep & (w >= float(torch.tensor(c["min_p"], dtype=torch.float32)))
    kept = torch.where(keep, w, torch.zeros_like(w))
    by_index = torch.zeros_like(kept).scatter_(1, order, kept)
    upto = torch.cumsum(by_index, 1)
    total = kept.sum(1, keepdim=True)
    token = ((upto <= u.double()[:, None] * total) | (by_index == 0)).to(torch.int32)
    token = torch.argmin(token, 1)  # the first kept index whose running sum passes u * total
    prob = by_index.gather(1, token[:, None]) / total
    s["token"].copy_(token)
    s["prob"].copy_(prob[:, 0])
    return {"token": s["token"], "prob": s["prob"]}


def run(s):
    c = s["c"]
    if c["op"] == "write":
        if not own:
            return _plain_write(s)
        g = _lib()
        if c["seqs"]:
            g.dev_qkv_norm_rope_cache_i8_seqs(s["xq"], s["qkv"], s["kv"], s["len"], s["freqs"], s["q_scale"], s["nq"],
                                              s["nk"], 1e-6)
            g.dev_cache_i8_read(s["rk"], s["rv"], s["kv"], c["pos"])
        else:
            g.dev_qkv_norm_rope_cache_i8(s["xq"], s["qkv"], s["kv"], s["freqs"], c["pos"], s["q_scale"], s["nq"],
                                         s["nk"], 1e-6)
            g.dev_cache_i8_read(s["rk"], s["rv"], s["kv"], c["pos"])
        return {"xq": s["xq"], "k": s["rk"], "v": s["rv"]}
    if c["op"] == "decode":
        if not own:
            s["xo"].copy_(_attend_decode(s, torch.float32))
            return s["xo"]
        _lib().dev_attention_decode_i8(s["xo"], s["xq"], s["kv"], s["len"], c["tail"], s["asc"], c["cap"], c["slide"],
                                       s["pkv"], c["plen"])
        return s["xo"]
    if c["op"] == "prefill":
        if not own:
            out = _attend_prefill(s, torch.float32, slice(None))
            s["xo"].copy_(out.transpose(0, 1).reshape(s["xo"].shape))
            return s["xo"]
        _lib().dev_attention_prefill_i8(s["xo"], s["xq"], s["kv"], c["spos"], c["slide"], c["cap"], c["mask"])
        return s["xo"]
    if not own:
        return _plain_sample(s)
    _lib().dev_sample(s["token"], s["logits"], s["u"], c["temp"], c["top_k"], c["top_p"], c["min_p"], prob=s["prob"])
    return {"token": s["token"], "prob": s["prob"]}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def _exact_row_codes(x):
    """code * scale in 64 bits of fp32 rows x, by the quantiser's definition."""
    amax = x.abs().max(-1, keepdim=True).values
    scale = (amax.double() * float(torch.tensor(1.0 / 127.0, dtype=torch.float32))).float()
    inv = (127.0 / amax.double()).float()  # a quotient rounded once
    t = (x.double() * inv.double()).float().double()
    code = torch.sign(t) * torch.floor((t.abs() + 0.5).float().double())
    return code.clamp(-127, 127) * scale.double()


def _exact_rotated(x, w, freqs, scale):
    """As the rows are defined: the norm's factor and every step after it rounded to 32 bits, worked in 64."""
    r = lambda t: t.float().double()
    hd = x.shape[-1]
    x = x.double()
    if w is not None:
        eps = float(torch.tensor(1e-6, dtype=torch.float32))
        factor = r((x.pow(2).mean(-1, keepdim=True) + eps).rsqrt())
        x = r(r(x * factor) * r(w.double() + 1.0))
    f = freqs.double().reshape(freqs.shape[0], 1, hd // 2, 2)
    re, im, cos, sin = x[..., :hd // 2], x[..., hd // 2:], f[..., 0], f[..., 1]
    lo = r(r(re * cos) - r(im * sin))
    hi = r(r(re * sin) + r(im * cos))
    return r(torch.cat([lo, hi], -1) * float(torch.tensor(scale, dtype=torch.float32)))


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "write":
        n, nh, nkv, hd = c["rows"], c["nh"], c["nkv"], c["hd"]
        q, k, v = s["qkv"].view(n, -1, hd).split([nh, nkv, nkv], 1)
        q = _exact_rotated(q, s["nq"], s["freqs"], s["q_scale"])
        k = _exact_row_codes(_exact_rotated(k, s["nk"], s["freqs"], 1.0).float())
        v = _exact_row_codes(v)
        lay = (lambda t: t[:, :, None]) if c["seqs"] else (lambda t: t.permute(1, 0, 2)[None])
        return {"xq": q if c["seqs"] else q.permute(1, 0, 2), "k": lay(k), "v": lay(v)}
    if c["op"] == "decode":
        out = torch.empty((c["nseq"], c["nh"], c["hd"]), dtype=torch.float64, device="cuda")
        lens = _lens(c)
        for h in range(c["nh"]):
            j = h * c["nkv"] // c["nh"]
            for b in range(c["nseq"]):
                keys = [s["own"]["k"][b, j, :lens[b]].double() * s["own"]["ks"][b, j, :lens[b], None].double()]
                vals = [s["own"]["v"][b, j, :lens[b]].double() * s["own"]["vs"][b, j, :lens[b], None].double()]
                if s["prefix"]:
                    keys.insert(0, s["prefix"]["k"][0, j].double() * s["prefix"]["ks"][0, j, :, None].double())
                    vals.insert(0, s["prefix"]["v"][0, j].double() * s["prefix"]["vs"][0, j, :, None].double())
                keys, vals = torch.cat(keys), torch.cat(vals)
                lo = max(0, len(keys) - c["slide"]) if c["slide"] else 0
                z = (keys[lo:] * s["xq"][b, h].double()).sum(-1) / math.sqrt(c["hd"])
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                w = torch.exp(z - z.max())
                out[b, h] = (w[:, None] * vals[lo:]).sum(0) / w.sum()
        return out
    if c["op"] == "prefill":
        out = torch.empty((c["ntok"], c["nh"], c["hd"]), dtype=torch.float64, device="cuda")
        end = c["spos"] + c["ntok"]
        for h in range(c["nh"]):
            j = h * c["nkv"] // c["nh"]
            keys = s["own"]["k"][0, j].double() * s["own"]["ks"][0, j, :, None].double()
            vals = s["own"]["v"][0, j].double() * s["own"]["vs"][0, j, :, None].double()
            for i in range(0, c["ntok"], 1024):
                rows = min(1024, c["ntok"] - i)
                z = torch.einsum("id,td->it", s["xq"][h, i:i + rows].double(), keys)
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                if c["mask"]:
                    back = torch.arange(c["spos"] + i, c["spos"] + i + rows, device="cuda")[:, None] - torch.arange(end, device="cuda")
                    hidden = back < 0
                    if c["slide"]:
                        hidden |= back >= c["slide"]
                    z[hidden] = -math.inf
                out[i:i + rows, h] = torch.einsum("it,td->id", torch.softmax(z, -1), vals)
        return out.reshape(c["ntok"], -1)
    return _exact_sample(c, s)


def _exact_sample(c, s):
    """Tokens and probabilities row by row from the definition; the tokens as whole numbers."""
    temp, top_p, min_p = (float(torch.tensor(c[k], dtype=torch.float32)) for k in ("temp", "top_p", "min_p"))
    tokens, probs = [], []
    for x, u in zip(s["logits"].double().cpu(), s["u"].double().cpu().tolist()):
        order = sorted(torch.topk(x, min(len(x), 20000)).indices.tolist() if c["top_k"] else range(len(x)),
                       key=lambda i, v=x.tolist(): (-v[i], i))
        order = torch.tensor(order[:c["top_k"] or len(order)])
        w = torch.exp((x[order] - x[order[0]]) / temp)
        if top_p < 1.0:
            before = torch.cat([torch.zeros(1, dtype=torch.float64), torch.cumsum(w, 0)[:-1]])
            order, w = order[before < top_p * w.sum()], w[before < top_p * w.sum()]
        order, w = order[w >= min_p], w[w >= min_p]
        order, at = torch.sort(order)
        upto = torch.cumsum(w[at], 0)
        j = min(int((upto <= u * upto[-1]).sum()), len(order) - 1)
        tokens.append(int(order[j]))
        probs.append(float(w[at][j] / upto[-1]))
    return {"token": None, "prob": torch.tensor(probs, dtype=torch.float64)}
