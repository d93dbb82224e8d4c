"""Plain 64-bit forms of the 8-bit KV cache operators and of sampling (numpy),
and the inputs their tests share.  Test infrastructure; needs no GPU."""
import math

import numpy as np

F = np.float32


def quantize_rows(x):
    """quantize_acts' arithmetic on fp32 rows (..., hd): codes, scales."""
    x = np.asarray(x, F)
    amax = np.max(np.abs(x), axis=-1)
    live = amax > 0
    with np.errstate(divide="ignore"):
        scale = np.where(live, amax * F(1.0 / 127.0), F(1)).astype(F)
        inv = np.where(live, F(127) / amax, F(1)).astype(F)
    t = (x * inv[..., None]).astype(F)
    q = np.trunc((t + np.copysign(F(0.5), t)).astype(F))
    return np.clip(q, -127, 127).astype(np.int8), scale


def norm_rope(x, w, eps, freqs, scale):
    """Rows x (..., hd) at table rows freqs (..., hd): the norm's sum in 64 bits,
    every fp32 step rounded by itself."""
    x = np.asarray(x, F)
    hd = x.shape[-1]
    if w is not None:
        mean = np.sum(x.astype(np.float64) ** 2, -1, keepdims=True) / hd
        rms = (1.0 / np.sqrt(mean + np.float64(F(eps)))).astype(F)
        x = (x * rms) * (w + F(1))
    c, s = freqs[..., 0::2], freqs[..., 1::2]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([(a * c - b * s) * F(scale), (a * s + b * c) * F(scale)], -1).astype(F)


def tables(pos, hd):
    ang = np.asarray(pos, np.float64)[:, None] * 10000.0 ** (np.arange(hd // 2) * (-2.0 / hd))
    return np.stack([np.cos(ang), np.sin(ang)], -1).reshape(len(pos), hd).astype(F)


def cache(rng, nseq, nkv, clen, hd):
    """(k, v, ks, vs) of rows N(0, 1)."""
    k, ks = quantize_rows(rng.standard_normal((nseq, nkv, clen, hd), dtype=F))
    v, vs = quantize_rows(rng.standard_normal((nseq, nkv, clen, hd), dtype=F))
    return k, v, ks, vs


def rows_of(c, b, h, lo, hi):
    k, v, ks, vs = c
    return (k[b, h, lo:hi].astype(np.float64) * ks[b, h, lo:hi, None].astype(np.float64),
            v[b, h, lo:hi].astype(np.float64) * vs[b, h, lo:hi, None].astype(np.float64))


def attend(q, k, v, asc, cap):
    """One query row: its output and its largest |score| (natural units)."""
    if not len(k):
        return np.zeros(v.shape[-1]), 0.0
    s = (k @ q.astype(np.float64)) * asc
    big = float(np.max(np.abs(s)))
    if cap:
        s = np.tanh(s / cap) * cap
    p = np.exp(s - s.max())
    return (p @ v) / p.sum(), big


def decode(xq, own, lens, asc, cap, slide, prefix=None, plen=0):
    """xq (nseq, nh, hd) -> (out, tolerance); a sequence of length < 0 gives NaN rows."""
    nseq, nh, hd = xq.shape
    nkv = own[0].shape[1]
    out, big, most = np.full(xq.shape, np.nan), 0.0, 1
    for b in range(nseq):
        n = lens[b]
        if n < 0:
            continue
        skip = max(0, plen + n - slide) if slide else 0
        for h in range(nh):
            j = h * nkv // nh
            k, v = rows_of(own, b, j, max(0, skip - plen), n)
            if plen:
                pk, pv = rows_of(prefix, 0, j, min(skip, plen), plen)
                k, v = np.concatenate([pk, k]), np.concatenate([pv, v])
            out[b, h], m = attend(xq[b, h], k, v, asc, cap)
            big, most = max(big, m), max(most, len(k))
    vmax = max(np.max(np.abs(c[1]) * c[3][..., None]) for c in ((own,) if not plen else (own, prefix)))
    return out, tolerance(big, most, vmax)


def prefill(xq, kv, spos, slide, cap, mask):
    nh, ntok, hd = xq.shape
    nkv = kv[0].shape[1]
    out, big = np.empty((ntok, nh, hd)), 0.0
    for h in range(nh):
        k, v = rows_of(kv, 0, h * nkv // nh, 0, spos + ntok)
        for i in range(ntok):
            hi = spos + i + 1 if mask else spos + ntok
            lo = max(0, hi - slide) if mask and slide else 0
            out[i, h], m = attend(xq[h, i], k[lo:hi], v[lo:hi], 1.0, cap)
            big = max(big, m)
    return out.reshape(ntok, nh * hd), tolerance(big, spos + ntok, np.max(np.abs(kv[1]) * kv[3][..., None]))


def tolerance(score, n, vmax):
    """Largest error of an output element for scores up to |score| over n keys and
    values up to vmax.  A score is a handful of fp32 steps of its own size (the
    query's 23-bit form, the digits' sum, the scales, log2 e, the shift by the
    maximum): 8 half steps of 2^-24, which the exponential turns into a relative
    error of the weight; it enters the sum and, against it, the weights' total.
    The weights are multiplied as integers of 24 bits or more, or as two fp16 parts,
    2^-22 of each; a matrix product that adds by cutting off loses 2^-23 a time, over
    32 additions between the sums that are rounded: 2^-18, and the parts, 2^-17 in
    all.  Sums of n terms in fp32: sqrt(n) half steps, and 64 for exp2, the
    products and the final division."""
    return (2.0 ** -24 * (16.0 * score + math.sqrt(n) + 64.0) + 2.0 ** -17) * vmax


def sample(x, u, temperature, top_k, top_p, min_p):
    """One row: (token, prob), in 64 bits."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if temperature == 0:
        return int(np.argmax(x)), 1.0
    if top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.exp((x - top) / np.float64(F(temperature)))
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        before = np.cumsum(w[order]) - w[order]
        order = order[before < np.float64(F(top_p)) * w[order].sum()]
    order = order[w[order] >= np.float64(F(min_p))]
    order = np.sort(order)
    upto = np.cumsum(w[order])
    u = 0.0 if not u > 0 else float(F(u))
    j = min(int(np.searchsorted(upto, u * upto[-1], side="right")), len(order) - 1)
    while w[order[j]] == 0:
        j -= 1
    return int(order[j]), float(w[order[j]] / upto[-1])
