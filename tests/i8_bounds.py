"""How far attention over the 8-bit cache may be from its definition, element by element of the
output, relative to what that element is made of: the tolerance of i8_cases is relative to the
cache's largest value, under which weights and rows far below the largest ones do not show.

For one query row with weights p_t = exp(s_t) and values v_t = vs_t * vc_t, o = sum p v / sum p:

  A relative error d_t of the weights moves o by sum p_t (v_t - o) d_t / sum p, at most 2 d A with
  A = sum p |v| / sum p.  d has these parts:
    - the query's elements are whole multiples of its largest one's 2^-23 (8355000 steps), each off
      by half a step at most, evenly spread: a score moves by asc * ks * qmax * 2^-24 / sqrt(3)
      * |kc| (its standard deviation), taken six times; qmax counts as 1e-31 at least;
    - 8 half steps of fp32 of the score's own size (digits, scales, log2 e, the shift by the
      maximum), and of the cap's tanh, 2^-22 of the capped score;
    - 2^-22 of the exponential's instruction, and as much in tests of two fp16 parts a weight;
  Sums of n weights in fp32: sqrt(n) half steps of A, 64 for the sums' joining and the division.
  `unit`: the weights' products with the value scales, in steps of at most `unit` of the row's
  largest one, off by less than a step (evenly spread: a standard deviation of a half, taken six
  times, over n keys): 3 sqrt(n) unit * max(p vs) * 127 / sum p.  A row of zeros, whose scale is 1,
  counts as one of 2^-32 there.
  `cut`: matrix sums in fp32 that are cut off, 2^-23 a time for 32 times: 2^-18 of A, and of the parts."""
import math

import numpy as np


def attend(q, kc, ks, vc, vs, asc, cap=0.0, unit=0.0, cut=False):
    """One row: its output and the tolerance of each element."""
    q, kc, ks, vc, vs = (np.asarray(a, np.float64) for a in (q, kc, ks, vc, vs))
    n = len(ks)
    s = asc * ks * (kc @ q)
    move = 6 * asc * np.max(ks * np.sqrt((kc * kc).sum(1))) * max(np.max(np.abs(q)), 1e-31) * 2.0 ** -24 / math.sqrt(3)
    d = move + 2.0 ** -24 * 8 * np.max(np.abs(s))
    if cap:
        s = np.tanh(s / cap) * cap
        d += 2.0 ** -22 * np.max(np.abs(s))
    d += 2.0 ** -22 * (2 if cut else 1)
    p = np.exp(s - s.max())
    v = vc * vs[:, None]
    total = p.sum()
    size = p @ np.abs(v) / total
    tol = (2 * d + 2.0 ** -24 * (math.sqrt(n) + 64) + (2.0 ** -17 if cut else 0.0)) * size
    tol += 3 * math.sqrt(n) * unit * np.max(p * np.where(vc.any(1), vs, 2.0 ** -32)) * 127 / total
    return p @ v / total, tol


def check(got, want, tol):
    got = got.cpu().numpy() if hasattr(got, "cpu") else got
    assert np.all(np.isfinite(got))
    over = np.abs(got - want) / np.maximum(tol, 1e-300)
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 1, f"at {at}: {got[at]:.9g} for {want[at]:.9g}, allowed {tol[at]:.3g}"
