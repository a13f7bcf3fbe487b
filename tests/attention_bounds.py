"""Attention over cached values in 64 bits, and how far it may be from them by the weights that the second product takes (numpy, CPU)."""
import numpy as np

from mx4_plain import LEAST, ROUNDING

ONE = 2.0 ** -24  # a rounding of 32 bits, relative
# a weight's rounding and what is left of one that is too small for it, relative to itself and to the row's largest
PARTS = {"f32": (0.0, 2.0 ** -124), "f16": (2.0 ** -16, 2.0 ** -124), "bf16": (2.0 ** -16, 2.0 ** -124)}  # three bf16 parts, two, two
HALF = (2.0 ** -11, 2.0 ** -32)  # one f16, 2^7 as large as the weight: to nearest in 11 bits, down to steps of 2^-24


def attend(q, k, v, scale, kind, window=0, weights=None):
    """One sequence: its newest rows q [n, heads, head] over its tokens k, v [length, kv heads, head].  y and its bound:
      a score    3 head / 8 + 40 roundings of 2 ONE, of the size that its products' magnitudes bound (three parts of q at most, a sum of eight products at a
                 time), and four of the score itself (scale, its conversion to powers of two, the product, what is left of the maximum)
      a weight   the score's error and the maximum's, as relative; an exponential within 2^-22; then `weights`
      the sums   3 / 8 of a rounding of 2 ONE a token and 100 more
    """
    n, heads, head = q.shape
    length, kv = k.shape[0], k.shape[1]
    rounding, least = PARTS[kind] if weights is None else weights
    at = np.arange(length)[None] - (length - n + np.arange(n))[:, None]
    see = (at <= 0) & (at > -window if window else True)
    y, far = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        kk, vv = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = np.where(see, q[:, h] @ kk.T * scale, -np.inf)
        top = s.max(1, initial=-np.inf, keepdims=True)
        some = np.isfinite(top)
        size = np.abs(q[:, h]) @ np.abs(kk).T * abs(scale)
        off = np.where(see, (3 * head / 8 + 40) * 2 * ONE * size + 4 * ONE * np.abs(np.where(see, s, 0.0)), 0.0)
        w = np.exp(s - np.where(some, top, 0.0))
        z = np.where(some, w.sum(1, keepdims=True), 1.0)
        wrong = w * (np.expm1(off + off.max(1, initial=0.0, keepdims=True)) + 2.0 ** -22 + rounding + (3 * see.sum(1, keepdims=True) / 8 + 100) * 2 * ONE)
        y[:, h] = w @ vv / z
        e = ((wrong + least * see) @ np.abs(vv) + np.abs(y[:, h]) * wrong.sum(1, keepdims=True)) / z * 1.01
        far[:, h] = e + ROUNDING[kind] * (np.abs(y[:, h]) + e) + LEAST[kind]
    return y, far
