"""The attention half of a block in 64 bits, written from its definitions (numpy, CPU), and how far 32-bit arithmetic and one rounding
to a type may be from it."""
import numpy as np

from mx4_plain import LEAST, ROUNDING

ONE = 2.0 ** -24  # a rounding of 32 bits, relative


def rms_norm(x, residual, weight, eps, kind):
    """sum, y and their bounds.  A sum of squares is a chain of at most cols / 64 + 16 additions in a lane and its partners, all of one
    sign; its root halves that; the sum before it, the division, the root and two products add eight."""
    s = x if residual is None else x + residual
    mean = (s * s).mean(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = s / np.sqrt(mean + eps) * (1.0 if weight is None else weight)
    far = (x.shape[1] / 64 + 24) * ONE * np.abs(y)
    return s, ROUNDING[kind] * np.abs(s) * (1 + 2 * ONE) + ONE * np.abs(s) + LEAST[kind], y, far + ROUNDING[kind] * (np.abs(y) + far) + LEAST[kind]


def rotate(x, positions, dims, sections, base, kind, neighbours=False, by_axis=False, backward=False):
    """x [tokens, heads, head], positions [axes, tokens]: y and its bound.  Cosine and sine are within 2^-22, two roundings of a result
    below one and one of the argument's remainder, and within what 2^-48 of the position turns; a product and a sum in 32 bits each add one."""
    y = x.copy()
    far = np.zeros_like(x)
    pair = 0
    for axis, n in enumerate(sections):
        for i in range(n):
            rate = base ** (-i / n) if by_axis else base ** (-2.0 * pair / dims)
            a = positions[axis].astype(np.float64) * rate * (-1 if backward else 1)
            u, v = (2 * pair, 2 * pair + 1) if neighbours else (pair, pair + dims // 2)
            c, s = np.cos(a)[:, None], np.sin(a)[:, None]
            y[..., u] = x[..., u] * c - x[..., v] * s
            y[..., v] = x[..., u] * s + x[..., v] * c
            off = (2.0 ** -22 + np.abs(positions[axis])[:, None] * 2.0 ** -48 + 3 * ONE) * (np.abs(x[..., u]) + np.abs(x[..., v]))
            far[..., u] = off + ROUNDING[kind] * (np.abs(y[..., u]) + off) + LEAST[kind]
            far[..., v] = off + ROUNDING[kind] * (np.abs(y[..., v]) + off) + LEAST[kind]
            pair += 1
    return y, far


def attend(q, k, v, scale, kind, window=0, absent=()):
    """One sequence: its newest rows q [n, heads, head] over its tokens k, v [length, kv heads, head]; `absent` tokens no row sees.
    y and its bound:
      a score       sums of `head` products, one rounding for each eight of each of up to three parts of q and 40 more, of the size that the
                    magnitudes bound; three roundings (scale, its conversion to powers of two, the product) and one of what is left of the maximum
      a weight      the score's error, as relative; an exponential within 2^-22; f16: in two parts of 8 bits, the last rounded, 2^-16; bf16: so, or
                    in one of 11 bits, 2^-12, and below 2^-21 of the row's largest within 2^-32 of that.  It is relative to
                    the row's largest, and what is below 32 bits' normal numbers, of the exponential or of one of up to three parts, may become
                    zero: 4 times 2^-126 and no more, as the arithmetic's own maximum is not above the row's
      the sums      one rounding for each eight weights of each part and 100 more
    """
    n, heads, head = q.shape
    length, kv = k.shape[0], k.shape[1]
    y, far = np.zeros(q.shape), np.full(q.shape, LEAST[kind])
    here = np.array([j not in set(absent) for j in range(length)], bool)
    for i in range(n):
        p = length - n + i
        see = here & (np.arange(length) <= p) & (np.arange(length) > p - window if window else True)
        if not see.any():
            continue
        for h in range(heads):
            kk, vv = k[see, h // (heads // kv)], v[see, h // (heads // kv)]
            s, size = kk @ q[i, h] * scale, np.abs(kk) @ np.abs(q[i, h]) * abs(scale)
            off = (3 * head / 8 + 40) * 2 * ONE * size + 4 * ONE * np.abs(s)
            w = np.exp(s - s.max())
            ew = np.expm1(off + off.max()) + 2.0 ** -22 + {"f32": 0.0, "f16": 2.0 ** -16, "bf16": 2.0 ** -12}[kind]
            least = 2.0 ** -32 if kind == "bf16" else 2.0 ** -124
            z = w.sum()
            sums = (3 * see.sum() / 8 + 100) * 2 * ONE
            y[i, h] = w @ vv / z
            e = ((w * (ew + sums) + least) @ np.abs(vv) + np.abs(y[i, h]) * (w * (ew + sums)).sum()) / z * 1.01
            far[i, h] = e + ROUNDING[kind] * (np.abs(y[i, h]) + e) + LEAST[kind]
    return y, far
