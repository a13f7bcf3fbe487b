"""The operators on MX4 weights in 64 bits, written from their definitions (numpy, CPU)."""
import numpy as np

CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([CODES, -CODES])
# half a unit in the last place of a number in [1, 2)
ROUNDING = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # smallest step of a type


def quantise(x):
    """codes [rows, blocks, 32] (0..15) and scales [rows, blocks] of a float64 matrix that holds numbers of at most 32 bits."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    fine = np.isfinite(v).all(2)
    a = np.where(fine[..., None], np.abs(v), 0.0)
    top = a.max(2)
    exponent = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1, -1000)
    power = np.maximum(exponent - 2, -127)
    u = np.ldexp(a, -power[..., None])
    far = np.abs(u[..., None] - CODES)  # nearest code, the even one where two are as near
    best = far.min(-1, keepdims=True)
    near = far == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = np.where(fine[..., None], code + 8 * np.signbit(v), 0)
    return code.astype(np.uint8), np.where(fine, power + 127, 255).astype(np.uint8)


def packed(code):
    return (code[..., 0::2] | code[..., 1::2] << 4).reshape(code.shape[0], -1)


def unpacked(codes):
    return np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)


def values(code, scales, cols):
    """float64 values of codes [..., blocks, 32] and scales [..., blocks]."""
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    v = VALUES[code] * s[..., None]
    return v.reshape(*scales.shape[:-1], -1)[..., :cols]


def product(x, w, kind, bias=None):
    """x w^T (+ bias) and how far sums in 32 bits and one rounding to `kind` may be from it: a sum takes at most a rounding for each
    eight products of each of the up to three parts of x, and forty where stretches are joined, of a size that the sum of the magnitudes bounds."""
    y = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    if bias is not None:
        y = y + bias
        size = size + np.abs(bias)
    sums = (3 * x.shape[1] / 8 + 40) * 2.0 ** -23 * size
    return y, sums, sums + ROUNDING[kind] * (np.abs(y) + sums) + LEAST[kind]


def experts(x, up, down, index, weight, kind, between=None):
    """The experts' products and their bound; up [E, 2F, D], down [E, D, F].  between: how far (relative, absolute) the numbers between the products
    may be off, if not by the rounding to `kind`."""
    f = down.shape[2]
    rel, least = between or (ROUNDING[kind], LEAST[kind])
    y, far = np.zeros((x.shape[0], down.shape[1])), np.zeros((x.shape[0], down.shape[1]))
    with np.errstate(over="ignore"):
        for e in range(up.shape[0]):
            t, j = np.nonzero(index == e)
            if not t.size:
                continue
            h, off, _ = product(x[t], up[e], "f32")
            gate, more, eg, eu = h[:, :f], h[:, f:], off[:, :f], off[:, f:]
            act = gate / (1 + np.exp(-gate))
            eg = 1.1 * eg + np.abs(act) * (2.0 ** -21 + 2.0 ** -23 * np.abs(gate))  # silu's slope is below 1.1; exp of a rounded argument
            h = act * more
            eh = eg * np.abs(more) + np.abs(act) * eu + eg * eu
            eh = eh + (rel + 2.0 ** -23) * (np.abs(h) + eh) + least
            z, sums, _ = product(h, down[e], "f32")
            ez = sums + eh @ np.abs(down[e]).T * 1.01
            w = weight[t, j][:, None]
            np.add.at(y, t, w * z)  # a token may name an expert twice
            np.add.at(far, t, np.abs(w) * ez + 2.0 ** -22 * index.shape[1] * np.abs(w * z))
    return y, far + ROUNDING[kind] * (np.abs(y) + far) + LEAST[kind]


def scores(x, sigmoid):
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            return 1 / (1 + np.exp(-x))
        top = np.where(np.isnan(x), -np.inf, x).max(1, keepdims=True)
        e = np.where(x == top, 1.0, np.exp(x - top))
        e = np.where(np.isneginf(top) & ~np.isnan(x), 0.0, e)
        total = e.sum(1, keepdims=True)
        return np.where(total == 0, 0.0, e / np.where(total == 0, 1.0, total))


def route(x, top, sigmoid=False, bias=None, groups=1, top_groups=1, two=False, renorm=True, scale=1.0):
    s = scores(x, sigmoid)
    both = s + (0 if bias is None else bias)
    rank = np.where(np.isnan(x), -np.inf, x) if bias is None else np.where(np.isnan(both), -np.inf, both)
    both = np.where(np.isnan(both), -np.inf, both)
    index = np.zeros((x.shape[0], top), int)
    for t in range(x.shape[0]):
        allowed = list(range(x.shape[1]))
        if groups > 1:
            size = x.shape[1] // groups
            of = lambda g: np.sort((both if two else rank)[t, g * size:(g + 1) * size])[::-1]  # noqa: E731
            best = [of(g)[0] + of(g)[1] if two else of(g)[0] for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
            allowed = [e for e in allowed if e // size in kept]
        index[t] = sorted(allowed, key=lambda e: (-rank[t, e], e))[:top]
    w = np.take_along_axis(s, index, 1)
    if renorm:
        total = w.sum(1, keepdims=True)
        w = np.where(total == 0, 0.0, w / np.where(total == 0, 1.0, total))
    return index, scale * w


def route_backward(x, index, dweight, sigmoid=False, renorm=True, scale=1.0):
    s = scores(x, sigmoid)
    c = np.take_along_axis(s, index, 1)
    d = scale * dweight
    if renorm:
        total = c.sum(1, keepdims=True)
        d = np.where(total == 0, 0.0, (d - (d * c).sum(1, keepdims=True) / np.where(total == 0, 1, total)) / np.where(total == 0, 1, total))
    full = np.zeros_like(s)
    np.put_along_axis(full, index, d, 1)
    return s * (1 - s) * full if sigmoid else s * (full - (s * full).sum(1, keepdims=True))
