"""Attention over the cache and the norm at sizes that their other kernels' forms serve: equal shares of one and two tiles of rows over sequences of uneven lengths,
prompts beside single tokens, rows of the norm in great number.  Bounds by the weights' own roundings (tests/attention_bounds.py)."""
import numpy as np
import pytest

import attention_bounds as B
import attention_plain as P

T = pytest.importorskip("tetris_amd")
torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import Case, many, out_like, untouched  # noqa: E402
from test_gpu_mx4 import TYPES, numbers, on_gpu, rounded_to, within  # noqa: E402


def wanted(c, window=0, weights=None):
    """Outputs and bounds of a case's sequences, one below the other."""
    parts = [B.attend(c.q[c.first[s]:c.first[s + 1]].reshape(m, c.heads, c.head), c.k[s], c.v[s], c.head ** -0.5, c.kind, window, weights) for s, m in enumerate(c.fresh)]
    return [np.concatenate([p[i] for p in parts]).reshape(-1, c.heads * c.head) for i in range(2)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head,rows,window", [(128, 1, 0), (128, 3, 0), (64, 4, 0), (96, 3, 700), (32, 4, 0), (192, 1, 0), (256, 2, 0), (128, 3, 900)])
def test_equal_shares_over_uneven_lengths(kind, head, rows, window):
    """48 copies of five sequences by two kv heads of eight heads each: 480 units of up to 43 quanta (13 with a window) and three for each unit's beginning.  Equal
    shares are taken from 16 * 1024 quanta on, for fewer workgroups at once from less; windows have 160 copies."""
    copies = 160 if window else 48
    c, one = many(kind, [5000, 37, 1290, 129, 2600], [rows] * 5, 16, 2, head, 64, copies, seed=head + rows)
    got = c.run(window=window)
    c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v = one
    want, far = wanted(c, window)
    got = got.reshape(copies, *want.shape)
    # a sequence's parts, and with them its roundings, go by where the shares' borders lie: each copy within the bound
    for g in got:
        within(g, want, far)
    assert np.array_equal(c.run(window=window), c.run(window=window))


@pytest.mark.parametrize("kind", TYPES)
def test_single_tokens_with_their_own_bound(kind):
    """Weights of bf16 and f16 calls of few rows have 16 bits, in chunks of one sequence and in several."""
    c = Case(kind, [1, 16, 4000, 150, 33], [1] * 5, 8, 2, 128, 16, seed=4)
    within(c.run(), *wanted(c))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head", [64, 96, 128])
def test_prompts_with_their_own_bound(kind, head):
    """Weights of bf16 calls of many rows have 11 bits."""
    c, one = many(kind, [300, 65], [300, 40], 4, 2, head, 16, 24, seed=head)
    got = c.run()
    c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v = one
    want, far = wanted(c, weights=B.HALF if kind == "bf16" else None)
    for g in got.reshape(24, *want.shape):
        within(g, want, far)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("window", [0, 90])
def test_a_prompt_beside_single_tokens(kind, window):
    """A prompt, one that goes on behind cached tokens, and sequences of one row each: one call, in an order of their own."""
    fresh = [1, 1, 257, 1, 0, 1, 65, 1]
    c = Case(kind, [700, 3, 257, 1290, 12, 64, 400, 1], fresh, 8, 2, 64, 32, seed=window)
    got = c.run(window=window, extra=3)
    want, far = wanted(c, window, B.HALF if kind == "bf16" else None)
    within(got, want, far)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", [(512, 2056, 0, 0), (700, 4096, 8, 8), (512, 4000, 1, 0), (600, 4104, 0, 0), (512, 8192, 0, 0), (513, 5001, 0, 0), (520, 8200, 0, 0),
                                                  (4096, 128, 0, 0), (2000, 96, 3, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_of_many_rows(kind, rows, cols, pad, offset, in_place):
    rng = np.random.default_rng(rows + cols)
    x, r = (rounded_to(rng.normal(size=(rows, cols)) * s, kind) for s in (1.0, 4.0))
    w = rounded_to(rng.normal(size=cols), "f32")
    dw = torch.from_numpy(w).float().cuda()
    dx, dr = on_gpu(x, kind, cols + pad, offset), on_gpu(r, kind, cols + pad, offset)
    y, around = out_like(rows, cols, kind, cols + pad, offset)
    total, around_total = (dr, None) if in_place else out_like(rows, cols, kind, cols + pad, offset)
    T.rms_norm(dx.data_ptr(), y.data_ptr(), TYPES[kind][0], rows, cols, d_weight=dw.data_ptr(), eps=1e-5, d_residual=dr.data_ptr(), d_sum=total.data_ptr(),
               ldx=cols + pad, ldy=cols + pad, ld_residual=cols + pad, ld_sum=cols + pad)
    s, far_s, want, far = P.rms_norm(x, r, w, 1e-5, kind)
    within(numbers(y), want, far)
    within(numbers(total), s, far_s)
    untouched(around, y)
    if not in_place:
        untouched(around_total, total)
