"""tests/attention_bounds.py against the other form in 64 bits (tests/attention_plain.py), and its roundings against numbers rounded on the CPU."""
import numpy as np
import pytest

import attention_bounds as B
import attention_plain as P


@pytest.mark.parametrize("n,length,window", [(1, 1, 0), (3, 40, 0), (40, 40, 7), (9, 4, 0), (2, 0, 0), (5, 33, 3)])
def test_the_same_outputs(n, length, window):
    rng = np.random.default_rng(n + length)
    q, k, v = rng.normal(size=(n, 6, 32)), rng.normal(size=(length, 2, 32)), rng.normal(size=(length, 2, 32))
    for kind, weights in (("f32", None), ("f16", None), ("bf16", (2.0 ** -12, 2.0 ** -32))):
        y, far = B.attend(q, k, v, 0.3, kind, window, weights)
        want, bound = P.attend(q, k, v, 0.3, kind, window)
        assert np.allclose(y, want, rtol=1e-12, atol=1e-15) and np.allclose(far, bound, rtol=1e-6)


def test_a_rounding_to_f16_is_within_two_to_the_minus_eleven_and_no_less():
    x = np.linspace(1, 2, 100001)
    off = np.abs(x.astype(np.float16).astype(np.float64) - x) / x
    assert 2.0 ** -12 < off.max() <= B.HALF[0]
    small = np.linspace(0, 2.0 ** -14, 10001)
    assert np.abs(small.astype(np.float16).astype(np.float64) - small).max() / 2.0 ** 7 <= B.HALF[1]


def test_two_bf16_parts_are_within_two_to_the_minus_sixteen():
    x = np.random.default_rng(0).uniform(1, 2, 100000).astype(np.float32)
    high = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    left = x - high
    low = ((left.view(np.uint32) + 0x7fff + (left.view(np.uint32) >> 16 & 1)) & 0xffff0000).view(np.float32)  # to nearest even
    off = np.abs(high.astype(np.float64) + low - x) / x
    assert 2.0 ** -18 < off.max() <= B.PARTS["bf16"][0]
