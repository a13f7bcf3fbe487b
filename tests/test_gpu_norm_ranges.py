"""The norm (include/tetris_attention.h) of rows whose squares 32 bits do not hold, against 64 bits."""
import numpy as np
import pytest

import attention_plain as P

T = pytest.importorskip("tetris_amd")
torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import out_like, untouched  # noqa: E402
from test_gpu_mx4 import TYPES, numbers, on_gpu, rounded_to, within  # noqa: E402


def norm(x, kind, eps, residual=None, weight=None):
    rows, cols = x.shape
    dx, dr = on_gpu(x, kind), None if residual is None else on_gpu(residual, kind)
    y = torch.full((rows, cols), 77.0, dtype=TYPES[kind][1], device="cuda")
    dw = None if weight is None else torch.from_numpy(weight).float().cuda()
    T.rms_norm(dx.data_ptr(), y.data_ptr(), TYPES[kind][0], rows, cols, eps=eps, d_residual=0 if dr is None else dr.data_ptr(),
               d_weight=0 if dw is None else dw.data_ptr())
    return numbers(y)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 8, 100, 1000, 2048, 4096, 4099, 12000])
@pytest.mark.parametrize("exponent", [-140, -120, -80, -63, -50, 62, 64, 90, 123])
def test_rows_of_very_large_and_very_small_numbers(kind, cols, exponent):
    """Without eps, rows of numbers around 2^exponent, ordinary rows beside them, and one with numbers of all sizes up to that.  The bound is the
    ordinary one: scaling by a power of two is exact."""
    rng = np.random.default_rng(cols)
    exponent = max(exponent, -130) if kind == "bf16" else exponent  # (its least number is 2^-133)
    x = rng.normal(size=(5, cols))
    x[:, 0] = 1.0
    x[1] *= 2.0 ** exponent
    x[2] *= np.exp2(rng.integers(min(exponent, 0), max(exponent, 0) + 1, cols).astype(float))
    x[2, 0] = 2.0 ** exponent
    x[4] *= -2.0 ** exponent
    x, w = rounded_to(x, kind), rounded_to(rng.normal(size=cols), "f32")
    _, _, want, far = P.rms_norm(x, None, w, 0.0, kind)
    # (a product that is below 32 bits' normal numbers is off by half their step)
    within(norm(x, kind, 0.0, weight=w), want, far + 2.0 ** -149 * (1 + np.abs(w)))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [100, 4096, 12000])
@pytest.mark.parametrize("eps", [1e-38, 1e-30, 2.0, 3e38])
def test_eps_beside_them(kind, cols, eps):
    rng = np.random.default_rng(cols + 1)
    x = rng.normal(size=(4, cols)) * np.exp2(np.array([-63.0, -50.0, 63.5, 100.0]))[:, None]
    x, r = rounded_to(x, kind), rounded_to(x * rng.normal(size=x.shape), kind)
    _, _, want, far = P.rms_norm(x, r, None, float(np.float32(eps)), kind)
    within(norm(x, kind, eps, residual=r), want, far + 2.0 ** -149)


def test_rows_that_have_no_norm():
    x = torch.zeros(3, 4096, device="cuda")
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    y = torch.full_like(x, 77.0)
    T.rms_norm(x.data_ptr(), y.data_ptr(), T.F32, 3, 4096, eps=0.0)
    assert y[0].isnan().all() and y[2].isnan().all()  # 0 / 0
    assert y[1, 5].isnan() and (y[1, :5] == 0).all() and (y[1, 6:] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,pad,offset", [(3, 100, 3, 1), (4, 2048, 8, 8), (512, 4096, 0, 0), (514, 4100, 1, 0), (600, 8192, 0, 0), (5, 8200, 8, 0), (3, 20001, 0, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_their_sums(kind, rows, cols, pad, offset, in_place):
    """Every third row large and every third small, their sums written beside the norm or in the residual's place, nothing around them."""
    rng = np.random.default_rng(rows + cols)
    by = np.exp2(np.array([0.0, 80.0, -70.0]))[np.arange(rows) % 3, None]
    x, r = (rounded_to(rng.normal(size=(rows, cols)) * by, kind) for _ in range(2))
    w = rounded_to(rng.normal(size=cols), "f32")
    dw = torch.from_numpy(w).float().cuda()
    ld = cols + pad
    dx, dr = on_gpu(x, kind, ld, offset), on_gpu(r, kind, ld, offset)
    (y, around), (other, around_other) = (out_like(rows, cols, kind, ld, offset) for _ in range(2))
    total = dr if in_place else other
    T.rms_norm(dx.data_ptr(), y.data_ptr(), TYPES[kind][0], rows, cols, d_weight=dw.data_ptr(), eps=0.0, d_residual=dr.data_ptr(), d_sum=total.data_ptr(), ldx=ld,
               ldy=ld, ld_residual=ld, ld_sum=ld)
    s, far_s, want, far = P.rms_norm(x, r, w, 0.0, kind)
    within(numbers(y), want, far)
    within(numbers(total), s, far_s)
    untouched(around, y)
    untouched(around_other, other)
