"""The operators on MX4 weights (include/tetris_mx4.h) against their definitions in 64 bits (tests/mx4_plain.py)."""
import numpy as np
import pytest

import mx4_plain as P

T = pytest.importorskip("tetris_amd")
torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (T.F32, torch.float32), "f16": (T.F16, torch.float16), "bf16": (T.BF16, torch.bfloat16)}


def on_gpu(x, kind, ld=None, offset=0):
    """x (numpy) as rows of `ld` elements whose first lies `offset` elements into an allocation; NaN around the rows."""
    rows, cols = x.shape
    ld = ld or cols
    whole = torch.full((offset + rows * ld + 8,), float("nan"), dtype=TYPES[kind][1], device="cuda")
    view = whole[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(torch.from_numpy(np.ascontiguousarray(x)).to(TYPES[kind][1]))
    return view


def numbers(t):
    return t.detach().cpu().double().numpy()


def rounded_to(x, kind):
    return torch.from_numpy(np.asarray(x, np.float64)).to(TYPES[kind][1]).double().numpy()


def within(got, want, far):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= far)
    assert not bad.any(), "%d of %d off, the worst by %g where %g is allowed, at %s" % (
        bad.sum(), bad.size, np.abs(got - want)[bad].max(), far[bad].min(), np.argwhere(bad)[0])


def quantised(x, kind):
    """codes and scales of a tensor view by the library."""
    rows, cols = x.shape
    codes = torch.full((rows, T.mx4_code_bytes(cols)), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows, T.mx4_scale_bytes(cols)), 0xEE, dtype=torch.uint8, device="cuda")
    T.mx4_quantize(x.data_ptr(), TYPES[kind][0], rows, cols, codes.data_ptr(), scales.data_ptr(), ld=x.stride(0))
    return codes, scales


def random_weights(rng, rows, cols, spread=3):
    """MX4 rows with scales 2^-spread .. 2^spread: (codes on the GPU, scales on the GPU, float64 values)."""
    blocks = -(-cols // 32)
    code = rng.integers(0, 16, (rows, blocks, 32)).astype(np.uint8)
    code.reshape(rows, -1)[:, cols:] = 0
    scales = rng.integers(127 - spread, 128 + spread, (rows, blocks)).astype(np.uint8)
    return torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda(), P.values(code, scales, cols)


# ---- quantisation ----


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", [(1, 1, 0, 0), (3, 31, 0, 0), (5, 33, 3, 1), (7, 64, 0, 0), (1, 32, 0, 1), (130, 1000, 0, 0), (9, 2056, 8, 8)])
def test_quantise(kind, rows, cols, pad, offset):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rounded_to(rng.normal(size=(rows, cols)) * np.exp2(rng.integers(-6, 6, (rows, cols))), kind)
    code, scales = P.quantise(x)
    got_codes, got_scales = quantised(on_gpu(x, kind, cols + pad, offset), kind)
    assert np.array_equal(got_scales.cpu().numpy(), scales)
    assert np.array_equal(got_codes.cpu().numpy(), P.packed(code))
    for back in TYPES:
        y = torch.full((rows, cols + pad), 77.0, dtype=TYPES[back][1], device="cuda")
        T.mx4_dequantize(got_codes.data_ptr(), got_scales.data_ptr(), rows, cols, y.data_ptr(), TYPES[back][0], ld=cols + pad)
        assert np.array_equal(numbers(y[:, :cols]), P.values(code, scales, cols))
        assert (y[:, cols:] == 77.0).all()


def test_quantise_ties_range_and_what_is_no_number():
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 4.0, 6.0, 0.0, -0.0]
    beside = [np.nextafter(np.float32(v), np.float32(s)) for v in ties[:8] for s in (0, 9)]
    rows = [np.array((ties + beside + [-v for v in ties])[:32] + [0] * 0, np.float32)]
    for power in (-126, -100, 0, 100, 125):
        rows.append(np.ldexp(np.array(ties + [-v for v in ties] + [4.5] * 8, np.float32), power).astype(np.float32))
    rows.append(np.full(32, 2.0 ** -149, np.float32))  # smaller than any code of the smallest scale
    rows.append(np.array([2.0 ** -128, 2.0 ** -129, 1.5 * 2.0 ** -128] + [0] * 29, np.float32))  # halves of the smallest scale's codes
    rows.append(np.full(32, np.finfo(np.float32).max, np.float32))
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, -0.0, np.float32))
    for odd in (np.nan, np.inf, -np.inf):
        rows.append(np.array([1.0, odd] + [2.0] * 30, np.float32))
    x = np.stack([np.resize(r, 32) for r in rows]).astype(np.float64)
    code, scales = P.quantise(x)
    got_codes, got_scales = quantised(on_gpu(x, "f32"), "f32")
    assert np.array_equal(got_scales.cpu().numpy(), scales)
    assert np.array_equal(got_codes.cpu().numpy(), P.packed(code))
    y = torch.empty(x.shape, dtype=torch.float32, device="cuda")
    T.mx4_dequantize(got_codes.data_ptr(), got_scales.data_ptr(), x.shape[0], 32, y.data_ptr(), T.F32)
    assert np.array_equal(numbers(y), P.values(code, scales, 32), equal_nan=True)


def test_dequantise_every_code_at_every_scale():
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1)).reshape(256, 1, 32)
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    codes = torch.from_numpy(P.packed(code)).cuda()
    s = torch.from_numpy(scales).cuda()
    want = P.values(code, scales, 32)
    for kind in TYPES:
        y = torch.empty(256, 32, dtype=TYPES[kind][1], device="cuda")
        T.mx4_dequantize(codes.data_ptr(), s.data_ptr(), 256, 32, y.data_ptr(), TYPES[kind][0])
        assert np.array_equal(numbers(y), rounded_to(want, kind), equal_nan=True)


# ---- products ----

SIZES = [(1, 32, 32), (1, 4096, 80), (2, 33, 17), (5, 1001, 100), (16, 128, 48), (17, 264, 64), (40, 96, 33), (64, 512, 1000), (65, 128, 31),
         (100, 77, 257), (129, 200, 300), (257, 1032, 70), (300, 64, 520),
         # more rows than are streamed: tiles of 32 rows, of 64, and of 128
         (1030, 1001, 70), (1100, 96, 33), (1500, 200, 2100), (3999, 100, 4091)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(kind, m, k, n):
    rng = np.random.default_rng(m + 3 * k + 5 * n)
    codes, scales, w = random_weights(rng, n, k)
    x = rounded_to(rng.normal(size=(m, k)), kind)
    bias = rng.normal(size=n).astype(np.float32) if (m + n) % 2 else None
    W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), n, k)
    want, _, far = P.product(x, w, kind, bias)
    d_bias = torch.from_numpy(bias).cuda() if bias is not None else None
    for ldx, offset, ldy in ((k, 0, n), (k + 3, 1, n + 5)):
        dx = on_gpu(x, kind, ldx, offset)
        y = torch.full((m, ldy), 55.0, dtype=TYPES[kind][1], device="cuda")
        W.linear(dx.data_ptr(), y.data_ptr(), m, TYPES[kind][0], d_bias=d_bias.data_ptr() if bias is not None else 0, ldx=ldx, ldy=ldy)
        within(numbers(y[:, :n]), want, far)
        assert (y[:, n:] == 55.0).all()
    W.close()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 32), (3, 1001, 65), (64, 256, 100), (65, 128, 300), (130, 96, 40), (300, 520, 257), (513, 1024, 600), (1025, 96, 40), (1300, 520, 257)])
def test_linear_of_rounded_rows(kind, m, k, n):
    rng = np.random.default_rng(m + k + n)
    codes, scales, w = random_weights(rng, n, k)
    x = rounded_to(rng.normal(size=(m, k)) * np.exp2(rng.integers(-3, 4, (m, k))), kind)
    W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), n, k)
    want, _, far = P.product(P.values(*P.quantise(x), k), w, kind)
    for ldx, offset in ((k, 0), (k + 1, 1)):
        dx = on_gpu(x, kind, ldx, offset)
        y = torch.full((m, n), float("nan"), dtype=TYPES[kind][1], device="cuda")
        W.linear(dx.data_ptr(), y.data_ptr(), m, TYPES[kind][0], ldx=ldx, mx4_input=True)
        within(numbers(y), want, far)


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [3, 200, 1100])
def test_linear_where_numbers_are_no_numbers(m, rounded):
    rng = np.random.default_rng(m)
    k, n = 96, 40
    code = rng.integers(1, 8, (n, 3, 32)).astype(np.uint8)  # positive weights
    scales = np.full((n, 3), 127, np.uint8)
    scales[7, 1] = 255
    x = np.abs(rng.normal(size=(m, k))) + 0.1
    x[1, 5], x[2, 40] = np.inf, np.nan
    W = T.MX4Weights(torch.from_numpy(P.packed(code)).cuda().data_ptr(), torch.from_numpy(scales).cuda().data_ptr(), n, k)
    for kind in TYPES:
        y = torch.zeros(m, n, dtype=TYPES[kind][1], device="cuda")
        W.linear(on_gpu(x, kind).data_ptr(), y.data_ptr(), m, TYPES[kind][0], mx4_input=rounded)
        got = numbers(y)
        assert np.isnan(got[:, 7]).all() and np.isnan(got[2]).all()
        rest = np.delete(got, 7, 1)
        assert (np.isnan(rest[1]) if rounded else np.isposinf(rest[1])).all()
        assert np.isfinite(np.delete(rest, [1, 2], 0)).all()


def test_linear_at_the_ends_of_the_scales():
    rng = np.random.default_rng(1)
    k, n = 64, 32
    code = rng.integers(0, 16, (n, 2, 32)).astype(np.uint8)
    for scale, size in ((0, 2.0 ** 40), (60, 1.0), (200, 2.0 ** -90), (254, 2.0 ** -120)):
        scales = np.full((n, 2), scale, np.uint8)
        w = rounded_to(P.values(code, scales, k), "f32")  # 6 * 2^127 is infinite in 32 bits
        d = torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda()
        W = T.MX4Weights(d[0].data_ptr(), d[1].data_ptr(), n, k)
        for m in (2, 150, 1100):
            x = rounded_to(rng.normal(size=(m, k)) * size, "bf16")
            with np.errstate(invalid="ignore"):
                want, _, far = P.product(x, w, "f32")
            for kind in ("f32", "bf16"):
                y = torch.zeros(m, n, dtype=TYPES[kind][1], device="cuda")
                W.linear(on_gpu(x, kind).data_ptr(), y.data_ptr(), m, TYPES[kind][0])
                got, fine = numbers(y), np.isfinite(want)
                assert np.array_equal(got[~fine], want[~fine], equal_nan=True) and (fine.all() or scale == 254)
                within(got[fine], want[fine], (far + P.ROUNDING[kind] * np.abs(want))[fine])


@pytest.mark.parametrize("least,most", [(104, 140), (103, 140), (104, 141), (90, 150)])
def test_f16_rows_and_weights_at_the_ends_of_f16(least, most):
    """Scales 2^-23 .. 2^13 make weights that are exact in f16; others are multiplied in parts."""
    rng = np.random.default_rng(least + most)
    k, n = 128, 48
    code = rng.integers(0, 16, (n, 4, 32)).astype(np.uint8)
    scales = rng.integers(least, most + 1, (n, 4)).astype(np.uint8)
    scales[0, 0], scales[1, 1] = least, most
    scales[2, 2], code[2, 2] = 0, 8  # zeros need no scale
    d = torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda()
    W = T.MX4Weights(d[0].data_ptr(), d[1].data_ptr(), n, k)
    for m in (5, 1100):
        x = rounded_to(rng.normal(size=(m, k)) * 2.0 ** -12, "f16")  # f16's subnormal numbers among them
        want, _, far = P.product(x, P.values(code, scales, k), "f16")
        y = torch.zeros(m, n, dtype=torch.float16, device="cuda")
        W.linear(on_gpu(x, "f16").data_ptr(), y.data_ptr(), m, T.F16)
        fine = np.abs(want) + far < 65504
        within(numbers(y)[fine], want[fine], far[fine])
        assert fine.mean() > 0.3


@pytest.mark.parametrize("kind,m,k", [("bf16", 2200000, 1024), ("f32", 360000, 1024), ("f16", 600000, 1000)])
def test_rows_beyond_32_bit_offsets(kind, m, k):
    """Rows of 4.5 GB as they lie, and of 1.5 GB and 1.2 GB whose parts and copies pass 2^31 bytes."""
    rng = np.random.default_rng(m)
    n = 40
    code = rng.integers(0, 16, (n, -(-k // 32), 32)).astype(np.uint8)
    code.reshape(n, -1)[:, k:] = 0
    scales = rng.integers(90, 160, code.shape[:2]).astype(np.uint8)  # beyond f16
    d = torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda()
    W = T.MX4Weights(d[0].data_ptr(), d[1].data_ptr(), n, k)
    x = torch.empty(m, k, dtype=TYPES[kind][1], device="cuda").normal_() * 2.0 ** -9
    y = torch.empty(m, n, dtype=torch.float32 if kind == "f32" else TYPES[kind][1], device="cuda")
    W.linear(x.data_ptr(), y.data_ptr(), m, TYPES[kind][0])
    rows = np.unique(np.concatenate([rng.integers(0, m, 60), [0, m - 1, m // 2], (2**31 // (2 * k) + np.arange(-2, 3)) % m]))
    at = torch.from_numpy(rows).cuda()
    want, _, far = P.product(numbers(x[at]), P.values(code, scales, k), kind)
    got, fine = numbers(y[at]), np.abs(want) + far < (65504 if kind == "f16" else np.inf)
    within(got[fine], want[fine], far[fine])


def test_experts_of_rows_beyond_32_bit_offsets():
    rng = np.random.default_rng(17)
    tokens, count, width, hidden = 1150000, 3, 1024, 32
    up, down = random_weights(rng, count * 2 * hidden, width), random_weights(rng, count * width, hidden)
    layer = T.ExpertLayer(T.MX4Weights(up[0].data_ptr(), up[1].data_ptr(), 2 * hidden, width, experts=count, gated=True),
                          T.MX4Weights(down[0].data_ptr(), down[1].data_ptr(), width, hidden, experts=count))
    x = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda").normal_() * 0.01
    index = torch.randint(0, count, (tokens, 1), dtype=torch.int32, device="cuda")
    weight = torch.rand(tokens, 1, device="cuda")
    y = torch.empty_like(x)
    layer.run(x.data_ptr(), index.data_ptr(), weight.data_ptr(), y.data_ptr(), tokens, 1, T.BF16)
    rows = np.unique(np.concatenate([rng.integers(0, tokens, 60), [0, tokens - 1], 2**31 // (2 * width) + np.arange(-3, 3)]))
    at = torch.from_numpy(rows).cuda()
    want, far = P.experts(numbers(x[at]), up[2].reshape(count, 2 * hidden, width), down[2].reshape(count, width, hidden), index[at].cpu().numpy(),
                          numbers(weight[at]), "bf16")
    within(numbers(y[at]), want, far)


def test_weights_from_numbers_are_those_from_their_codes():
    rng = np.random.default_rng(2)
    n, k, m = 70, 100, 9
    w = rounded_to(rng.normal(size=(n, k)), "bf16")
    x = rounded_to(rng.normal(size=(m, k)), "f32")
    W = T.MX4Weights.quantize(on_gpu(w, "bf16", k + 1, 1).data_ptr(), T.BF16, n, k, ld=k + 1)
    y = torch.empty(m, n, device="cuda")
    W.linear(on_gpu(x, "f32").data_ptr(), y.data_ptr(), m, T.F32)
    want, _, far = P.product(x, P.values(*P.quantise(w), k), "f32")
    within(numbers(y), want, far)


def test_codes_past_the_last_column_count_for_nothing():
    rng = np.random.default_rng(3)
    n, k, m = 40, 70, 4
    code = rng.integers(0, 16, (n, 3, 32)).astype(np.uint8)
    scales = np.full((n, 3), 127, np.uint8)
    d = torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda()
    W = T.MX4Weights(d[0].data_ptr(), d[1].data_ptr(), n, k)
    x = rounded_to(rng.normal(size=(m, k)), "f32")
    y = torch.empty(m, n, device="cuda")
    W.linear(on_gpu(x, "f32").data_ptr(), y.data_ptr(), m, T.F32)
    want, _, far = P.product(x, P.values(code, scales, k), "f32")
    within(numbers(y), want, far)


# ---- experts ----


def expert_case(rng, tokens, count, top, width, hidden, kind, pick=None, size=1.0, share=1.0, between=None):
    up = random_weights(rng, count * 2 * hidden, width)
    down = random_weights(rng, count * width, hidden)
    x = rounded_to(rng.normal(size=(tokens, width)) * width ** -0.5 / 3 * size, kind)
    index = np.stack([rng.permutation(count)[:top] for _ in range(tokens)]) if pick is None else pick
    weight = (rng.uniform(0.1, 1.0, (tokens, top)) * share).astype(np.float32)
    layer = T.ExpertLayer(T.MX4Weights(up[0].data_ptr(), up[1].data_ptr(), 2 * hidden, width, experts=count, gated=True),
                          T.MX4Weights(down[0].data_ptr(), down[1].data_ptr(), width, hidden, experts=count))
    want, far = P.experts(x, up[2].reshape(count, 2 * hidden, width), down[2].reshape(count, width, hidden), index, weight.astype(np.float64), kind, between)
    return layer, x, index, weight, want, far


def run_experts(layer, x, index, weight, kind, ldx=None, offset=0, stream=0):
    tokens, width = x.shape
    dx = on_gpu(x, kind, ldx, offset)
    di, dw = torch.from_numpy(index.astype(np.int32)).cuda(), torch.from_numpy(weight).cuda()
    y = torch.full((tokens, width), float("nan"), dtype=TYPES[kind][1], device="cuda")
    layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), tokens, index.shape[1], TYPES[kind][0], ldx=ldx or width, stream=stream)
    torch.cuda.synchronize()
    return numbers(y)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,count,top,width,hidden", [
    (1, 4, 2, 64, 32), (1, 1, 1, 33, 5), (3, 8, 3, 100, 48), (20, 70, 4, 128, 40), (17, 3, 3, 256, 72), (64, 8, 2, 264, 100), (50, 60, 8, 96, 31),
    (200, 4, 2, 128, 96), (260, 2, 1, 72, 130), (300, 3, 2, 520, 64),
    # more slots than are streamed, in tiles of 32 rows; of 64 and of 128 in the first product, and in the second
    (600, 3, 2, 520, 64), (1100, 2, 1, 72, 130), (1200, 2, 2, 72, 1040), (3000, 2, 2, 72, 1040), (1200, 2, 2, 2100, 48), (3000, 2, 2, 2100, 48)])
def test_experts(kind, tokens, count, top, width, hidden):
    rng = np.random.default_rng(tokens + count + width)
    layer, x, index, weight, want, far = expert_case(rng, tokens, count, top, width, hidden, kind)
    within(run_experts(layer, x, index, weight, kind), want, far)
    within(run_experts(layer, x, index, weight, kind, width + 1, 1), want, far)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [7, 90, 700])
def test_experts_of_uneven_load(kind, tokens):
    rng = np.random.default_rng(tokens)
    count, top = 5, 2
    pick = np.zeros((tokens, top), int)
    pick[:, 0], pick[:, 1] = 3, np.where(np.arange(tokens) % 9 == 0, 1, 4)  # one has all tokens, one a ninth, two have none
    layer, x, index, weight, want, far = expert_case(rng, tokens, count, top, 96, 64, kind, pick)
    within(run_experts(layer, x, index, weight, kind), want, far)


@pytest.mark.parametrize("tokens", [6, 200, 400])
def test_experts_that_are_none(tokens):
    rng = np.random.default_rng(tokens)
    pick = rng.integers(-2, 6, (tokens, 3))
    pick[0], pick[1] = -1, [2**31 - 1, -2**31, 4]
    layer, x, index, weight, want, far = expert_case(rng, tokens, 4, 3, 64, 40, "bf16", pick)
    got = run_experts(layer, x, index, weight, "bf16")
    within(got, want, far)
    assert (got[:2] == 0).all()


# Two truncated bf16 parts: the second has 8 of the bits that the first, of 8, leaves.
PAIR = 2.0 ** -14, 2.0 ** -125


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,count,top,width,hidden", [(1, 1, 1, 64, 8), (1, 16, 5, 130, 64), (9, 3, 1, 64, 40), (64, 2, 1, 72, 200), (21, 3, 3, 48, 130), (8, 64, 8, 256, 31), (1, 64, 64, 40, 24)])
def test_few_slots_keep_more_than_their_type_between_the_products(kind, tokens, count, top, width, hidden):
    rng = np.random.default_rng(tokens + 5 * hidden)
    layer, x, index, weight, want, far = expert_case(rng, tokens, count, top, width, hidden, kind, between=PAIR)
    within(run_experts(layer, x, index, weight, kind), want, far)
    within(run_experts(layer, x, index, weight, kind, width + 3, 1), want, far)


def test_few_slots_of_f16_go_beyond_its_range_between_the_products():
    rng = np.random.default_rng(23)
    layer, x, index, weight, want, far = expert_case(rng, 6, 4, 2, 96, 64, "f16", size=4000.0, share=1e-7, between=PAIR)
    assert 1.0 < np.abs(want).max() < 60000.0
    within(run_experts(layer, x, index, weight, "f16"), want, far)


@pytest.mark.parametrize("kind", TYPES)
def test_experts_workspace_made_for_more_slots_than_are_few(kind):
    rng = np.random.default_rng(12)
    layer, x, index, weight, want, far = expert_case(rng, 66, 3, 1, 64, 256, kind)
    s = torch.cuda.Stream()
    layer.prepare(66, 1, TYPES[kind][0], stream=s.cuda_stream)
    for tokens in (66, 65, 64, 63):
        dx, y = on_gpu(x[:tokens], kind), torch.zeros(tokens, 64, dtype=TYPES[kind][1], device="cuda")
        di, dw = torch.from_numpy(index[:tokens].astype(np.int32)).cuda(), torch.from_numpy(weight[:tokens]).cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):  # a workspace that had to grow would be refused
            layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), tokens, 1, TYPES[kind][0], stream=s.cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        within(numbers(y), want[:tokens], far[:tokens])


def test_experts_keep_tokens_apart():
    rng = np.random.default_rng(11)
    layer, x, index, weight, want, far = expert_case(rng, 40, 4, 2, 64, 40, "f32")
    x[5, 3] = np.nan
    got = run_experts(layer, x, index, weight, "f32")
    assert np.isnan(got[5]).all()
    within(np.delete(got, 5, 0), np.delete(want, 5, 0), np.delete(far, 5, 0))


# ---- routing ----


def spaced(rng, tokens, experts):
    """Logits of a token on a grid of 1/16: as bf16 they are exact, and some are equal."""
    return rng.integers(-40, 40, (tokens, experts)) / 16.0


def run_route(x, kind, top, bias=None, ld=None, offset=0, **how):
    tokens, experts = x.shape
    r = T.Router(experts, top, **how)
    dx = on_gpu(x, kind, ld, offset)
    index = torch.full((tokens, top), -9, dtype=torch.int32, device="cuda")
    weight = torch.full((tokens, top), -9.0, device="cuda")
    db = None if bias is None else torch.from_numpy(bias).cuda()
    r.route(dx.data_ptr(), TYPES[kind][0], tokens, index.data_ptr(), weight.data_ptr(), d_bias=0 if bias is None else db.data_ptr(), ld=ld)
    return index.cpu().numpy(), numbers(weight)


# exp and the division are within a few units in the last place, the sum of up to 1024 scores within its ten levels of additions
SCORE = 32 * 2.0 ** -24


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (3, 2, 2), (5, 8, 3), (9, 60, 8), (7, 64, 4), (33, 65, 32), (4, 128, 8), (6, 200, 6), (5, 256, 8),
                                               (3, 300, 5), (2, 512, 16), (3, 1000, 8), (2, 1024, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(kind, tokens, experts, top, score):
    rng = np.random.default_rng(tokens * experts)
    x = spaced(rng, tokens, experts)
    for renorm in (False, True):
        index, weight = run_route(x, kind, top, score=T.SCORE_SIGMOID if score == "sigmoid" else T.SCORE_SOFTMAX, renorm=renorm, scale=1.5, ld=experts + 3, offset=1)
        want_index, want = P.route(x, top, score == "sigmoid", renorm=renorm, scale=1.5)
        assert np.array_equal(index, want_index)
        within(weight, want, SCORE * np.abs(want) + 1e-37)


@pytest.mark.parametrize("experts,groups,top_groups,top", [(16, 4, 2, 3), (60, 12, 3, 8), (64, 64, 5, 4), (256, 8, 4, 8), (160, 8, 3, 6), (1024, 16, 1, 32), (12, 2, 2, 4)])
@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_of_groups(experts, groups, top_groups, top, two, with_bias):
    if two and experts == groups:
        pytest.skip("groups of one expert have no second best")
    rng = np.random.default_rng(experts + groups)
    tokens = 12
    # scores are a few thousandths apart at least: sixteenths between -2.5 and 2.5 through the sigmoid, a bias of hundredths that no two sums share
    x = rng.integers(-40, 40, (tokens, experts)) / 16.0 + np.arange(experts) * 2.0 ** -17
    bias = (rng.permutation(experts) * 2.0 ** -14).astype(np.float32) if with_bias else None
    s = P.scores(x, True) + (0 if bias is None else bias.astype(np.float64))
    apart = np.diff(np.sort(s, 1), axis=1).min()
    index, weight = run_route(x, "f32", top, bias, score=T.SCORE_SIGMOID, groups=groups, top_groups=top_groups, group_by=T.GROUP_TWO if two else T.GROUP_MAX)
    want_index, want = P.route(x, top, True, bias, groups, top_groups, two)
    if apart < 2.0 ** -22:  # equal to 32 bits: the choice is checked by what it is worth
        rank = x if bias is None else s
        worth = np.take_along_axis(rank, index, 1), np.take_along_axis(rank, want_index, 1)
        within(worth[0], worth[1], np.full(worth[0].shape, 2.0 ** -20))
    else:
        assert np.array_equal(index, want_index)
        within(weight, want, SCORE * np.abs(want))


def test_route_ties_go_to_the_first():
    x = np.zeros((2, 130))
    index, weight = run_route(x, "bf16", 5)
    assert (index == np.arange(5)).all() and np.allclose(weight, 0.2, rtol=1e-6)
    index, _ = run_route(x, "f32", 5, groups=13, top_groups=2)
    assert (index == np.arange(5)).all()
    x[:, 70:] = 1.0
    index, _ = run_route(x, "f32", 3, bias=np.full(130, 0.25, np.float32), score=T.SCORE_SIGMOID)
    assert (index == [70, 71, 72]).all()
    index, _ = run_route(np.array([[-0.0, 0.0, -1.0]]), "f32", 2)
    assert (index == [0, 1]).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_masked_and_infinite_logits(score):
    inf, nan = np.inf, np.nan
    x = np.full((7, 70), -1.0)
    x[0] = -inf  # nothing left
    x[1] = -inf
    x[1, 66] = 2.0  # one left, two asked for
    x[2] = np.finfo(np.float32).min  # the lowest number in place of -inf
    x[3, 5], x[3, 6], x[3, 9] = inf, inf, -inf
    x[4, 3], x[4, 4] = nan, 5.0
    x[5] = nan
    x[6, 69] = 80.0
    how = dict(score=T.SCORE_SIGMOID if score == "sigmoid" else T.SCORE_SOFTMAX)
    for renorm in (False, True):
        index, weight = run_route(x, "f32", 2, renorm=renorm, **how)
        want_index, want = P.route(x, 2, score == "sigmoid", renorm=renorm)
        assert np.array_equal(index, want_index)
        assert np.array_equal(np.isnan(weight), np.isnan(want))
        fine = ~np.isnan(want)
        within(weight[fine], want[fine], SCORE * want[fine] + 1e-37)
    index, weight = run_route(x[:1], "f32", 2, groups=7, top_groups=2, **how)
    assert (index == [0, 1]).all() and (weight == 0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (5, 8, 3), (9, 60, 8), (4, 65, 32), (3, 256, 8), (2, 1000, 6)])
def test_route_backward(kind, score, renorm, tokens, experts, top):
    rng = np.random.default_rng(tokens + experts)
    x = spaced(rng, tokens, experts)
    sigmoid = score == "sigmoid"
    index, _ = P.route(x, top, sigmoid)
    dw = rng.normal(size=(tokens, top)).astype(np.float32)
    r = T.Router(experts, top, score=T.SCORE_SIGMOID if sigmoid else T.SCORE_SOFTMAX, renorm=renorm, scale=1.5)
    di, dd = torch.from_numpy(index.astype(np.int32)).cuda(), torch.from_numpy(dw).cuda()
    y = torch.full((tokens, experts + 2), 99.0, dtype=TYPES[kind][1], device="cuda")
    dx = on_gpu(x, kind, experts + 1, 1)
    r.backward(dx.data_ptr(), TYPES[kind][0], tokens, di.data_ptr(), dd.data_ptr(), y.data_ptr(), ld=experts + 1, ld_out=experts + 2)
    want = P.route_backward(x, index, dw.astype(np.float64), sigmoid, renorm, 1.5)
    # each gradient is a score times differences of numbers as large as the largest of d, divided by the chosen scores' sum
    s = P.scores(x, sigmoid)
    size = 1.5 * np.abs(dw).max(1, keepdims=True) / (np.take_along_axis(s, index, 1).sum(1, keepdims=True) if renorm else 1.0)
    within(numbers(y[:, :experts]), want, s * size * (top + 32) * 2.0 ** -22 + P.ROUNDING[kind] * np.abs(want) + P.LEAST[kind])
    assert (y[:, experts:] == 99.0).all()
    # and against differences of the weights themselves
    for step in [rng.normal(size=x.shape) for _ in range(3)]:
        h = 1e-5
        if renorm or sigmoid or experts > 1:
            def weights(z):
                c = np.take_along_axis(P.scores(z, sigmoid), index, 1)
                return 1.5 * (c / c.sum(1, keepdims=True) if renorm else c)
            slope = ((weights(x + h * step) - weights(x - h * step)) / (2 * h) * dw).sum()
            got = (numbers(y[:, :experts]) * step).sum()
            room = (np.abs(step) * (s * size * (top + 32) * 2.0 ** -22 + P.ROUNDING[kind] * np.abs(want) + P.LEAST[kind])).sum()
            assert abs(got - slope) <= room + 1e-8 * (1 + np.abs(dw).sum())


def test_route_backward_of_rows_without_scores():
    x = np.full((3, 66), -np.inf)
    x[1, 65] = 1.0
    index = np.array([[0, 1], [65, 0], [-1, 70]], np.int32)
    dw = np.ones((3, 2), np.float32)
    x[2] = 0.5
    for renorm in (False, True):
        y = torch.full((3, 66), 9.0, device="cuda")
        di, dd = torch.from_numpy(index).cuda(), torch.from_numpy(dw).cuda()
        T.Router(66, 2, renorm=renorm).backward(on_gpu(x, "f32").data_ptr(), T.F32, 3, di.data_ptr(), dd.data_ptr(), y.data_ptr())
        assert (numbers(y) == 0).all()


# ---- streams, graphs, nothing to do, refusals that need a handle ----


def test_nothing_to_do():
    codes, scales, _ = random_weights(np.random.default_rng(0), 64, 32)
    W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 64, 32)
    W.linear(0, 0, 0, T.F32)
    W.prepare(0, T.F32)
    T.Router(8, 2).route(0, T.F32, 0, 0, 0)
    T.Router(8, 2).backward(0, T.F32, 0, 0, 0, 0)
    up = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 64, 32, gated=True)
    down = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 32, 32)
    T.ExpertLayer(up, down).run(0, 0, 0, 0, 0, 1, T.F32)


def test_refusals_of_weights_that_do_not_fit():
    codes, scales, _ = random_weights(np.random.default_rng(0), 64, 64)
    d = torch.zeros(4096, device="cuda")
    p = d.data_ptr()
    up = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 64, 64, gated=True)
    plain = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 32, 64)
    pair = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 32, 64, experts=2)

    def refused(call):
        with pytest.raises(T.TetrisError) as e:
            call()
        assert e.value.code == T.EINVAL

    refused(lambda: up.linear(p, p, 1, T.F32))
    refused(lambda: pair.linear(p, p, 1, T.F32))
    refused(lambda: plain.linear(p, p, -1, T.F32))
    refused(lambda: plain.linear(p, p, 1, 3))
    refused(lambda: plain.linear(p, p, 1, T.F32, ldx=63))
    refused(lambda: plain.linear(p, p, 1, T.F32, ldy=31))
    refused(lambda: plain.linear(0, p, 1, T.F32))
    refused(lambda: plain.linear(p, 0, 1, T.F32))
    refused(lambda: plain.linear(p + 2, p, 1, T.F32))
    refused(lambda: T.ExpertLayer(up, up).run(p, p, p, p, 1, 1, T.F32))
    refused(lambda: T.ExpertLayer(plain, plain).run(p, p, p, p, 1, 1, T.F32))
    refused(lambda: T.ExpertLayer(up, pair).run(p, p, p, p, 1, 1, T.F32))
    down = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 64, 32)
    refused(lambda: T.ExpertLayer(up, down).run(p, 0, p, p, 1, 1, T.F32))
    refused(lambda: T.ExpertLayer(up, down).run(p, p, p, p, 1, 0, T.F32))
    refused(lambda: T.ExpertLayer(up, down).run(p, p, p, p, 1, 1, 7))
    refused(lambda: T.ExpertLayer(up, down).prepare(-1, 1, T.F32))


@pytest.mark.parametrize("tokens", [5, 300])
def test_graph_of_a_routed_layer(tokens):
    """Scores' product, routing and experts captured once and replayed on new numbers, with other work between the replays."""
    rng = np.random.default_rng(tokens)
    count, top, width, hidden = 8, 2, 136, 40
    layer, x, _, _, _, _ = expert_case(rng, tokens, count, top, width, hidden, "bf16")
    codes, scales, _ = random_weights(rng, count, width)
    gate = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), count, width)
    router = T.Router(count, top)
    dx = on_gpu(x, "bf16", width + 1)
    logits = torch.empty(tokens, count, dtype=torch.bfloat16, device="cuda")
    index = torch.empty(tokens, top, dtype=torch.int32, device="cuda")
    weight = torch.empty(tokens, top, device="cuda")
    y = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda")

    def step(stream):
        gate.linear(dx.data_ptr(), logits.data_ptr(), tokens, T.BF16, ldx=width + 1, stream=stream)
        router.route(logits.data_ptr(), T.BF16, tokens, index.data_ptr(), weight.data_ptr(), stream=stream)
        layer.run(dx.data_ptr(), index.data_ptr(), weight.data_ptr(), y.data_ptr(), tokens, top, T.BF16, ldx=width + 1, stream=stream)

    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(T.TetrisError) as e:
        with torch.cuda.graph(graph, stream=s):
            step(s.cuda_stream)
    assert e.value.code == T.EINVAL and "prepare" in str(e.value)
    torch.cuda.synchronize()
    gate.prepare(tokens, T.BF16, stream=s.cuda_stream)
    layer.prepare(tokens, top, T.BF16, stream=s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(s.cuda_stream)
    for seed in range(3):
        new = np.random.default_rng(seed).normal(size=x.shape) * 0.1
        dx.copy_(torch.from_numpy(new).to(torch.bfloat16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        first = y.clone(), index.clone(), weight.clone()
        y.zero_()
        step(0)
        torch.cuda.synchronize()
        assert torch.equal(y, first[0]) and torch.equal(index, first[1]) and torch.equal(weight, first[2])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rounded", [False, True])
def test_workspace_made_for_more_rows_is_enough_for_fewer(kind, rounded):
    rng = np.random.default_rng(9)
    k, n = 200, 40
    codes, scales, w = random_weights(rng, n, k)
    s = torch.cuda.Stream()
    for most in (2000, 1000):
        W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), n, k)
        W.prepare(most, TYPES[kind][0], mx4_input=rounded, stream=s.cuda_stream)
        for m in (most, 1025, 1000, 700, 17, 1):
            if m > most:
                continue
            x = rounded_to(rng.normal(size=(m, k)), kind)
            dx = on_gpu(x, kind, k + 1, 1)  # lies badly: is copied or split
            y = torch.zeros(m, n, dtype=TYPES[kind][1], device="cuda")
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                W.linear(dx.data_ptr(), y.data_ptr(), m, TYPES[kind][0], ldx=k + 1, mx4_input=rounded, stream=s.cuda_stream)
            graph.replay()
            torch.cuda.synchronize()
            want, _, far = P.product(P.values(*P.quantise(x), k) if rounded else x, w, kind)
            within(numbers(y), want, far)


@pytest.mark.parametrize("kind", TYPES)
def test_experts_workspace_made_for_more_tokens_is_enough_for_fewer(kind):
    rng = np.random.default_rng(10)
    layer, x, index, weight, want, far = expert_case(rng, 900, 4, 2, 72, 40, kind)
    s = torch.cuda.Stream()
    layer.prepare(900, 2, TYPES[kind][0], stream=s.cuda_stream)
    for tokens in (900, 500, 100, 20, 1):
        dx, y = on_gpu(x[:tokens], kind, 73, 1), torch.zeros(tokens, 72, dtype=TYPES[kind][1], device="cuda")
        di, dw = torch.from_numpy(index[:tokens].astype(np.int32)).cuda(), torch.from_numpy(weight[:tokens]).cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), tokens, 2, TYPES[kind][0], ldx=73, stream=s.cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        within(numbers(y), want[:tokens], far[:tokens])


def test_two_streams_at_once():
    rng = np.random.default_rng(5)
    tokens = 150
    layer, x, index, weight, want, far = expert_case(rng, tokens, 6, 2, 128, 64, "f32")
    dx, di, dw = on_gpu(x, "f32"), torch.from_numpy(index.astype(np.int32)).cuda(), torch.from_numpy(weight).cuda()
    ys = [torch.zeros(tokens, 128, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ys]
    for _ in range(5):
        for s, y in zip(streams, ys):
            layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), tokens, 2, T.F32, stream=s.cuda_stream)
    torch.cuda.synchronize()
    within(numbers(ys[0]), want, far)
    assert torch.equal(ys[0], ys[1])


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tokens", [3, 100])
def test_block_of_experts_end_to_end(tokens, graph):
    from tetris_amd import expert_block

    args = ["--tokens", str(tokens), "--width", "256", "--hidden", "96", "--experts", "12", "--top", "3", "--classes", "50", "--steps", "3"]
    out = expert_block.main(args + (["--graph"] if graph else []))
    # roundings to bf16: what lies between the products and the output of the block, those of the scores; 2^-8 bounds each
    assert out["block_error"] <= 3 * 2.0 ** -8 and out["scores_error"] <= 2.0 ** -8
