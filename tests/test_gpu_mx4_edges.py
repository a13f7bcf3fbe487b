"""The operators on MX4 weights (include/tetris_mx4.h) at the edges of what they accept, against their definitions in 64 bits
(tests/mx4_plain.py)."""
import threading

import numpy as np
import pytest

import mx4_plain as P

T = pytest.importorskip("tetris_amd")
torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_mx4 import PAIR, SCORE, TYPES, expert_case, numbers, on_gpu, rounded_to, run_experts, run_route, within  # noqa: E402


def weights(rng, rows, cols, least=124, most=130):
    """MX4 rows with scales of `least` to `most`: (codes on the GPU, scales on the GPU, float64 values)."""
    blocks = -(-cols // 32)
    code = rng.integers(0, 16, (rows, blocks, 32), dtype=np.uint8)
    code.reshape(rows, -1)[:, cols:] = 0
    scales = rng.integers(least, most + 1, (rows, blocks), dtype=np.uint8)
    return torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda(), P.values(code, scales, cols)


@pytest.mark.parametrize("kind,top", [("f32", 700), ("f32", 1024), ("f16", 1024), ("bf16", 1024)])
def test_one_token_of_more_slots_than_32_bit_offsets_reach(kind, top):
    """Between the products the numbers' parts of one such token take more than 2 GiB.  All but 200 of the hidden numbers are zero, which keeps the bound narrow."""
    rng = np.random.default_rng(top)
    width, hidden = 8, 1 << 20
    live = np.sort(rng.permutation(hidden)[:200])
    live[-1] = hidden - 1
    few_codes, few_scales, few_up = weights(rng, 400, width, 90, 130)  # not exact in f16
    at = torch.from_numpy(np.concatenate([live, hidden + live])).cuda()
    codes = torch.zeros(2 * hidden, 16, dtype=torch.uint8, device="cuda")
    scales = torch.full((2 * hidden, 1), 127, dtype=torch.uint8, device="cuda")
    codes[at], scales[at] = few_codes, few_scales
    down_codes, down_scales, down = weights(rng, width, hidden)
    layer = T.ExpertLayer(T.MX4Weights(codes.data_ptr(), scales.data_ptr(), 2 * hidden, width, gated=True),
                          T.MX4Weights(down_codes.data_ptr(), down_scales.data_ptr(), width, hidden))
    x = rounded_to(rng.normal(size=(1, width)), kind)
    index = np.zeros((1, top), np.int32)
    index[0, 5::7] = -1
    weight = (rng.uniform(0.1, 1.0, (1, top)) * 1e-3).astype(np.float32)
    dx, di, dw = on_gpu(x, kind), torch.from_numpy(index).cuda(), torch.from_numpy(weight).cuda()
    y = torch.full((1, width), float("nan"), dtype=TYPES[kind][1], device="cuda")
    print("one token,", kind, top, flush=True)
    layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), 1, top, TYPES[kind][0])
    torch.cuda.synchronize()
    # every slot names the one expert: its outputs times the sum of the weights
    between = PAIR if kind == "f16" else (P.ROUNDING[kind], P.LEAST[kind])
    one, off = P.experts(x, few_up[None], down[None][:, :, live], np.zeros((1, 1), int), np.ones((1, 1)), "f32", between)
    total = weight[index == 0].astype(np.float64).sum()
    want = total * one
    far = total * (off + 2.0 ** -22 * top * np.abs(one))
    within(numbers(y), want, far + P.ROUNDING[kind] * (np.abs(want) + far) + P.LEAST[kind])


@pytest.mark.parametrize("tokens,count,top,width,hidden", [(40, 4, 2, 96, 64), (200, 4, 2, 128, 96), (600, 3, 2, 520, 64), (1200, 2, 2, 72, 1040), (3000, 2, 2, 72, 1040), (1200, 2, 2, 2100, 48)])
def test_f16_goes_beyond_its_range_between_the_products(tokens, count, top, width, hidden):
    """More slots than are few: streamed, and in tiles of 32, 64 and 128 rows."""
    rng = np.random.default_rng(tokens + hidden)
    layer, x, index, weight, want, far = expert_case(rng, tokens, count, top, width, hidden, "f16", size=4000.0, share=1e-8, between=PAIR)
    assert 1.0 < np.abs(want).max() < 60000.0
    within(run_experts(layer, x, index, weight, "f16"), want, far)
    within(run_experts(layer, x, index, weight, "f16", width + 3, 1), want, far)


def sigmoid_gradient(x, index, dweight, renorm, scale):
    """The gradient of the weights carried to the logits, and the size of the numbers that it is a difference of; 1 - s from the logit."""
    s, rest = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    c, d = np.take_along_axis(s, index, 1), scale * dweight
    share, size = s, np.abs(d).max(1, keepdims=True)
    if renorm:
        total = c.sum(1, keepdims=True)
        d = d - (d * (c / total)).sum(1, keepdims=True)
        share = s / total
    full = np.zeros_like(s)
    np.put_along_axis(full, index, d, 1)
    return share * rest * full, share * rest * size


def run_backward(x, kind, index, dweight, **how):
    di, dd = torch.from_numpy(index.astype(np.int32)).cuda(), torch.from_numpy(dweight).cuda()
    y = torch.full(x.shape, 99.0, dtype=TYPES[kind][1], device="cuda")
    T.Router(x.shape[1], index.shape[1], **how).backward(on_gpu(x, kind).data_ptr(), TYPES[kind][0], x.shape[0], di.data_ptr(), dd.data_ptr(), y.data_ptr())
    return numbers(y)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("least,most", [(8, 30), (-30, -8), (-30, 30)])
def test_sigmoid_gradient_of_large_logits(kind, renorm, least, most):
    rng = np.random.default_rng(most - least + renorm)
    tokens, experts, top = 20, 70, 6
    x = rounded_to(rng.uniform(least, most, (tokens, experts)), kind)
    index, _ = P.route(x, top, True)
    dweight = rng.normal(size=(tokens, top)).astype(np.float32)
    got = run_backward(x, kind, index, dweight, score=T.SCORE_SIGMOID, renorm=renorm, scale=1.5)
    want, size = sigmoid_gradient(x, index, dweight.astype(np.float64), renorm, 1.5)
    within(got, want, size * (top + 32) * 2.0 ** -22 + P.ROUNDING[kind] * np.abs(want) + P.LEAST[kind])


@pytest.mark.parametrize("score,about", [("softmax", -86), ("sigmoid", -86), ("softmax", -95)])
def test_gradient_of_weights_of_small_scores(score, about):
    """Scores of some 1e-38 and 1e-41, of which the weights are quotients: the softmax's are chosen against the largest logit, as by a bias."""
    rng = np.random.default_rng(87)
    tokens, experts, top = 9, 70, 4
    x = rounded_to(rng.uniform(about - 0.5, about, (tokens, experts)), "f32")
    index = np.stack([1 + rng.permutation(experts - 1)[:top] for _ in range(tokens)])
    dweight = (rng.normal(size=(tokens, top)) * 100).astype(np.float32)
    if score == "softmax":
        x[:, 0] = 0.0
    got = run_backward(x, "f32", index, dweight, score=T.SCORE_SOFTMAX if score == "softmax" else T.SCORE_SIGMOID, scale=1.5)
    # the sum of the exponentials is 1 to 32 bits, and so is the sigmoid's complement: one formula is good for both
    want, size = sigmoid_gradient(x, index, dweight.astype(np.float64), True, 1.5)
    step = 2.0 ** -149 / np.exp(about - 0.5)  # of the scores, relative; a score, the sum and the mean are each off by up to two
    within(got[:, 1:], want[:, 1:], (size * ((top + 32) * 2.0 ** -22 + 8 * step) + P.LEAST["f32"])[:, 1:])
    assert (got[:, 0] == 0).all()


def test_workspace_that_grows_step_by_step_stays_bounded():
    """Batches of one more row each time, as a server without prepare() sees them."""
    rng = np.random.default_rng(4)
    k, n, most = 8192, 32, 300
    codes, scales, w = weights(rng, n, k)
    W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), n, k)
    x = rounded_to(rng.normal(size=(most, k)), "f32")
    dx, y = on_gpu(x, "f32", k + 1, 1), torch.zeros(most, n, device="cuda")  # lies badly: is copied
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for m in range(1, most + 1):
        W.linear(dx.data_ptr(), y.data_ptr(), m, T.F32, ldx=k + 1)
    torch.cuda.synchronize()
    held = before - torch.cuda.mem_get_info()[0]
    # the last buffer is below twice what 300 rows take (4 bytes a number), those kept are no more than it; whole pages of 2 MiB, a dozen buffers
    assert held <= 4 * most * k * 4 + 16 * 2 ** 21
    want, _, far = P.product(x, w, "f32")
    within(numbers(y), want, far)


def test_threads_on_their_own_default_streams_have_their_own_workspaces():
    """hipStreamPerThread is one value that names a stream of each thread."""
    per_thread = 2  # its value, from the HIP headers
    rng = np.random.default_rng(6)
    k, n, m = 8192, 64, 1000
    codes, scales, w = weights(rng, n, k)
    W = T.MX4Weights(codes.data_ptr(), scales.data_ptr(), n, k)
    xs = [rounded_to(rng.normal(size=(m, k)), "f32") for _ in range(2)]
    dxs, ys = [on_gpu(x, "f32", k + 1, 1) for x in xs], [torch.zeros(m, n, device="cuda") for _ in xs]
    torch.cuda.synchronize()
    before, failures = torch.cuda.mem_get_info()[0], []
    ready = threading.Barrier(len(xs))

    def run(dx, y):
        try:
            W.prepare(m, T.F32, stream=per_thread)
            ready.wait(30)
            for _ in range(20):
                W.linear(dx.data_ptr(), y.data_ptr(), m, T.F32, ldx=k + 1, stream=per_thread)
            torch.cuda.synchronize()
        except Exception as e:  # shown by the test's own thread
            failures.append(e)

    threads = [threading.Thread(target=run, args=a) for a in zip(dxs, ys)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    assert before - torch.cuda.mem_get_info()[0] >= 2 * m * k * 4
    for x, y in zip(xs, ys):
        want, _, far = P.product(x, w, "f32")
        within(numbers(y), want, far)


def test_workspace_of_very_many_tokens_stays_bounded():
    """In one pass their numbers before the weighted sum would take 8.6 GB."""
    rng = np.random.default_rng(8)
    tokens, count, top, width, hidden = 260000, 2, 2, 4096, 32
    up, down = weights(rng, count * 2 * hidden, width), weights(rng, count * width, hidden)
    layer = T.ExpertLayer(T.MX4Weights(up[0].data_ptr(), up[1].data_ptr(), 2 * hidden, width, experts=count, gated=True),
                          T.MX4Weights(down[0].data_ptr(), down[1].data_ptr(), width, hidden, experts=count))
    x = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda").normal_() * 0.01
    index = torch.randint(-1, count, (tokens, top), dtype=torch.int32, device="cuda")
    weight, y = torch.rand(tokens, top, device="cuda"), torch.empty_like(x)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    layer.run(x.data_ptr(), index.data_ptr(), weight.data_ptr(), y.data_ptr(), tokens, top, T.BF16)
    torch.cuda.synchronize()
    # 2 GiB of them, and what lies between the products, a sixteenth of that
    assert before - torch.cuda.mem_get_info()[0] <= 2.25 * 2 ** 30
    rows = np.unique(np.concatenate([rng.integers(0, tokens, 60), [0, tokens - 1], (2 ** 31 // (top * width * 4) + np.arange(-12, 3)) % tokens]))
    at = torch.from_numpy(rows).cuda()
    want, far = P.experts(numbers(x[at]), up[2].reshape(count, 2 * hidden, width), down[2].reshape(count, width, hidden), index[at].cpu().numpy(),
                          numbers(weight[at]), "bf16")
    within(numbers(y[at]), want, far)


def scaled_experts(rng, tokens, count, top, width, hidden, up_scales, down_scales):
    """As expert_case of f16, with the ranges of the scales."""
    up, down = weights(rng, count * 2 * hidden, width, *up_scales), weights(rng, count * width, hidden, *down_scales)
    x = rounded_to(rng.normal(size=(tokens, width)) * width ** -0.5 / 3, "f16")
    index = np.stack([rng.permutation(count)[:top] for _ in range(tokens)])
    weight = rng.uniform(0.1, 1.0, (tokens, top)).astype(np.float32)
    layer = T.ExpertLayer(T.MX4Weights(up[0].data_ptr(), up[1].data_ptr(), 2 * hidden, width, experts=count, gated=True),
                          T.MX4Weights(down[0].data_ptr(), down[1].data_ptr(), width, hidden, experts=count))
    want, far = P.experts(x, up[2].reshape(count, 2 * hidden, width), down[2].reshape(count, width, hidden), index, weight.astype(np.float64), "f16", PAIR)
    assert np.abs(want).max() < 60000
    return layer, x, index, weight, want, far


FITS, BEYOND = (124, 130), (90, 130)  # scales of weights that are exact in f16, and of some that are not


@pytest.mark.parametrize("up_scales,down_scales", [(BEYOND, FITS), (FITS, BEYOND), (BEYOND, BEYOND)])
@pytest.mark.parametrize("tokens,count,top,width,hidden", [(20, 8, 2, 96, 40), (60, 3, 2, 136, 64), (600, 3, 2, 520, 64), (1100, 2, 1, 72, 130), (1200, 2, 2, 72, 1040), (3000, 2, 2, 72, 1040),
                                                          (1200, 2, 2, 2100, 48)])
def test_experts_of_f16_whose_weights_are_not_exact_in_it(tokens, count, top, width, hidden, up_scales, down_scales):
    rng = np.random.default_rng(tokens + width)
    layer, x, index, weight, want, far = scaled_experts(rng, tokens, count, top, width, hidden, up_scales, down_scales)
    within(run_experts(layer, x, index, weight, "f16"), want, far)
    within(run_experts(layer, x, index, weight, "f16", width + 1, 1), want, far)


@pytest.mark.parametrize("up_scales,down_scales", [(BEYOND, FITS), (FITS, BEYOND), (FITS, FITS)])
def test_experts_workspace_of_f16_in_parts_is_enough_for_fewer(up_scales, down_scales):
    rng = np.random.default_rng(13)
    layer, x, index, weight, want, far = scaled_experts(rng, 900, 4, 2, 72, 40, up_scales, down_scales)
    s = torch.cuda.Stream()
    layer.prepare(900, 2, T.F16, stream=s.cuda_stream)
    for tokens in (900, 500, 100, 33, 32, 1):
        dx, y = on_gpu(x[:tokens], "f16", 73, 1), torch.zeros(tokens, 72, dtype=torch.float16, device="cuda")
        di, dw = torch.from_numpy(index[:tokens].astype(np.int32)).cuda(), torch.from_numpy(weight[:tokens]).cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):  # a workspace that had to grow would be refused
            layer.run(dx.data_ptr(), di.data_ptr(), dw.data_ptr(), y.data_ptr(), tokens, 2, T.F16, ldx=73, stream=s.cuda_stream)
        for _ in range(2):
            y.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            within(numbers(y), want[:tokens], far[:tokens])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [3, 200, 1100])
def test_linear_beside_numbers_that_are_none(m, rounded, kind):
    """A row with an infinity, one with a NaN and a feature with a NaN block; all other outputs are those of the definition."""
    rng = np.random.default_rng(m)
    k, n = 96, 40
    code = rng.integers(1, 8, (n, 3, 32)).astype(np.uint8)  # positive weights
    scales = np.full((n, 3), 127, np.uint8)
    scales[7, 1] = 255
    x = rounded_to(np.abs(rng.normal(size=(m, k))) + 0.1, kind)
    x[1, 5], x[2, 40] = np.inf, np.nan
    d = torch.from_numpy(P.packed(code)).cuda(), torch.from_numpy(scales).cuda()
    W = T.MX4Weights(d[0].data_ptr(), d[1].data_ptr(), n, k)
    dx, y = on_gpu(x, kind), torch.zeros(m, n, dtype=TYPES[kind][1], device="cuda")
    W.linear(dx.data_ptr(), y.data_ptr(), m, TYPES[kind][0], mx4_input=rounded)
    got = numbers(y)
    assert np.isnan(got[:, 7]).all() and np.isnan(got[2]).all()
    features, rows = np.delete(np.arange(n), 7), np.delete(np.arange(m), [1, 2])
    assert (np.isnan(got[1, features]) if rounded else np.isposinf(got[1, features])).all()
    read = P.values(*P.quantise(x[rows]), k) if rounded else x[rows]
    want, _, far = P.product(read, P.values(code[features], scales[features], k), kind)
    within(got[np.ix_(rows, features)], want, far)


@pytest.mark.parametrize("experts,groups,top_groups,top", [(1024, 16, 4, 32), (1024, 64, 9, 8), (1000, 8, 3, 8), (512, 8, 4, 8)])
@pytest.mark.parametrize("two", [False, True])
def test_route_of_groups_of_many_experts(experts, groups, top_groups, top, two):
    """Ranks that are multiples of 2^-11 and so apart in 32 bits; what pairs of them add up to is where groups could be equal, which is ruled out."""
    rng = np.random.default_rng(experts + groups)
    tokens, size = 5, experts // groups
    x = np.float32(rng.uniform(-3, 3, experts)).astype(np.float64)
    s = P.scores(x[None], True)[0]
    steps = rng.permutation(4096)[:experts]
    bias = (steps * 2.0 ** -11 - s).astype(np.float32)
    best = np.sort(steps.reshape(groups, size), 1)[:, ::-1]
    assert np.unique(best[:, 0] + (best[:, 1] if two else 0)).size == groups
    rows = np.stack([x] * tokens)
    index, weight = run_route(rows, "f32", top, bias, score=T.SCORE_SIGMOID, groups=groups, top_groups=top_groups, group_by=T.GROUP_TWO if two else T.GROUP_MAX)
    want_index, want = P.route(rows, top, True, bias, groups, top_groups, two)
    assert np.array_equal(index, want_index)
    within(weight, want, SCORE * np.abs(want))
