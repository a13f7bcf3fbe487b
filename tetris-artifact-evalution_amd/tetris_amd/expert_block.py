"""A block of experts served with weights in 4 bits, end to end: `python -m tetris_amd.expert_block [--tokens 64] [--graph]`.

The weights of a router, of the experts and of a classifier are quantised once (MX4Weights.quantize).  A step then is
    logits = x Wr^T            MX4Weights.linear
    index, weight = top(logits)  Router.route
    y = x + sum_j weight_j expert_{index_j}(x)   ExpertLayer.run, and an addition
    scores = y Wc^T + b        MX4Weights.linear
all on one stream; with --graph it is captured once and replayed.  Prints a step's time and how far its outputs are from the
same block computed in 64 bits with the values that the 4-bit codes stand for.  Random weights and inputs; torch provides
memory, streams and the check.
"""
import argparse
import json
import time


def build(torch, T, width, hidden, experts, top, classes, tokens, seed=0):
    """The block's weights, buffers and workspaces on the current device, as a dict."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def weights(n, k, **how):
        w = (torch.randn(how.get("experts", 1) * n, k, generator=g, device="cuda") / k ** 0.5).to(torch.bfloat16)
        return w, T.MX4Weights.quantize(w.data_ptr(), T.BF16, n, k, **how)

    b = dict(width=width, hidden=hidden, experts=experts, top=top, classes=classes, tokens=tokens)
    b["router_w"], b["router"] = weights(experts, width)
    b["up_w"], up = weights(2 * hidden, width, experts=experts, gated=True)
    b["down_w"], down = weights(width, hidden, experts=experts)
    b["head_w"], b["head"] = weights(classes, width)
    b["layer"], b["choice"] = T.ExpertLayer(up, down), T.Router(experts, top)
    b["bias"] = torch.randn(classes, generator=g, device="cuda")
    b["x"] = torch.randn(tokens, width, generator=g, device="cuda").to(torch.bfloat16)
    b["logits"] = torch.empty(tokens, experts, dtype=torch.bfloat16, device="cuda")
    b["index"] = torch.empty(tokens, top, dtype=torch.int32, device="cuda")
    b["weight"] = torch.empty(tokens, top, device="cuda")
    b["y"] = torch.empty_like(b["x"])
    b["scores"] = torch.empty(tokens, classes, dtype=torch.bfloat16, device="cuda")
    return b


def prepare(T, b, stream=0):
    """Workspaces for steps on `stream`."""
    for w in (b["router"], b["head"]):
        w.prepare(b["tokens"], T.BF16, stream=stream)
    b["layer"].prepare(b["tokens"], b["top"], T.BF16, stream=stream)


def step(T, b, stream=0):
    """One pass; torch's current stream has to be `stream` (the addition is torch's)."""
    n = b["tokens"]
    b["router"].linear(b["x"].data_ptr(), b["logits"].data_ptr(), n, T.BF16, stream=stream)
    b["choice"].route(b["logits"].data_ptr(), T.BF16, n, b["index"].data_ptr(), b["weight"].data_ptr(), stream=stream)
    b["layer"].run(b["x"].data_ptr(), b["index"].data_ptr(), b["weight"].data_ptr(), b["y"].data_ptr(), n, b["top"], T.BF16, stream=stream)
    b["y"].add_(b["x"])
    b["head"].linear(b["y"].data_ptr(), b["scores"].data_ptr(), n, T.BF16, d_bias=b["bias"].data_ptr(), stream=stream)


def check(torch, T, b):
    """(error of the block's output, error of its scores), each over the 2-norm, against 64 bits for the experts that the step chose."""

    def values(w, k):
        codes = torch.empty(w.shape[0], T.mx4_code_bytes(k), dtype=torch.uint8, device="cuda")
        scales = torch.empty(w.shape[0], T.mx4_scale_bytes(k), dtype=torch.uint8, device="cuda")
        v = torch.empty(w.shape, dtype=torch.float32, device="cuda")
        T.mx4_quantize(w.data_ptr(), T.BF16, w.shape[0], k, codes.data_ptr(), scales.data_ptr())
        T.mx4_dequantize(codes.data_ptr(), scales.data_ptr(), w.shape[0], k, v.data_ptr(), T.F32)
        return v.double()

    x, f = b["x"].double(), b["hidden"]
    up = values(b["up_w"], b["width"]).view(b["experts"], 2 * f, -1)
    down = values(b["down_w"], f).view(b["experts"], b["width"], f)
    y = x.clone()
    for e in range(b["experts"]):
        t, j = torch.nonzero(b["index"] == e, as_tuple=True)
        h = x[t] @ up[e].t()
        h = torch.nn.functional.silu(h[:, :f]) * h[:, f:]
        y.index_add_(0, t, (h @ down[e].t()) * b["weight"][t, j].double()[:, None])
    scores = b["y"].double() @ values(b["head_w"], b["width"]).t() + b["bias"].double()

    def off(got, want):
        return float((got.double() - want).norm() / want.norm())

    return off(b["y"], y), off(b["scores"], scores)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("tokens", 64), ("width", 2048), ("hidden", 1024), ("experts", 64), ("top", 4), ("classes", 1000), ("steps", 50)):
        p.add_argument("--" + name, type=int, default=default)
    p.add_argument("--graph", action="store_true", help="capture a step and replay it")
    a = p.parse_args(argv)
    import torch

    import tetris_amd as T

    b = build(torch, T, a.width, a.hidden, a.experts, a.top, a.classes, a.tokens)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        prepare(T, b, stream.cuda_stream)
        step(T, b, stream.cuda_stream)
        stream.synchronize()
        run = lambda: step(T, b, stream.cuda_stream)  # noqa: E731
        if a.graph:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(T, b, stream.cuda_stream)
            run = graph.replay
        for _ in range(5):
            run()
        stream.synchronize()
        began = time.perf_counter()
        for _ in range(a.steps):
            run()
        stream.synchronize()
        took = (time.perf_counter() - began) / a.steps
    torch.cuda.synchronize()
    block, scores = check(torch, T, b)
    out = {"us_per_step": round(took * 1e6, 2), "tokens": a.tokens, "graph": a.graph, "block_error": block, "scores_error": scores}
    print(json.dumps(out))
    return out


if __name__ == "__main__":
    main()
