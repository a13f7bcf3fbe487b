"""A block of experts served with weights in 4 bits, end to end: `python -m tetris_amd.expert_block [--tokens 64] [--context 1000] [--graph]`.

The weights of a router, of the experts and of a classifier are quantised once (MX4Weights.quantize), and with --context N those
of an attention before the experts, over a cache in MX4 that holds N tokens of each of `tokens` sequences.  With it a step begins with
    h, x = norm(x)             rms_norm
    q, k, v = h Wa^T           MX4Weights.linear
    q, k turned, k and v into the cache   Rotary.rotate, MX4Cache.append
    a = attention of q over the cache     MX4Cache.attend
    h, x = norm(a Wo^T + x)    MX4Weights.linear, rms_norm with the residual
and the experts' part takes h in x's place.  A step then is
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


PAGE = 64  # tokens of a page of the cache


def build(torch, T, width, hidden, experts, top, classes, tokens, seed=0, context=0, heads=16, kv_heads=4, head=128):
    """The block's weights, buffers and workspaces on the current device, as a dict; context: cached tokens of each token's sequence,
    the token itself among them, or no attention."""
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
    b["context"] = context
    if context:
        b.update(heads=heads, kv_heads=kv_heads, head_size=head)
        qw, kw = heads * head, kv_heads * head
        b["in_w"], b["in"] = weights(qw + 2 * kw, width)
        b["out_w"], b["out"] = weights(width, qw)
        b["gain"] = [1.0 + 0.1 * torch.randn(width, generator=g, device="cuda") for _ in range(2)]
        each = -(-context // PAGE)
        b["memory"] = torch.empty(tokens * each * T.cache_page_bytes(kv_heads, head, PAGE), dtype=torch.uint8, device="cuda")
        b["cache"] = T.MX4Cache(b["memory"].data_ptr(), tokens * each, kv_heads, head, page=PAGE)
        b["rotary"] = T.Rotary(head)
        b["table"] = torch.randperm(tokens * each, generator=g, device="cuda").int().view(tokens, each).contiguous()
        b["length"] = torch.full((tokens,), context, dtype=torch.int32, device="cuda")
        place = torch.arange(context, device="cuda")
        slots = b["table"].long()[:, place // PAGE] * PAGE + place % PAGE
        b["slot"], b["position"] = slots[:, -1].contiguous(), b["length"] - 1
        b["past"] = torch.randn(tokens, context, 2, kw, generator=g, device="cuda").to(torch.bfloat16)  # (its last token is this step's)
        for s, past in zip(slots, b["past"]):
            k, v, s = past[:, 0].contiguous(), past[:, 1].contiguous(), s.contiguous()
            b["cache"].append(k.data_ptr(), v.data_ptr(), T.BF16, context, s.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
            torch.cuda.current_stream().synchronize()
        rows = torch.empty(tokens, qw + 2 * kw, dtype=torch.bfloat16, device="cuda")
        b["qkv"], b["q"], b["k"], b["a"] = rows, torch.empty_like(rows[:, :qw]).contiguous(), torch.empty_like(rows[:, :kw]).contiguous(), torch.empty_like(rows[:, :qw]).contiguous()
        b["h"], b["attended"], b["sum"] = (torch.empty_like(b["x"]) for _ in range(3))
    return b


def prepare(T, b, stream=0):
    """Workspaces for steps on `stream`."""
    for w in (b["router"], b["head"]):
        w.prepare(b["tokens"], T.BF16, stream=stream)
    b["layer"].prepare(b["tokens"], b["top"], T.BF16, stream=stream)
    if b["context"]:
        for w in (b["in"], b["out"]):
            w.prepare(b["tokens"], T.BF16, stream=stream)
        b["cache"].prepare(b["heads"], b["tokens"], b["context"], T.BF16, stream=stream)


def attend(T, b, stream=0):
    """The attention's part of a step: b["h"], what the experts take, and b["sum"], what their output is added to."""
    n, width, kv = b["tokens"], b["width"], b["kv_heads"]
    qw, kw = b["heads"] * b["head_size"], kv * b["head_size"]
    rows = b["qkv"].data_ptr()
    T.rms_norm(b["x"].data_ptr(), b["h"].data_ptr(), T.BF16, n, width, d_weight=b["gain"][0].data_ptr(), stream=stream)
    b["in"].linear(b["h"].data_ptr(), rows, n, T.BF16, stream=stream)
    for to, at, heads in (("q", 0, b["heads"]), ("k", qw, kv)):
        b["rotary"].rotate(rows + 2 * at, b[to].data_ptr(), T.BF16, n, heads, b["position"].data_ptr(), ldx=qw + 2 * kw, stream=stream)
    b["cache"].append(b["k"].data_ptr(), rows + 2 * (qw + kw), T.BF16, n, b["slot"].data_ptr(), ldv=qw + 2 * kw, stream=stream)
    b["cache"].attend(b["q"].data_ptr(), b["a"].data_ptr(), T.BF16, b["heads"], n, b["length"].data_ptr(), b["table"].data_ptr(), b["context"],
                      stream=stream)
    b["out"].linear(b["a"].data_ptr(), b["attended"].data_ptr(), n, T.BF16, stream=stream)
    T.rms_norm(b["attended"].data_ptr(), b["h"].data_ptr(), T.BF16, n, width, d_weight=b["gain"][1].data_ptr(), d_residual=b["x"].data_ptr(),
               d_sum=b["sum"].data_ptr(), stream=stream)


def step(T, b, stream=0):
    """One pass; torch's current stream has to be `stream` (the addition is torch's)."""
    n = b["tokens"]
    if b["context"]:
        attend(T, b, stream)
    x, residual = (b["h"], b["sum"]) if b["context"] else (b["x"], b["x"])
    b["router"].linear(x.data_ptr(), b["logits"].data_ptr(), n, T.BF16, stream=stream)
    b["choice"].route(b["logits"].data_ptr(), T.BF16, n, b["index"].data_ptr(), b["weight"].data_ptr(), stream=stream)
    b["layer"].run(x.data_ptr(), b["index"].data_ptr(), b["weight"].data_ptr(), b["y"].data_ptr(), n, b["top"], T.BF16, stream=stream)
    b["y"].add_(residual)
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

    f = b["hidden"]
    x, y = (b["h"].double(), b["sum"].double()) if b["context"] else (b["x"].double(), b["x"].double().clone())
    up = values(b["up_w"], b["width"]).view(b["experts"], 2 * f, -1)
    down = values(b["down_w"], f).view(b["experts"], b["width"], f)
    for e in range(b["experts"]):
        t, j = torch.nonzero(b["index"] == e, as_tuple=True)
        h = x[t] @ up[e].t()
        h = torch.nn.functional.silu(h[:, :f]) * h[:, f:]
        y.index_add_(0, t, (h @ down[e].t()) * b["weight"][t, j].double()[:, None])
    scores = b["y"].double() @ values(b["head_w"], b["width"]).t() + b["bias"].double()

    def off(got, want):
        return float((got.double() - want).norm() / want.norm())

    return off(b["y"], y), off(b["scores"], scores)


def check_attention(torch, T, b):
    """Errors of the attention's queries, outputs and sum over the 2-norm, each against 64 bits from what the operator before it gave."""
    n, heads, kv, head = b["tokens"], b["heads"], b["kv_heads"], b["head_size"]
    x, rows = b["x"].double(), b["qkv"].double()
    angle = b["position"].double()[:, None] * 10000.0 ** (-torch.arange(head // 2, device="cuda", dtype=torch.float64) / (head // 2))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(v):
        z = torch.complex(*v.view(n, -1, head).chunk(2, 2)) * turn
        return torch.cat([z.real, z.imag], 2).view(n, -1)

    q = turned(rows[:, : heads * head])
    past = b["past"].clone()
    past[:, -1, 0], past[:, -1, 1] = b["k"], b["qkv"][:, (heads + kv) * head:]
    flat = past.permute(2, 0, 1, 3).reshape(-1, kv * head).contiguous()
    codes = torch.empty(flat.shape[0], T.mx4_code_bytes(kv * head), dtype=torch.uint8, device="cuda")
    scales = torch.empty(flat.shape[0], T.mx4_scale_bytes(kv * head), dtype=torch.uint8, device="cuda")
    held = torch.empty(flat.shape, dtype=torch.float32, device="cuda")
    T.mx4_quantize(flat.data_ptr(), T.BF16, flat.shape[0], kv * head, codes.data_ptr(), scales.data_ptr())
    T.mx4_dequantize(codes.data_ptr(), scales.data_ptr(), flat.shape[0], kv * head, held.data_ptr(), T.F32)
    k, v = held.double().view(2, n, b["context"], kv, 1, head).expand(-1, -1, -1, -1, heads // kv, -1).reshape(2, n, b["context"], heads, head).permute(0, 1, 3, 2, 4)
    p = torch.softmax((b["q"].double().view(n, heads, 1, head) * k).sum(-1) * head ** -0.5, -1)
    a = (p[..., None] * v).sum(2).view(n, -1)

    def off(got, want):
        return float((got.double() - want).norm() / want.norm())

    return off(b["q"], q), off(b["a"], a), off(b["sum"], x + b["attended"].double())


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("tokens", 64), ("width", 2048), ("hidden", 1024), ("experts", 64), ("top", 4), ("classes", 1000), ("steps", 50), ("context", 0)):
        p.add_argument("--" + name, type=int, default=default)
    p.add_argument("--graph", action="store_true", help="capture a step and replay it")
    a = p.parse_args(argv)
    import torch

    import tetris_amd as T

    b = build(torch, T, a.width, a.hidden, a.experts, a.top, a.classes, a.tokens, context=a.context)
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
    if a.context:
        out["context"] = a.context
        out["query_error"], out["attention_error"], out["sum_error"] = check_attention(torch, T, b)
    print(json.dumps(out))
    return out


if __name__ == "__main__":
    main()
