"""The attention half of a served block as a serving program calls it, next to the experts' half that this framework has:
the residual's addition with a root-mean-square norm, rotary positions, a cache of keys and values in MX4 (4-bit floating
point, a power-of-two scale for each block of 32 along a head), and attention over that cache.

A case is a dict of plain values.  `op` says which operator it goes through:
  norm    s = x + residual (where there is one) and y = s / sqrt(mean(s^2) + eps) * weight
  rotary  pairs of a head's elements turned by position * base^(-2 i / dims), each pair by one of up to three positions of
          its token; `backward`: the gradient carried through
  cache   keys and values of new tokens rounded to MX4 into their slots of the pages, and read back
  attend  each sequence's newest tokens over all that is cached of it: causal, grouped heads, pages in any order, a window
          or none
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
PAIRS = [[v, u] for u in CODES + [-c for c in CODES] for v in CODES + [-c for c in CODES]]  # by byte: low half first
SCALES = [2.0 ** (i - 127) for i in range(255)] + [math.nan]
EPS = 1e-6


def _norm(name, dtype, rows, cols, residual=True):
    return {"op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "residual": residual, **({"name": name} if name else {})}


def _rotary(name, dtype, tokens, heads, head, dims, axes=1, pairing="halves", far=4096, backward=False):
    return {"op": "rotary", "dtype": dtype, "tokens": tokens, "heads": heads, "head": head, "dims": dims, "axes": axes, "pairing": pairing,
            "far": far, "backward": backward, **({"name": name} if name else {})}


def _cache(name, dtype, tokens, heads, head, page):
    return {"op": "cache", "dtype": dtype, "tokens": tokens, "heads": heads, "head": head, "page": page, **({"name": name} if name else {})}


def _attend(name, dtype, sequences, length, rows, heads, kv_heads, head, page, ragged=False, window=0):
    return {"op": "attend", "dtype": dtype, "sequences": sequences, "length": length, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "head": head, "page": page, "ragged": ragged, "window": window, **({"name": name} if name else {})}


def listed():
    return [
        # the tokens of one decoding step: latency
        _norm("norm_step", "bf16", 8, 4096),
        # a prompt's tokens, or a training batch's: one pass over memory
        _norm("norm_prompt", "bf16", 8192, 4096),
        # one decoding step's queries, far into their sequences: latency
        _rotary("rotary_step", "bf16", 8, 32, 128, 128, far=100000),
        # patches of images and frames with a time, a height and a width; a part of each head stays as it is
        _rotary("rotary_video", "f16", 15000, 16, 80, 72, axes=3, pairing="neighbours"),
        # the gradient of a prompt's queries
        _rotary("rotary_backward", "f32", 4096, 32, 128, 128, backward=True),
        # one new token of each of 64 running sequences: latency
        _cache("cache_step", "f16", 64, 8, 128, 64),
        # prompts written into the cache when they arrive, and what was cached of them read back
        _cache("cache_prompt", "bf16", 16384, 8, 128, 64),
        # one new token of one sequence: too few heads to fill the chip
        _attend("attend_token", "bf16", 1, 4000, 1, 32, 8, 128, 64),
        # a full decoding batch of uneven lengths, some slots without a sequence
        _attend("attend_batch", "bf16", 64, 8192, 1, 64, 8, 128, 64, ragged=True),
        # two sequences of very many tokens, small pages
        _attend("attend_long", "f16", 2, 131072, 1, 16, 4, 128, 16),
        # five drafted tokens of each sequence checked at once, through a window, in 32 bits
        _attend("attend_drafts", "f32", 24, 6000, 5, 24, 6, 64, 32, ragged=True, window=2048),
        # prompts of uneven lengths that arrive together: matrix cores
        _attend("attend_prompt", "bf16", 4, 4096, 4096, 32, 8, 128, 64, ragged=True),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    op = rng.choice(["norm", "rotary", "cache", "attend", "attend", "attend"])
    if op == "norm":
        cols = log(17, 8200)
        rows = log(1, min(8192, 2 ** 26 // (cols * SIZE[dtype])))
        return _norm("", dtype, rows, cols if rng.random() < 0.4 else max(64, cols // 64 * 64), residual=rng.random() < 0.7)
    if op == "rotary":
        head = rng.choice([64, 80, 96, 128, 256])
        dims = rng.choice([head, head, head // 2, head - 8])
        tokens = log(1, 16384)
        return _rotary("", dtype, tokens, rng.randint(1, max(1, min(64, 2 ** 27 // (tokens * head * SIZE[dtype])))), head, dims, axes=rng.choice([1, 1, 2, 3]),
                       pairing=rng.choice(["halves", "neighbours"]), far=log(1, 1000000), backward=rng.random() < 0.4)
    head = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128, 48])
    if op == "cache":
        return _cache("", dtype, min(log(1, 16384), 2 ** 26 // (kv_heads * head * (SIZE[dtype] + 1))), kv_heads, head, page)
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    kind = rng.choice(["token", "token", "drafts", "prompt"])
    if kind == "prompt":
        length = log(1, min(2048, 2 ** 24 // (kv_heads * group * head)))
        sequences = rng.randint(1, max(1, min(4, 2 ** 28 // (length * length * kv_heads * group), 2 ** 24 // (length * kv_heads * group * head))))
        rows = length if rng.random() < 0.6 else rng.randint(1, length)
    else:
        sequences = log(1, min(64, 2 ** 21 // (kv_heads * group * head)))
        length = log(1, max(1, min(65536, 2 ** 27 // (sequences * kv_heads * head))))
        rows = 1 if kind == "token" else rng.randint(2, 8)
    return _attend("", dtype, sequences, length, rows, kv_heads * group, kv_heads, head, page, ragged=rng.random() < 0.6,
                   window=rng.choice([0, 0, 0, log(1, length)]))


def _lengths(case):
    """Cached tokens of each sequence, its new ones among them, and how many new ones: sizes, which go with the case."""
    most, count = case["length"], case["sequences"]
    if not case["ragged"]:
        lengths = [most] * count
    else:
        spread = random.Random("%d of %d" % (count, most))
        lengths = [max(1, int(most * spread.uniform(0.02, 1.0))) for _ in range(count)]
        lengths[spread.randrange(count)] = most
        if count >= 16:
            lengths[3], lengths[count - 2] = 0, 1  # a slot without a sequence, and one that has just begun
    return lengths, [min(case["rows"], max(n, 1)) for n in lengths]


def _sections(case):
    """Pairs of a head that turn with each axis: as even as it goes, the first axis with what is left."""
    pairs, axes = case["dims"] // 2, case["axes"]
    return [pairs - pairs // axes * (axes - 1)] + [pairs // axes] * (axes - 1)


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _table(values, device):
    return torch.tensor(values, dtype=torch.float32, device=device)


def _to_mx4(x):
    """Codes and scales of blocks of 32 along the last axis: the scale is 2^(floor(log2 of the largest magnitude) - 2), at least 2^-127;
    elements go to the nearest value, to the even code where two are as near, and to 6 beyond; a block that holds an infinity or NaN is NaN."""
    v = x.float().reshape(*x.shape[:-1], -1, 32)
    power = ((v.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=0)  # biased as a scale byte
    fine = torch.isfinite(v).all(-1)
    scales = torch.where(fine, power, 255)
    a = v.abs() * _table(SCALES[:255], x.device)[254 - power.clamp(max=254)][..., None]
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte())
    code = torch.where(fine[..., None], code + 8 * torch.signbit(v).byte(), 0).to(torch.uint8)
    return (code[..., 0::2] + 16 * code[..., 1::2]).flatten(-2), scales.to(torch.uint8)


def _of_mx4(codes, scales):
    """The values of MX4 blocks, codes [..., 16 * blocks] and scales [..., blocks], in 32 bits."""
    v = _table(PAIRS, codes.device)[codes.int()].view(*scales.shape, 32) * _table(SCALES, codes.device)[scales.int()][..., None]
    return v.flatten(-2)


def _plain_norm(s):
    total = s["x"].float()
    if s["residual"] is not None:
        total = total + s["residual"].float()
    y = (total / torch.sqrt((total * total).mean(1, keepdim=True) + EPS) * s["weight"]).to(s["x"].dtype)
    return {"y": y} if s["residual"] is None else {"y": y, "sum": total.to(s["x"].dtype)}


def _plain_rotary(s):
    c, x = s["case"], s["x"].float()
    half = c["dims"] // 2
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=x.device), torch.tensor(_sections(c), device=x.device), output_size=half)
    rate = torch.exp(torch.arange(half, device=x.device, dtype=torch.float64) * (-math.log(c["base"]) / half))
    angle = s["position"].double()[axis].t() * rate  # in 64 bits: a far position in 32 has no angle left
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["backward"]:
        sin = -sin
    x = x.view(c["tokens"], c["heads"], c["head"])
    part = x[..., : c["dims"]]
    u, v = (part[..., :half], part[..., half:]) if c["pairing"] == "halves" else (part[..., 0::2], part[..., 1::2])
    a, b = u * cos - v * sin, u * sin + v * cos
    turned = torch.cat([a, b], 2) if c["pairing"] == "halves" else torch.stack([a, b], 3).flatten(2)
    return torch.cat([turned, x[..., c["dims"]:]], 2).to(s["x"].dtype).view(c["tokens"], -1)


def _plain_cache(s):
    for name in ("k", "v"):
        codes, scales = _to_mx4(s[name].view(s["case"]["tokens"], s["case"]["heads"], -1))
        s["%s_codes" % name][s["slot"]] = codes
        s["%s_scales" % name][s["slot"]] = scales
    return {name: _of_mx4(s["%s_codes" % name][s["slot"]], s["%s_scales" % name][s["slot"]]).flatten(1).to(s[name].dtype) for name in ("k", "v")}


def _plain_attend(s):
    """All sequences filled up to the longest of them, and to the most new tokens."""
    c, q = s["case"], s["q"]
    kv, group, head, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["head"], c["page"]
    longest, most, count = s["longest"], s["most"], c["sequences"]
    place = torch.arange(longest, device=q.device)
    slot = s["table"].long()[:, place // page] * page + place % page
    k = _of_mx4(s["k_codes"][slot], s["k_scales"][slot]).permute(0, 2, 3, 1).contiguous()  # sequence, head, element, token
    v = _of_mx4(s["v_codes"][slot], s["v_scales"][slot]).permute(0, 2, 1, 3).contiguous()
    length, first = s["length"].long(), s["first"].long()
    fresh = first[1:] - first[:-1]
    step = torch.arange(most, device=q.device)
    row = torch.minimum(first[:-1, None] + step, first[1:, None] - 1)
    rows = q.float().view(-1, kv, group, head)[row].permute(0, 2, 3, 1, 4).reshape(count, kv, group * most, head)
    score = torch.matmul(rows, k).view(count, kv, group, most, longest) * s["scale"]
    last = (length - fresh)[:, None] + step  # the newest place that a row sees
    seen = place <= last[..., None]
    if c["window"]:
        seen = seen & (place > last[..., None] - c["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isneginf(top), 0.0, top))
    y = torch.matmul(p.view(count, kv, group * most, longest), v).view(count, kv, group, most, head)
    y = y / p.sum(-1, keepdim=True).clamp(min=1e-37)
    y = y.permute(0, 3, 1, 2, 4).reshape(count, most, -1)
    return y[step < fresh[:, None]].to(q.dtype)


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _maker(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols, strong=8.0):
    """Normal, with a channel in 64 that is `strong` times as large."""
    big = (torch.rand(cols, generator=g, device="cuda") < 1.0 / 64).float()
    return _normal(g, rows, cols) * (1.0 + (strong - 1.0) * big)


def prepare(case, seed):
    g = _maker(seed)
    s = {"case": dict(case)}
    c, dtype = s["case"], DTYPES[case["dtype"]]
    if c["op"] == "norm":
        s["x"] = _normal(g, c["rows"], c["cols"]).to(dtype)
        s["residual"] = _activations(g, c["rows"], c["cols"], 30.0).to(dtype) if c["residual"] else None
        s["weight"] = 1.0 + 0.2 * _normal(g, c["cols"])
    elif c["op"] == "rotary":
        c["base"] = 10000.0
        s["x"] = _normal(g, c["tokens"], c["heads"] * c["head"]).to(dtype)
        s["position"] = torch.randint(0, c["far"], (c["axes"], c["tokens"]), generator=g, device="cuda", dtype=torch.int32)
    elif c["op"] == "cache":
        width = c["heads"] * c["head"]
        s["k"], s["v"] = _activations(g, c["tokens"], width, 4.0).to(dtype), _normal(g, c["tokens"], width).to(dtype)
        pages = 2 + 2 * ((c["tokens"] + c["page"] - 1) // c["page"])  # others' pages lie between
        order = torch.randperm(pages, generator=g, device="cuda")
        if c["tokens"] <= 64:  # a token of each sequence, each in a page of its own where there are as many
            pages = c["tokens"] * 2
            place = torch.randint(0, c["page"], (c["tokens"],), generator=g, device="cuda")
            s["slot"] = torch.randperm(pages, generator=g, device="cuda")[: c["tokens"]] * c["page"] + place
        else:  # prompts: page after page
            place = torch.arange(c["tokens"], device="cuda")
            s["slot"] = order[place // c["page"]] * c["page"] + place % c["page"]
        s["pages"] = pages
        _empty_pages(s, c["heads"])
    else:
        _fill(s, g, dtype)
    if own:
        _lay_out(s)
    return s


def _empty_pages(s, heads):
    """The cache of the plain forms: codes and scales by slot."""
    c, slots = s["case"], s["pages"] * s["case"]["page"]
    for name in ("k", "v"):
        s["%s_codes" % name] = torch.zeros(slots, heads, c["head"] // 2, dtype=torch.uint8, device="cuda")
        s["%s_scales" % name] = torch.zeros(slots, heads, c["head"] // 32, dtype=torch.uint8, device="cuda")


def _fill(s, g, dtype):
    """Sequences in the cache: keys with a few strong channels, pages in any order; pages past a sequence's end are another's."""
    c = s["case"]
    lengths, fresh = _lengths(c)
    kv, head, page = c["kv_heads"], c["head"], c["page"]
    need = [(n + page - 1) // page for n in lengths]
    s["pages"] = sum(need) + 1
    order = torch.randperm(s["pages"], generator=g, device="cuda")
    width = max(max(need), 1)
    begin = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    column = torch.arange(width, device="cuda")
    s["table"] = order[(begin[:, None] + column).clamp(max=s["pages"] - 1)].int().contiguous()
    s["length"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["first"] = torch.tensor([sum(fresh[:i]) for i in range(len(fresh) + 1)], dtype=torch.int32, device="cuda")
    s["rows"], s["most"], s["longest"], s["scale"] = sum(fresh), max(fresh), max(max(lengths), 1), 1.0 / math.sqrt(head)
    _empty_pages(s, kv)
    slots = s["pages"] * page
    slot = torch.arange(slots, device="cuda")
    if own:
        _lay_out_cache(s)
    for at in range(0, slots, 65536):
        part = slot[at: at + 65536].contiguous()
        k, v = _activations(g, part.numel(), kv * head, 4.0).to(dtype), _normal(g, part.numel(), kv * head).to(dtype)
        for name, x in (("k", k), ("v", v)):
            s["%s_codes" % name][part], s["%s_scales" % name][part] = _to_mx4(x.view(part.numel(), kv, head))
        if own:
            s["cache"].append(k.data_ptr(), v.data_ptr(), s["type"], part.numel(), part.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
            torch.cuda.current_stream().synchronize()
    s["q"] = _normal(g, s["rows"], c["heads"] * head).to(dtype)


def _package(s):
    path = os.path.join(os.getcwd(), "tetris-artifact-evalution_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tetris_amd as T

    s["T"], s["type"] = T, {"f32": T.F32, "f16": T.F16, "bf16": T.BF16}[s["case"]["dtype"]]
    return T


def _lay_out_cache(s):
    T, c = _package(s), s["case"]
    kv = c["kv_heads"] if c["op"] == "attend" else c["heads"]
    s["memory"] = torch.zeros(s["pages"] * T.cache_page_bytes(kv, c["head"], c["page"]), dtype=torch.uint8, device="cuda")
    s["cache"] = T.MX4Cache(s["memory"].data_ptr(), s["pages"], kv, c["head"], page=c["page"])


def _lay_out(s):
    """What a program that serves keeps: the cache in its pages, buffers for outputs, workspace."""
    T, c = _package(s), s["case"]
    if c["op"] == "norm":
        s["out"] = {"y": torch.empty_like(s["x"]), **({"sum": torch.empty_like(s["x"])} if c["residual"] else {})}
    elif c["op"] == "rotary":
        s["out"] = torch.empty_like(s["x"])
        s["rotary"] = T.Rotary(c["head"], dims=c["dims"], base=c["base"], sections=_sections(c),
                               pairing=T.PAIR_HALVES if c["pairing"] == "halves" else T.PAIR_NEIGHBOURS)
    elif c["op"] == "cache":
        _lay_out_cache(s)
        s["out"] = {"k": torch.empty_like(s["k"]), "v": torch.empty_like(s["v"])}
    else:
        s["out"] = torch.empty_like(s["q"])
        s["cache"].prepare(c["heads"], c["sequences"], s["longest"], s["type"], rows=s["rows"], most_rows=s["most"], window=c["window"])


# ---- a pass ---------------------------------------------------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"norm": _plain_norm, "rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend}[c["op"]](s)
    T, out, stream = s["T"], s["out"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm":
        T.rms_norm(s["x"].data_ptr(), out["y"].data_ptr(), s["type"], c["rows"], c["cols"], d_weight=s["weight"].data_ptr(), eps=EPS,
                   d_residual=s["residual"].data_ptr() if c["residual"] else 0, d_sum=out["sum"].data_ptr() if c["residual"] else 0, stream=stream)
    elif c["op"] == "rotary":
        s["rotary"].rotate(s["x"].data_ptr(), out.data_ptr(), s["type"], c["tokens"], c["heads"], s["position"].data_ptr(),
                           backward=c["backward"], stream=stream)
    elif c["op"] == "cache":
        s["cache"].append(s["k"].data_ptr(), s["v"].data_ptr(), s["type"], c["tokens"], s["slot"].data_ptr(), stream=stream)
        s["cache"].read(s["slot"].data_ptr(), out["k"].data_ptr(), out["v"].data_ptr(), s["type"], c["tokens"], stream=stream)
    else:
        s["cache"].attend(s["q"].data_ptr(), out.data_ptr(), s["type"], c["heads"], c["sequences"], s["length"].data_ptr(),
                          s["table"].data_ptr(), s["longest"], d_first=s["first"].data_ptr(), rows=s["rows"], most_rows=s["most"],
                          ld_table=s["table"].shape[1], window=c["window"], scale=s["scale"], stream=stream)
    return out


def _pairs(case):
    """Pairs of a new token and a cached one that it sees, and the cached tokens that some new token sees."""
    pairs = seen = 0
    for n, m in zip(*_lengths(case)):
        w = case["window"] or n + 1
        full = [min(n - m + i + 1, w) for i in (0, m - 1)]
        if full[0] == full[1]:
            pairs += m * max(full[0], 0)
        else:
            pairs += sum(max(0, min(n - m + i + 1, w)) for i in range(m))
        seen += min(n, m - 1 + w)
    return pairs, seen


def work(case):
    c, b = case, SIZE[case["dtype"]]
    if c["op"] == "norm":
        return {"bytes": c["rows"] * c["cols"] * b * (4 if c["residual"] else 2) + 4 * c["cols"], "flops": 5 * c["rows"] * c["cols"]}
    if c["op"] == "rotary":
        return {"bytes": c["tokens"] * (2 * c["heads"] * c["head"] * b + 4 * c["axes"]), "flops": 3 * c["tokens"] * c["heads"] * c["dims"]}
    if c["op"] == "cache":  # codes and scales are the first call's output and the second's input
        values = 2 * c["tokens"] * c["heads"] * c["head"]
        return {"bytes": values * 2 * b + 2 * values * 17 // 32 + 16 * c["tokens"], "flops": 8 * values}
    pairs, seen = _pairs(c)
    return {"bytes": 2 * seen * c["kv_heads"] * c["head"] * 17 // 32 + 2 * sum(_lengths(c)[1]) * c["heads"] * c["head"] * b,
            "flops": 4 * pairs * c["heads"] * c["head"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------


def _exact_values(codes, scales):
    """sign, two bits of exponent, one of mantissa: (1 + m/2) 2^(e-1), or m/2 where e is zero; times 2^(scale - 127)."""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    e, m = ((c >> 1) & 3).double(), (c & 1).double()
    v = torch.where(e > 0, (1 + m / 2) * torch.pow(2.0, e - 1), m / 2) * (1 - 2 * (c >> 3).double())
    return v * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def _exact_rounded(x):
    """x to the values of MX4, straight from the definition: steps of half a power of two, ties to even, at most 6."""
    v = x.double().view(x.shape[0], -1, 32)
    top = v.abs().amax(2, keepdim=True)
    power = torch.pow(2.0, (torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2).clamp(min=-127))
    u = v.abs() / power
    step = torch.pow(2.0, torch.floor(torch.log2(u.clamp(min=1.0))) - 1)
    u = (torch.round(u / step) * step).clamp(max=6.0)
    return (torch.copysign(u, v) * power).view(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "norm":
        total = s["x"].double() + (0.0 if s["residual"] is None else s["residual"].double())
        y = total * torch.rsqrt(total.square().sum(1, keepdim=True) / c["cols"] + EPS) * s["weight"].double()
        return {"y": y} if s["residual"] is None else {"y": y, "sum": total}
    if c["op"] == "rotary":
        y = s["x"].double().view(c["tokens"], c["heads"], c["head"])
        half, pair = c["dims"] // 2, 0
        out = y.clone()
        for axis, size in enumerate(_sections(c)):  # as complex numbers, one pair after another
            for i in range(pair, pair + size):
                at = (i, i + half) if c["pairing"] == "halves" else (2 * i, 2 * i + 1)
                angle = s["position"][axis].double() / c["base"] ** (2.0 * i / c["dims"]) * (-1.0 if c["backward"] else 1.0)
                turned = torch.complex(y[..., at[0]], y[..., at[1]]) * torch.polar(torch.ones_like(angle), angle)[:, None]
                out[..., at[0]], out[..., at[1]] = turned.real, turned.imag
            pair += size
        return out.view(c["tokens"], -1)
    if c["op"] == "cache":
        return {"k": _exact_rounded(s["k"]), "v": _exact_rounded(s["v"])}
    lengths, fresh = _lengths(c)
    group, out = c["heads"] // c["kv_heads"], []
    q, at = s["q"].double().view(s["rows"], c["heads"], c["head"]), 0
    for i, (n, m) in enumerate(zip(lengths, fresh)):
        begin = max(0, n - m - c["window"]) if c["window"] else 0
        y = torch.zeros(m, c["heads"], c["head"], dtype=torch.float64, device="cuda")
        place = torch.arange(begin, n, device="cuda")
        slot = s["table"][i].long()[place // c["page"]] * c["page"] + place % c["page"]
        last = torch.arange(m, device="cuda")[:, None] + (n - m)
        hidden = (place > last) | (place <= last - c["window"] if c["window"] else torch.zeros_like(place > last))
        for h in range(c["kv_heads"] if n > begin else 0):
            k, v = (_exact_values(s["%s_codes" % x][slot, h], s["%s_scales" % x][slot, h]) for x in ("k", "v"))
            for j in range(h * group, h * group + group):
                p = torch.softmax((q[at: at + m, j] @ k.t() * s["scale"]).masked_fill(hidden, -math.inf), 1)
                y[:, j] = torch.nan_to_num(p, nan=0.0) @ v
        out.append(y.view(m, -1))
        at += m
    return torch.cat(out)
