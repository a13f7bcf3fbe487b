"""The attention half of a block (include/tetris_attention.h) against its definitions in 64 bits (tests/attention_plain.py)."""
import numpy as np
import pytest

import attention_plain as P
import mx4_plain as X

T = pytest.importorskip("tetris_amd")
torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_mx4 import TYPES, numbers, on_gpu, rounded_to, within  # noqa: E402


def out_like(rows, cols, kind, ld=None, offset=0):
    """An output's rows and the whole allocation around them, filled with 77."""
    ld = ld or cols
    whole = torch.full((offset + rows * ld + 8,), 77.0, dtype=TYPES[kind][1], device="cuda")
    return whole[offset:offset + rows * ld].view(rows, ld)[:, :cols], whole


def untouched(whole, view):
    view.fill_(77.0)
    assert (whole == 77.0).all()


# ---- norm ----


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", [(1, 1, 0, 0), (3, 8, 0, 0), (5, 33, 3, 1), (2, 512, 8, 8), (7, 513, 0, 0), (130, 1000, 0, 0), (3, 2048, 0, 0),
                                                  (2, 2056, 8, 0), (2, 4096, 0, 0), (2, 4099, 1, 3), (1, 8192, 0, 0), (3, 12000, 0, 0), (1, 20001, 0, 0)])
@pytest.mark.parametrize("form", ["plain", "residual", "in place", "no sum"])
def test_norm(kind, rows, cols, pad, offset, form):
    rng = np.random.default_rng(rows * 7 + cols)
    x, r = (rounded_to(rng.normal(size=(rows, cols)) * s, kind) for s in (1.0, 4.0))
    w = rounded_to(rng.normal(size=cols), "f32") if form != "no sum" else None
    dw = None if w is None else torch.from_numpy(w).float().cuda()
    dx, dr = on_gpu(x, kind, cols + pad, offset), on_gpu(r, kind, cols + pad, offset)
    y, around = out_like(rows, cols, kind, cols + pad, offset)
    total, around_total = out_like(rows, cols, kind, cols + pad, offset)
    if form == "in place":
        total = dr
    how = {} if form == "plain" else dict(d_residual=dr.data_ptr(), ld_residual=cols + pad)
    if form != "no sum":
        how.update(d_sum=total.data_ptr(), ld_sum=cols + pad)
    T.rms_norm(dx.data_ptr(), y.data_ptr(), TYPES[kind][0], rows, cols, d_weight=0 if dw is None else dw.data_ptr(), eps=1e-5, ldx=cols + pad, ldy=cols + pad, **how)
    s, far_s, want, far = P.rms_norm(x, None if form == "plain" else r, w, 1e-5, kind)
    within(numbers(y), want, far)
    untouched(around, y)
    if form != "no sum":
        within(numbers(total), s, far_s)
        if form != "in place":
            untouched(around_total, total)


def test_norm_of_zeros_and_of_what_is_no_number():
    x = torch.ones(4, 100, device="cuda")
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    y = torch.full_like(x, 77.0)
    T.rms_norm(x.data_ptr(), y.data_ptr(), T.F32, 4, 100, eps=1e-6)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2, 5].isnan() and (y[2, :5] == 0).all()
    within(numbers(y[3]), np.full(100, 1 / np.sqrt(1 + 1e-6)), 2.0 ** -21)


# ---- rotary positions ----


def turned(x, heads, kind, positions, pad=0, offset=0, backward=False, in_place=False, **rotary):
    tokens, width = x.shape[0], x.shape[1]
    dx = on_gpu(x, kind, width + pad, offset)
    y, around = (dx, None) if in_place else out_like(tokens, width, kind, width + pad, offset)
    p = torch.from_numpy(positions.astype(np.int32)).cuda()
    T.Rotary(width // heads, **rotary).rotate(dx.data_ptr(), y.data_ptr(), TYPES[kind][0], tokens, heads, p.data_ptr(), backward=backward,
                                              ldx=width + pad, ldy=width + pad)
    got = numbers(y)
    if around is not None:
        untouched(around, y)
    return got


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pairing", [T.PAIR_HALVES, T.PAIR_NEIGHBOURS])
@pytest.mark.parametrize("tokens,heads,head,dims,sections,pad,offset,far", [
    (1, 1, 2, 2, [1], 0, 0, 10), (3, 5, 64, 64, [32], 0, 0, 4096), (7, 3, 80, 72, [16, 10, 10], 8, 0, 1000), (2, 4, 128, 120, [60], 0, 0, 1 << 20),
    (5, 2, 96, 48, [8, 8, 8], 3, 1, 100), (1, 64, 128, 128, [64], 0, 0, 2 ** 31 - 1), (4, 2, 256, 256, [40, 0, 44, 44], 0, 8, 65536), (2500, 3, 64, 32, [16], 0, 0, 10 ** 6),
    (2, 3, 1024, 1024, [512], 0, 0, 500), (3, 2, 6, 6, [1, 1, 1], 1, 1, 7)])
def test_rotary(kind, pairing, tokens, heads, head, dims, sections, pad, offset, far):
    rng = np.random.default_rng(tokens + head)
    x = rounded_to(rng.normal(size=(tokens, heads * head)), kind)
    positions = rng.integers(0, far, (len(sections), tokens))
    positions[:, 0] = 0
    positions[0, -1] = far - 1
    for rate in (T.RATE_HEAD, T.RATE_AXIS):
        how = dict(dims=dims, sections=sections, base=10000.0 if rate == T.RATE_HEAD else 500000.0)
        for backward in (False, True):
            want, off = P.rotate(x.reshape(tokens, heads, head), positions, kind=kind, neighbours=pairing == T.PAIR_NEIGHBOURS, by_axis=rate == T.RATE_AXIS,
                                 backward=backward, **how)
            got = turned(x, heads, kind, positions, pad, offset, backward, pairing=pairing, rate=rate, **how)
            within(got.reshape(tokens, heads, head), want, off)
        assert np.array_equal(got, turned(x, heads, kind, positions, pad, offset, True, True, pairing=pairing, rate=rate, **how))


def test_rotary_gradient_by_differences():
    """With L(x) = sum(dy * rotate(x)), (L(x + h d) - L(x - h d)) / 2h is sum(backward(dy) * d): exactly, as L is linear, but for roundings.  Sums of
    products are taken in 64 bits, and the bound of an element is that of test_rotary, with 2 h d for the element's size."""
    rng = np.random.default_rng(9)
    tokens, heads, head, h = 5, 3, 64, 0.5
    how = dict(dims=48, sections=[10, 14], base=100.0)
    positions = rng.integers(0, 50, (2, tokens))
    x, d, dy = (rounded_to(rng.normal(size=(tokens, heads * head)), "f32") for _ in range(3))
    up, down = rounded_to(x + h * d, "f32"), rounded_to(x - h * d, "f32")
    lhs = (dy * (turned(up, heads, "f32", positions, **how) - turned(down, heads, "f32", positions, **how))).sum()
    rhs = (turned(dy, heads, "f32", positions, backward=True, **how) * (up - down)).sum()
    shape = (tokens, heads, head)
    far = sum((np.abs(dy).reshape(shape) * P.rotate(v.reshape(shape), positions, kind="f32", **how)[1]).sum() for v in (up, down))
    far += (P.rotate(dy.reshape(shape), positions, kind="f32", backward=True, **how)[1] * np.abs(up - down).reshape(shape)).sum()
    assert abs(lhs - rhs) <= far


# ---- cache ----


class Cache:
    """A pool whose memory is all ones at first: every scale is a NaN's."""

    def __init__(self, pages, kv_heads, head, page):
        self.memory = torch.full((pages * T.cache_page_bytes(kv_heads, head, page),), 255, dtype=torch.uint8, device="cuda")
        self.handle = T.MX4Cache(self.memory.data_ptr(), pages, kv_heads, head, page=page)
        self.pages, self.kv_heads, self.head, self.page = pages, kv_heads, head, page

    def append(self, k, v, kind, slots, pad=0, offset=0):
        """k, v: [tokens, kv heads * head] in 64 bits."""
        s = torch.tensor(slots, dtype=torch.int64, device="cuda")
        dk, dv = (on_gpu(x, kind, x.shape[1] + pad, offset) for x in (k, v))
        self.handle.append(dk.data_ptr(), dv.data_ptr(), TYPES[kind][0], len(slots), s.data_ptr(), ldk=k.shape[1] + pad, ldv=v.shape[1] + pad)
        torch.cuda.synchronize()

    def read(self, kind, slots, pad=0, offset=0):
        s = torch.tensor(slots, dtype=torch.int64, device="cuda")
        width = self.kv_heads * self.head
        (k, around_k), (v, around_v) = (out_like(len(slots), width, kind, width + pad, offset) for _ in range(2))
        self.handle.read(s.data_ptr(), k.data_ptr(), v.data_ptr(), TYPES[kind][0], len(slots), ldk=width + pad, ldv=width + pad)
        got = numbers(k), numbers(v)
        untouched(around_k, k)
        untouched(around_v, v)
        return got


def of_mx4(x):
    """The values that rows become in the cache (widths are multiples of 32)."""
    return X.values(*X.quantise(x), x.shape[1])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("kv_heads,page,tokens,pad,offset", [(1, 16, 1, 0, 0), (3, 32, 50, 0, 0), (2, 48, 77, 8, 8), (5, 64, 40, 1, 3)])
def test_append_and_read(kind, head, kv_heads, page, tokens, pad, offset):
    rng = np.random.default_rng(head + tokens)
    c = Cache(5, kv_heads, head, page)
    slots = rng.permutation(5 * page)[:tokens]
    k, v = (rounded_to(rng.normal(size=(tokens, kv_heads * head)) * np.exp2(rng.integers(-4, 5, (tokens, kv_heads * head))), kind) for _ in range(2))
    before = c.memory.clone()
    c.append(k, v, kind, slots, pad, offset)
    # a token's bytes, and no others (a code or scale of all ones may be one that was written)
    assert (c.memory != before).sum() <= tokens * 2 * kv_heads * 17 * head // 32
    for back in TYPES:
        got = c.read(back, slots, pad, offset)
        assert np.array_equal(got[0], rounded_to(of_mx4(k), back)) and np.array_equal(got[1], rounded_to(of_mx4(v), back))
    others = np.setdiff1d(np.arange(5 * page), slots)
    assert all(np.isnan(x).all() for x in c.read("f32", others))
    # written again in part: the others keep their values
    again = rounded_to(rng.normal(size=(1, kv_heads * head)), kind)
    c.append(again, -again, kind, slots[:1])
    got = c.read("f32", slots)
    assert np.array_equal(got[0][:1], of_mx4(again)) and np.array_equal(got[1][:1], of_mx4(-again))
    assert np.array_equal(got[0][1:], of_mx4(k)[1:]) and np.array_equal(got[1][1:], of_mx4(v)[1:])


def test_slots_outside_of_the_cache_are_passed_over():
    rng = np.random.default_rng(3)
    c = Cache(2, 2, 64, 16)
    x = rounded_to(rng.normal(size=(5, 128)), "f32")
    before = c.memory.clone()
    c.append(x, x, "f32", [-1, 32, 2 ** 31, -2 ** 40, 2 ** 32])
    assert torch.equal(before, c.memory)
    c.append(x, x, "f32", [-1, 4, 32, 31, 2 ** 32 + 4])
    k, v = c.read("f32", [4, 31, -1, 32, 2 ** 32 + 4])
    assert np.array_equal(k[:2], of_mx4(x)[[1, 3]]) and np.array_equal(v, k) and (k[2:] == 0).all()


def test_infinities_and_nan_make_their_block_nan():
    c = Cache(1, 1, 64, 16)
    k, v = np.ones((2, 64)), np.ones((2, 64))
    k[0, 3], v[1, 40] = np.inf, np.nan
    c.append(k, v, "f32", [0, 1])
    gk, gv = c.read("f32", [0, 1])
    assert np.isnan(gk[0, :32]).all() and (gk[0, 32:] == 1).all() and (gk[1] == 1).all()
    assert (gv[0] == 1).all() and (gv[1, :32] == 1).all() and np.isnan(gv[1, 32:]).all()


# ---- attention ----


class Case:
    """Sequences in a cache: their values in 64 bits, tables, queries, and what attention makes of them."""

    def __init__(self, kind, lengths, fresh, heads, kv_heads, head, page, seed=0, strength=1.0, spare=1, dense=None):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.lengths, self.fresh, self.heads, self.kv_heads, self.head, self.page = kind, lengths, fresh, heads, kv_heads, head, page
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.most = max(max(lengths), 1)
        self.table = np.full((len(lengths), -(-self.most // page) + 1), -1, np.int32)
        self.cache = Cache(self.pages, kv_heads, head, page)
        self.k, self.v, used = [], [], 0
        for s, n in enumerate(lengths):
            self.table[s, :need[s]] = order[used:used + need[s]]
            used += need[s]
            k, v = (rounded_to(rng.normal(size=(n, kv_heads * head)) * w, kind) for w in (strength, 1.0))
            if n:
                self.put(s, range(n), k, v)
            self.k.append(of_mx4(k).reshape(n, kv_heads, head) if n else np.zeros((0, kv_heads, head)))
            self.v.append(of_mx4(v).reshape(n, kv_heads, head) if n else np.zeros((0, kv_heads, head)))
        self.first = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        self.q = rounded_to(rng.normal(size=(max(self.first[-1], 1), heads * head)), kind)

    def put(self, s, places, k, v):
        """Keys and values of sequence s into the cache."""
        self.cache.append(k, v, self.kind, [int(self.table[s, j // self.page]) * self.page + j % self.page for j in places])

    def run(self, window=0, scale=None, pad=0, offset=0, extra=0, first=True, most_rows=None, stream=0, out=None):
        rows = int(self.first[-1]) + extra
        width = self.heads * self.head
        q = on_gpu(np.concatenate([self.q[:self.first[-1]], np.zeros((extra, width))]), self.kind, width + pad, offset)
        y, around = out_like(rows, width, self.kind, width + pad, offset)
        dl, dt, df = (torch.from_numpy(np.ascontiguousarray(v, np.int32)).cuda() for v in (self.lengths, self.table, self.first))
        self.cache.handle.attend(q.data_ptr(), y.data_ptr(), TYPES[self.kind][0], self.heads, len(self.lengths), dl.data_ptr(), dt.data_ptr(), self.most,
                                 d_first=df.data_ptr() if first else 0, rows=rows, most_rows=max(self.fresh) if most_rows is None else most_rows,
                                 ld_table=self.table.shape[1], window=window, scale=scale, ldq=width + pad, ldy=width + pad)
        got = numbers(y)
        untouched(around, y)
        assert (got[self.first[-1]:] == 77.0).all()
        return got[:self.first[-1]]

    def want(self, window=0, scale=None, absent={}):
        y, far = [np.zeros((0, self.heads, self.head))], [np.zeros((0, self.heads, self.head))]
        for s, m in enumerate(self.fresh):
            q = self.q[self.first[s]:self.first[s + 1]].reshape(m, self.heads, self.head)
            one = P.attend(q, self.k[s], self.v[s], self.head ** -0.5 if scale is None else scale, self.kind, window, absent.get(s, ()))
            y.append(one[0])
            far.append(one[1])
        return np.concatenate(y).reshape(-1, self.heads * self.head), np.concatenate(far).reshape(-1, self.heads * self.head)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head", [32, 64, 96, 128, 160, 192, 224, 256])
def test_one_token_of_each_sequence(kind, head):
    c = Case(kind, [1, 16, 17, 0, 31, 33, 150, 1], [1] * 8, 6, 2, head, 16, seed=head)
    got = c.run(first=False)
    within(got, *c.want())
    assert (got[3] == 0).all()
    assert np.array_equal(got, c.run(pad=3, offset=1))  # rows that lie badly


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv_heads,page", [(1, 1, 16), (8, 8, 48), (5, 1, 64), (32, 2, 32), (33, 1, 16), (40, 2, 128), (6, 3, 4096)])
def test_head_groups_and_pages(kind, heads, kv_heads, page):
    c = Case(kind, [70, 5, 200], [1, 1, 1], heads, kv_heads, 64, page, seed=heads)
    within(c.run(), *c.want())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,fresh", [([40, 7, 90], [5, 3, 2]), ([3, 64], [3, 64]), ([130, 0, 12], [130, 2, 20]), ([9, 33], [0, 33]), ([300], [7]), ([257, 100], [200, 100])])
@pytest.mark.parametrize("window", [0, 1, 20, 64, 1000])
def test_several_rows_of_each_sequence(kind, lengths, fresh, window):
    c = Case(kind, lengths, fresh, 4, 2, 64, 16, seed=sum(lengths))
    got = c.run(window=window, extra=2)
    within(got, *c.want(window=window))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head,lengths,fresh,window", [(128, [3000, 1, 4500], [1, 1, 1], 0), (128, [2500, 1030], [4, 9], 0), (64, [6000], [3], 1500), (256, [2200], [2], 0),
                                                       (96, [2100, 64], [1, 1], 0), (128, [5000], [1], 700)])
def test_long_sequences_in_many_chunks(kind, head, lengths, fresh, window):
    c = Case(kind, lengths, fresh, 4, 1, head, 64, seed=head)
    within(c.run(window=window), *c.want(window=window))


@pytest.mark.parametrize("kind", TYPES)
def test_rows_behind_most_rows_are_left_as_they_are(kind):
    c = Case(kind, [50, 20], [6, 3], 2, 1, 64, 16)
    want, far = c.want()
    got = c.run(most_rows=4)
    done = [0, 1, 2, 3, 6, 7, 8]
    within(got[done], want[done], far[done])
    assert (got[4:6] == 77.0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [0.0, 3.0, -0.5])
def test_scales_and_strong_scores(kind, scale):
    """Scores of hundreds: the maximum is raised again and again, weights underflow, one token takes a row."""
    c = Case(kind, [500, 37], [2, 1], 4, 2, 64, 16, strength=8.0)
    got = c.run(scale=scale)
    assert np.isfinite(got).all()
    within(got, *c.want(scale=scale))


def test_scores_that_rise_all_the_way_and_fall():
    for sign in (1, -1):
        c = Case("f32", [400], [1], 2, 1, 32, 16)
        k = np.zeros((400, 32))
        k[:, 0] = of_mx4(np.repeat(np.arange(400.0)[:, None], 32, 1))[:, 0]
        c.put(0, range(400), k, rounded_to(c.v[0].reshape(400, 32), "f32"))
        c.k[0] = of_mx4(k).reshape(400, 1, 32)
        c.q = np.zeros((1, 64))
        c.q[0, [0, 32]] = sign * 1.0, sign * 0.25
        within(c.run(scale=1.0), *c.want(scale=1.0))


@pytest.mark.parametrize("head", [64, 96, 128])
def test_nan_and_infinities_where_they_are_masked(head):
    """A key or value that is no number reaches the rows that see it, in its block of the output, and no others; unwritten slots are all NaN here."""
    c = Case("f32", [60, 40], [30, 1], 4, 2, head, 16, seed=1)
    clean = c.run()
    within(clean, *c.want())
    bad = rounded_to(c.v[0].reshape(60, -1)[40:41], "f32")
    bad[0, head + 33] = np.nan  # token 40, kv head 1, block 1: rows 10 .. of sequence 0 see it
    c.put(0, [40], rounded_to(c.k[0].reshape(60, -1)[40:41], "f32"), bad)
    got = c.run().reshape(31, 4, head)
    ok = clean.reshape(31, 4, head)
    hit = np.zeros(got.shape, bool)
    hit[10:30, 2:, 32:64] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], ok[~hit])
    c.put(0, [40], rounded_to(c.k[0].reshape(60, -1)[40:41], "f32"), rounded_to(c.v[0].reshape(60, -1)[40:41], "f32"))
    bad = rounded_to(c.k[0].reshape(60, -1)[55:56], "f32")
    bad[0, 5] = -np.inf  # kv head 0 of token 55
    c.put(0, [55], bad, rounded_to(c.v[0].reshape(60, -1)[55:56], "f32"))
    got = c.run().reshape(31, 4, head)
    assert np.isnan(got[25:30, :2]).all()
    assert np.array_equal(got[:25], ok[:25]) and np.array_equal(got[25:30, 2:], ok[25:30, 2:]) and np.array_equal(got[30], ok[30])
    c.q[30] = np.inf
    got = c.run().reshape(31, 4, head)
    assert np.isnan(got[30]).all() and np.array_equal(got[:25], ok[:25])


def test_pages_outside_of_the_pool_are_not_seen():
    c = Case("bf16", [100, 40], [3, 1], 4, 2, 64, 16)
    c.table[0, 2], c.table[0, 6], c.table[1, 1] = -1, c.pages, 2 ** 31 - 1
    gone = {0: list(range(32, 48)) + list(range(96, 100)), 1: range(16, 32)}
    within(c.run(), *c.want(absent=gone))
    c.table[:] = -5
    assert (c.run() == 0).all()


def test_offsets_and_lengths_that_make_no_sense_stay_within_bounds():
    c = Case("f32", [40, 30], [2, 2], 2, 1, 64, 16)
    want, far = c.want()
    c.lengths = [-3, 30]
    got = c.run()
    assert (got[:2] == 0).all()
    within(got[2:], want[2:], far[2:])
    c.lengths = [40, 2 ** 31 - 1]  # counts as most_length
    c.table[1, 2:] = -1
    got = c.run()
    within(got[:2], want[:2], far[:2])


def test_the_same_page_twice():
    c = Case("f16", [32, 32], [1, 1], 2, 1, 64, 16)
    c.table[1] = c.table[0]
    c.table[0, 1] = c.table[0, 0]
    k, v = c.k[0], c.v[0]
    c.k = [np.concatenate([k[:16], k[:16]]), k]
    c.v = [np.concatenate([v[:16], v[:16]]), v]
    within(c.run(), *c.want())


def test_no_bits_change_from_run_to_run():
    c = Case("bf16", [3000, 700], [3, 1], 8, 2, 128, 32)
    got = c.run()
    assert all(np.array_equal(got, c.run()) for _ in range(3))


def test_a_sequence_alone_and_in_a_batch():
    """A sequence's outputs depend on what else is in the call only by how it is cut into chunks."""
    c = Case("f32", [700, 90, 3], [1, 1, 1], 4, 2, 128, 32)
    want, far = c.want()
    within(c.run(), want, far)
    for s in range(3):
        one = Case("f32", [700, 90, 3], [1, 1, 1], 4, 2, 128, 32)
        one.lengths, one.fresh, one.table, one.q = [c.lengths[s]], [1], c.table[s:s + 1], c.q[s:s + 1]
        one.first, one.most = np.array([0, 1]), c.lengths[s]
        within(one.run(first=False), want[s:s + 1], far[s:s + 1])


def test_pages_far_into_a_large_pool():
    """Offsets of bytes that pass 32 bits: a page of 16 tokens of 16 heads of 256 is 69632 bytes."""
    pages = 70000
    c = Cache.__new__(Cache)
    c.memory = torch.empty(pages * T.cache_page_bytes(16, 256, 16), dtype=torch.uint8, device="cuda")
    assert c.memory.numel() > 2 ** 32
    c.pages, c.kv_heads, c.head, c.page = pages, 16, 256, 16
    c.handle = T.MX4Cache(c.memory.data_ptr(), pages, 16, 256, page=16)
    case = Case("bf16", [40], [2], 16, 16, 256, 16)
    case.cache, case.table = c, np.array([[69999, 3, 65000, -1]], np.int32)
    case.put(0, range(40), case.k[0].reshape(40, -1), case.v[0].reshape(40, -1))
    within(case.run(), *case.want())


# ---- prompts: rows that share what is made of the values ----


def many(kind, lengths, fresh, heads, kv_heads, head, page, copies, **how):
    """Few sequences in the cache, each `copies` times in the call: enough rows for the kernel of prompts.  The case, its outputs and theirs."""
    c = Case(kind, lengths, fresh, heads, kv_heads, head, page, **how)
    one = c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v
    c.lengths, c.fresh = c.lengths * copies, c.fresh * copies
    c.table, c.q = np.tile(c.table, (copies, 1)), np.tile(c.q[:c.first[-1]], (copies, 1))
    c.first = np.concatenate([[0], np.cumsum(c.fresh)]).astype(np.int32)
    return c, one


def check_many(c, one, copies, **how):
    got = c.run(**how)
    c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v = one
    want, far = c.want(**{k: v for k, v in how.items() if k in ("window", "scale")})
    got = got.reshape(copies, *want.shape)
    within(got[0], want, far)
    assert all(np.array_equal(got[0], g, equal_nan=True) for g in got)
    return got[0]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("head", [32, 64, 96, 128, 160, 192, 224, 256])
def test_prompts(kind, head):
    c, one = many(kind, [130, 64, 97], [130, 64, 40], 4, 2, head, 16, 40, seed=head)
    check_many(c, one, 40)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv_heads,page,window,pad,offset", [(3, 3, 48, 0, 0, 0), (5, 1, 64, 33, 1, 3), (16, 2, 32, 100, 8, 8), (8, 1, 128, 1, 0, 0)])
def test_prompts_groups_pages_and_windows(kind, heads, kv_heads, page, window, pad, offset):
    c, one = many(kind, [150, 0, 65], [90, 3, 65], heads, kv_heads, 64, page, 64, seed=heads)
    check_many(c, one, 64, window=window, pad=pad, offset=offset)


def test_prompts_of_strong_scores():
    c, one = many("bf16", [200], [200], 4, 1, 128, 16, 64, strength=8.0)
    check_many(c, one, 64, scale=2.0)


def test_prompts_with_values_beyond_f16():
    """Values of 2^20, 2^-30 and zero next to ordinary ones: some workgroups multiply in bf16, none loses a bit of them."""
    for big in (2.0 ** 20, 2.0 ** -30, 0.0):
        c, one = many("bf16", [140], [140], 4, 2, 64, 16, 64)
        v = rounded_to(c.rng.normal(size=(140, 128)), "bf16")
        v[70:75, :64] *= big
        c.put(0, range(140), rounded_to(c.k[0].reshape(140, -1), "bf16"), v)
        one[6][0] = of_mx4(v).reshape(140, 2, 64)
        check_many(c, one, 64)


@pytest.mark.parametrize("head", [64, 96, 128])
def test_prompts_with_nan_that_some_rows_see(head):
    c, one = many("bf16", [100], [100], 4, 2, head, 16, 64)
    clean = check_many(c, one, 64).reshape(100, 4, head)
    c, one = many("bf16", [100], [100], 4, 2, head, 16, 64)
    v = rounded_to(c.v[0].reshape(100, -1), "bf16")
    v[40, head + 33] = np.nan  # kv head 1, block 1: rows 40 .. see it
    c.put(0, range(100), rounded_to(c.k[0].reshape(100, -1), "bf16"), v)
    got = c.run().reshape(64, 100, 4, head)
    hit = np.zeros(clean.shape, bool)
    hit[40:, 2:, 32:64] = True
    for g in got[[0, 63]]:
        assert np.isnan(g[hit]).all() and np.array_equal(g[~hit], clean[~hit])


def test_prompts_pages_outside_of_the_pool():
    c, one = many("bf16", [130], [130], 4, 2, 64, 16, 64)
    c.table[:, 3], c.table[:, 7] = -7, c.pages
    got = c.run().reshape(64, 130, -1)
    c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v = one
    want, far = c.want(absent={0: list(range(48, 64)) + list(range(112, 128))})
    within(got[0], want, far)
    within(got[63], want, far)


# ---- streams, graphs, workspaces ----


def test_a_workspace_made_for_some_sequences_serves_fewer():
    c = Case("bf16", [2000, 900, 3], [1, 1, 1], 8, 2, 128, 32)
    stream = torch.cuda.Stream()
    q, (y, _) = on_gpu(c.q, "bf16"), out_like(3, 1024, "bf16")
    length, table = torch.tensor(c.lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(c.table).cuda()
    torch.cuda.synchronize()
    c.cache.handle.prepare(8, 400, 2000, T.BF16, rows=2000, most_rows=5, stream=stream.cuda_stream)
    with torch.cuda.stream(stream):
        for n, most in ((3, 2000), (1, 2000), (2, 2000)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c.cache.handle.attend(q.data_ptr(), y.data_ptr(), T.BF16, 8, n, length.data_ptr(), table.data_ptr(), most, ld_table=table.shape[1],
                                      stream=stream.cuda_stream)
            y.fill_(77.0)
            graph.replay()
            stream.synchronize()
            want, far = c.want()
            within(numbers(y)[:n], want[:n], far[:n])
            assert (y[n:] == 77.0).all()


def test_captured_and_replayed():
    kind, heads, kv, head, page = "bf16", 8, 2, 128, 16
    c = Case(kind, [1500, 40], [1, 1], heads, kv, head, page, spare=8)
    tokens, width = 2, heads * head
    stream = torch.cuda.Stream()
    q = on_gpu(c.q, kind)
    y, _ = out_like(tokens, width, kind)
    length = torch.tensor(c.lengths, dtype=torch.int32, device="cuda")
    table = torch.from_numpy(c.table).cuda()

    def step(s):
        c.cache.handle.attend(q.data_ptr(), y.data_ptr(), T.BF16, heads, 2, length.data_ptr(), table.data_ptr(), 1600, ld_table=table.shape[1], stream=s)

    table = torch.cat([table, torch.full((2, 100), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with pytest.raises(T.TetrisError) as e:  # it would allocate
            with torch.cuda.graph(graph, stream=stream):
                step(stream.cuda_stream)
        assert e.value.code == T.EINVAL
        c.cache.handle.prepare(heads, 2, 1600, T.BF16, stream=stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(stream.cuda_stream)
    torch.cuda.synchronize()
    for turn in range(4):  # lengths and queries change between replays; eager work in between
        c.lengths = [1500 - 300 * turn, 40 - turn]
        c.q = rounded_to(c.rng.normal(size=c.q.shape), kind)
        q.copy_(torch.from_numpy(c.q).to(q.dtype))
        length.copy_(torch.tensor(c.lengths, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        got = numbers(y)
        case_k, case_v = c.k, c.v
        c.k, c.v = [k[:n] for k, n in zip(c.k, c.lengths)], [v[:n] for v, n in zip(c.v, c.lengths)]
        within(got, *c.want())
        c.k, c.v = case_k, case_v
        step(0)
        torch.cuda.synchronize()
        assert np.array_equal(got, numbers(y))


def test_two_streams_have_workspaces_of_their_own():
    cases = [Case("bf16", [4000], [1], 8, 2, 128, 32, seed=s) for s in range(2)]
    one = cases[0]
    width = 8 * 128
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [on_gpu(c.q, "bf16") for c in cases]
    ys = [out_like(1, width, "bf16")[0] for _ in cases]
    length, table = torch.tensor([4000], dtype=torch.int32, device="cuda"), torch.from_numpy(one.table).cuda()
    torch.cuda.synchronize()
    for _ in range(20):
        for q, y, s in zip(qs, ys, streams):
            one.cache.handle.attend(q.data_ptr(), y.data_ptr(), T.BF16, 8, 1, length.data_ptr(), table.data_ptr(), 4000, ld_table=table.shape[1],
                                    stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c, y in zip(cases, ys):
        one.q = c.q
        within(numbers(y), *one.want())


def test_a_step_of_the_whole_half():
    """Norm, rotary positions, append and attention as a decoding step makes them, on a stream, captured: outputs of every replay."""
    kind, heads, kv, head, page, width = "bf16", 4, 2, 64, 16, 256
    rng = np.random.default_rng(5)
    c = Case(kind, [33, 17], [1, 1], heads, kv, head, page, spare=0)
    c.table = np.concatenate([c.table, np.full((2, 2), -1, np.int32)], 1)
    x, r = (rounded_to(rng.normal(size=(2, width)), kind) for _ in range(2))
    dx, dr = on_gpu(x, kind), on_gpu(r, kind)
    h, q, y, total = (out_like(2, width, kind)[0] for _ in range(4))
    k = out_like(2, kv * head, kind)[0]
    place = torch.tensor([32, 16], dtype=torch.int32, device="cuda")
    slot = torch.tensor([int(c.table[0, 2]) * page, int(c.table[1, 1]) * page], dtype=torch.int64, device="cuda")
    length, table = torch.tensor(c.lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(c.table).cuda()
    rotary, stream = T.Rotary(head), torch.cuda.Stream()

    def step():
        s = stream.cuda_stream
        T.rms_norm(dx.data_ptr(), h.data_ptr(), T.BF16, 2, width, d_residual=dr.data_ptr(), d_sum=total.data_ptr(), stream=s)
        rotary.rotate(h.data_ptr(), q.data_ptr(), T.BF16, 2, heads, place.data_ptr(), stream=s)
        rotary.rotate(h.data_ptr(), k.data_ptr(), T.BF16, 2, kv, place.data_ptr(), ldx=width, stream=s)
        c.cache.handle.append(k.data_ptr(), h.data_ptr(), T.BF16, 2, slot.data_ptr(), ldv=width, stream=s)
        c.cache.handle.attend(q.data_ptr(), y.data_ptr(), T.BF16, heads, 2, length.data_ptr(), table.data_ptr(), 64, ld_table=table.shape[1], stream=s)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        c.cache.handle.prepare(heads, 2, 64, T.BF16, stream=stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.synchronize()
    for _ in range(3):
        x = rounded_to(rng.normal(size=(2, width)), kind)
        dx.copy_(torch.from_numpy(x).to(dx.dtype))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        s, far_s, want, far = P.rms_norm(x, r, None, 1e-6, kind)
        within(numbers(total), s, far_s)
        within(numbers(h), want, far)
        hh = numbers(h).reshape(2, heads, head)  # each operator from what the one before it gave
        want, far = P.rotate(hh, np.array([[32, 16]]), head, [32], 10000.0, kind)
        within(numbers(q).reshape(2, heads, head), want, far)
        within(numbers(k).reshape(2, kv, head), want[:, :kv], far[:, :kv])
        ck, cv = of_mx4(numbers(k)), of_mx4(hh.reshape(2, -1)[:, :kv * head])
        for i, n in enumerate((32, 16)):
            c.k[i][n], c.v[i][n] = ck[i].reshape(kv, head), cv[i].reshape(kv, head)
        c.q = numbers(q)
        within(numbers(y), *c.want())
        eager = numbers(y)
        step()
        torch.cuda.synchronize()
        assert np.array_equal(eager, numbers(y))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tokens,context", [(1, 1), (5, 70), (33, 129)])
def test_the_block_with_its_attention(tokens, context, graph):
    """python -m tetris_amd.expert_block: each operator from what the one before it gave; a rounding to bf16 bounds each error, 2^-8, and the sums
    and weights in 32 or 11 bits a sixteenth of that."""
    from tetris_amd import expert_block

    args = ["--tokens", str(tokens), "--width", "256", "--hidden", "96", "--experts", "12", "--top", "3", "--classes", "50", "--steps", "3", "--context", str(context)]
    out = expert_block.main(args + (["--graph"] if graph else []))
    assert out["query_error"] <= 2.0 ** -8 and out["sum_error"] <= 2.0 ** -8 and out["attention_error"] <= 17 / 16 * 2.0 ** -8
    assert out["block_error"] <= 3 * 2.0 ** -8 and out["scores_error"] <= 2.0 ** -8


# ---- more rows than a launch has, more rows than the call says ----


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("most_rows", [1, 3])
@pytest.mark.parametrize("length,fresh,window", [(3000, 500, 100), (900, 900, 40), (20, 400, 7)])
def test_most_rows_below_the_rows_of_a_window(kind, most_rows, length, fresh, window):
    """The rows' window begins far before the newest token: what is cut by most_rows has as many parts as the launch is made for."""
    c = Case(kind, [length, 50], [fresh, 1], 4, 2, 64, 16)
    want, far = c.want(window=window)
    got = c.run(window=window, most_rows=most_rows)
    done = list(range(most_rows)) + [fresh]
    within(got[done], want[done], far[done])
    assert (got[most_rows:fresh] == 77.0).all()


def test_most_rows_below_the_rows_of_a_window_in_equal_shares():
    c, one = many("bf16", [300], [40], 4, 2, 64, 16, 1700)
    got = c.run(window=100, most_rows=2).reshape(1700, 40, -1)
    c.lengths, c.fresh, c.table, c.first, c.q, c.k, c.v = one
    want, far = c.want(window=100)
    within(got[0, :2], want[:2], far[:2])
    within(got[-1, :2], want[:2], far[:2])
    assert (got[:, 2:] == 77.0).all() and (got[:, :2] == got[:1, :2]).all()


def test_norm_of_more_rows_than_a_launch_has():
    """2^26 rows of a wave each are 2^32 threads."""
    rows = (1 << 26) + 5
    x = torch.randn(rows, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    y = torch.full_like(x, 77.0)
    T.rms_norm(x.data_ptr(), y.data_ptr(), T.F32, rows, 1, eps=0.5)
    x = x.double()
    # the square and the sum's division half a step each, halved by the root; the root, the reciprocal and the product as much again each
    assert ((y - x / (x * x + 0.5).sqrt()).abs() <= 5 * 2.0 ** -24).all()


def test_rotary_of_more_tokens_than_a_launch_has():
    """2^24 tokens of a workgroup each are 2^32 threads; in place.  A turn by 1 or 2 radians of (1, 0)."""
    tokens, head = (1 << 24) + 3, 1024
    x = torch.zeros(tokens, head, dtype=torch.float16, device="cuda")
    x[:, 0] = 1
    position = torch.ones(tokens, dtype=torch.int32, device="cuda")
    position[-1] = 2
    T.Rotary(head).rotate(x.data_ptr(), x.data_ptr(), T.F16, tokens, 1, position.data_ptr())
    for part in (x[:1 << 22], x[1 << 22:-1]):
        assert (part[:, 0] == float(np.float16(np.cos(1)))).all() and (part[:, head // 2] == float(np.float16(np.sin(1)))).all()
    assert float(x[-1, 0]) == np.float16(np.cos(2)) and float(x[-1, head // 2]) == np.float16(np.sin(2))
    assert not x[-5:, 1:head // 2].any() and not x[-5:, head // 2 + 1:].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,heads", [(1, 4), (3, 4), (200, 16)])
def test_calls_for_no_tokens_at_all(kind, rows, heads):
    """most_length 0, with which there is no table: every row sees nothing."""
    c = Cache(1, 2, 64, 16)
    q = on_gpu(np.ones((2 * rows, heads * 64)), kind, heads * 64)
    y, around = out_like(2 * rows, heads * 64, kind, heads * 64)
    first, length = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, rows, 2 * rows], [0, 9]))
    c.handle.attend(q.data_ptr(), y.data_ptr(), TYPES[kind][0], heads, 2, length.data_ptr(), 0, 0, d_first=first.data_ptr(), rows=2 * rows, most_rows=rows)
    assert (numbers(y) == 0).all()
    untouched(around, y)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,kv_heads", [([40], 1), ([4100, 70], 2)])
def test_calls_made_for_the_longest_sequences(kind, lengths, kv_heads):
    """most_length 2^28, where sequences are short: few quanta of many, by chunks and by equal shares."""
    c = Case(kind, lengths, [1] * len(lengths), 2, kv_heads, 64, 4096)
    want, far = c.want()
    table = np.full((len(lengths), (1 << 28) // 4096), -1, np.int32)
    table[:, : c.table.shape[1]] = c.table
    c.table, c.most = table, 1 << 28
    within(c.run(), want, far)
