"""CPU-side checks of include/tetris_attention.h: exported symbols, sizes, and arguments refused before anything runs on a GPU; and
tests/attention_plain.py against hand-worked numbers."""
import ctypes
import os
import re

import numpy as np
import pytest

import attention_plain as P
from conftest import ROOT
from test_mx4_abi import refused

T = pytest.importorskip("tetris_amd")
A, B = 4096, 8192  # stand for aligned device addresses: nothing may be read there


def test_every_declared_symbol_is_exported():
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "tetris_attention.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(tetris_[a-z0-9_]+)\s*\(", hdr))
    assert len(names) == 9
    lib = ctypes.CDLL(T.LIB_PATH)
    assert not [n for n in sorted(names) if not hasattr(lib, n)]


def test_norm_refusals():
    def norm(x=A, y=B, dtype=T.F32, rows=1, cols=32, **how):
        return lambda: T.rms_norm(x, y, dtype, rows, cols, **how)

    for call in (norm(dtype=3), norm(rows=-1), norm(cols=0), norm(cols=(1 << 20) + 1), norm(x=0), norm(y=0), norm(eps=-1.0), norm(eps=float("nan")),
                 norm(ldx=31), norm(ldy=31), norm(d_residual=B * 2, ld_residual=31), norm(d_sum=B * 2, ld_sum=31), norm(x=A + 2), norm(y=B + 1, dtype=T.BF16),
                 norm(d_weight=B + 2), norm(d_residual=B * 2 + 2), norm(d_sum=B * 2 + 1), norm(x=B), norm(d_residual=B), norm(d_sum=B), norm(d_sum=A),
                 norm(d_residual=3 * A, d_sum=3 * A, ld_sum=40)):
        refused(call)
    T.rms_norm(0, 0, T.F32, 0, 32)  # nothing to do


def test_rotary_refusals():
    def rotate(x=A, y=B, dtype=T.F32, tokens=1, heads=2, positions=A, how={}, **rotary):
        r = T.Rotary(rotary.pop("head", 64), **rotary)
        return lambda: r.rotate(x, y, dtype, tokens, heads, positions, **how)

    for call in (rotate(head=0), rotate(head=1026), rotate(dims=0), rotate(dims=63), rotate(dims=66), rotate(sections=[31]), rotate(sections=[16, 17]),
                 rotate(sections=[33, -1]), rotate(pairing=2), rotate(rate=2), rotate(base=0.0), rotate(base=-1.0), rotate(base=float("inf")),
                 rotate(base=float("nan")), rotate(dtype=7), rotate(tokens=-1), rotate(heads=-1), rotate(x=0), rotate(y=0), rotate(positions=0),
                 rotate(x=A + 2), rotate(y=B + 1, dtype=T.F16), rotate(positions=A + 2), rotate(how=dict(ldx=127)), rotate(how=dict(ldy=127)),
                 rotate(x=A, y=A, how=dict(ldx=200, ldy=201)), rotate(tokens=5, sections=[16, 16], how=dict(ld_position=4))):
        refused(call)
    with pytest.raises(ValueError):
        T.Rotary(64, sections=[8, 8, 8, 4, 4])
    T.Rotary(64).rotate(0, 0, T.F32, 0, 2, 0)
    T.Rotary(64).rotate(0, 0, T.F32, 3, 0, 0)


def test_page_sizes():
    assert T.cache_page_bytes(8, 128, 64) == 8 * 64 * 2 * 68  # 64 bytes of codes and four scales, a key and a value
    assert T.cache_page_bytes(1, 32, 16) == 16 * 2 * 17
    assert [T.cache_page_bytes(*v) for v in ((0, 128, 64), (8, 120, 64), (8, 288, 64), (8, 128, 24), (8, 128, 8192), (1025, 128, 64))] == [0] * 6


def test_cache_refusals():
    for how in (dict(kv_heads=0), dict(kv_heads=1025), dict(head=0), dict(head=100), dict(head=288), dict(page=0), dict(page=8), dict(page=8192),
                dict(pages=0), dict(pages=-1), dict(pages=1 << 27), dict(d_pages=0), dict(d_pages=A + 8)):
        refused(lambda: T.MX4Cache(**{**dict(d_pages=A, pages=4, kv_heads=2, head=64, page=16), **how}))
    c = T.MX4Cache(A, 4, 2, 64, page=16)
    for move in (lambda k=A, v=B, dtype=T.F32, n=1, slot=A, **how: lambda: c.append(k, v, dtype, n, slot, **how),
                 lambda k=A, v=B, dtype=T.F32, n=1, slot=A, **how: lambda: c.read(slot, k, v, dtype, n, **how)):
        for call in (move(k=0), move(v=0), move(slot=0), move(dtype=-1), move(n=-1), move(ldk=127), move(ldv=127), move(k=A + 2), move(v=A + 1, dtype=T.F16),
                     move(slot=A + 4)):
            refused(call)
        move(k=0, v=0, slot=0, n=0)()
    none = T.MX4Cache.__new__(T.MX4Cache)
    none._h, none.kv_heads, none.head, none.page = None, 2, 64, 16
    refused(lambda: none.append(A, B, T.F32, 1, A))
    refused(lambda: none.read(A, A, B, T.F32, 1))
    refused(lambda: none.attend(A, B, T.F32, 4, 1, A, A, 16))
    refused(lambda: none.prepare(4, 1, 16, T.F32))


def test_attend_refusals():
    c = T.MX4Cache(A, 4, 2, 64, page=16)

    def attend(q=A, y=B, dtype=T.F32, heads=4, sequences=3, length=A, table=A, most_length=40, **how):
        return lambda: c.attend(q, y, dtype, heads, sequences, length, table, most_length, **how)

    for call in (attend(q=0), attend(y=0), attend(length=0), attend(table=0), attend(dtype=3), attend(heads=0), attend(heads=3), attend(heads=1026),
                 attend(sequences=-1), attend(most_length=-1), attend(most_length=(1 << 28) + 1, ld_table=1 << 30), attend(window=-1), attend(rows=-1, d_first=A),
                 attend(rows=5), attend(rows=1 << 29, d_first=A), attend(most_rows=-1), attend(ld_table=2), attend(ldq=255), attend(ldy=255),
                 attend(q=A + 2), attend(y=B + 2), attend(length=A + 1), attend(table=A + 2), attend(d_first=A + 2), attend(q=B)):
        refused(call)
    refused(lambda: c.prepare(3, 1, 40, T.F32))
    refused(lambda: c.prepare(4, 1, 40, 9))
    attend(sequences=0)()
    attend(rows=0, d_first=A)()


def test_scales_that_are_not_finite_are_refused():
    c = T.MX4Cache(A, 4, 2, 64, page=16)
    for scale in (float("nan"), float("inf"), -float("inf"), 3e38):
        refused(lambda: c.attend(A, B, T.F32, 4, 3, A, A, 40, scale=scale))


def test_plain_forms_of_worked_numbers():
    s, _, y, _ = P.rms_norm(np.array([[3.0, 3.0]]), np.array([[0.0, 1.0]]), np.array([1.0, 2.0]), 0.0, "f32")
    assert list(s[0]) == [3, 4] and np.allclose(y, [[3 / 12.5 ** 0.5, 8 / 12.5 ** 0.5]])
    x = np.array([[[1.0, 2.0, 5.0, 6.0, 9.0]]])
    y, _ = P.rotate(x, np.array([[1], [2]]), 4, [1, 1], 100.0, "f32")  # angles 1 and 2 / 10
    assert np.allclose(y[0, 0], [np.cos(1) - 5 * np.sin(1), 2 * np.cos(.2) - 6 * np.sin(.2), np.sin(1) + 5 * np.cos(1), 2 * np.sin(.2) + 6 * np.cos(.2), 9])
    y, _ = P.rotate(x, np.array([[1], [2]]), 4, [1, 1], 100.0, "f32", neighbours=True, by_axis=True)  # 1 and 2
    assert np.allclose(y[0, 0, :2], [np.cos(1) - 2 * np.sin(1), np.sin(1) + 2 * np.cos(1)])
    back, _ = P.rotate(y, np.array([[1], [2]]), 4, [1, 1], 100.0, "f32", neighbours=True, by_axis=True, backward=True)
    assert np.allclose(back, x)
    k, v = np.array([[[0.0]], [[np.log(3.0)]], [[7.0]]]), np.array([[[4.0]], [[8.0]], [[1.0]]])
    y, far = P.attend(np.array([[[1.0]], [[0.0]]]), k, v, 1.0, "f32")
    assert np.allclose(y[:, 0, 0], [7.0, 13 / 3]) and (far < 1e-3).all()
    assert np.allclose(P.attend(np.array([[[0.0]]]), k, v, 1.0, "f32", window=2)[0], 4.5)
    assert np.allclose(P.attend(np.zeros((5, 1, 1)), k, v, 1.0, "f32", absent=[0])[0][:, 0, 0], [0, 0, 0, 8, 4.5])
