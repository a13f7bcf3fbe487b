"""CPU-side checks of include/tetris_mx4.h: exported symbols, sizes, and arguments refused before anything runs on a GPU;
and tests/mx4_plain.py against hand-worked numbers."""
import ctypes
import os
import re

import numpy as np
import pytest

import mx4_plain as P
from conftest import ROOT

T = pytest.importorskip("tetris_amd")
A = 4096  # stands for an aligned device address: nothing may be read there


def refused(call):
    with pytest.raises(T.TetrisError) as e:
        call()
    assert e.value.code == T.EINVAL and len(str(e.value)) > 20


def test_every_declared_symbol_is_exported():
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "tetris_mx4.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(tetris_[a-z0-9_]+)\s*\(", hdr))
    assert len(names) == 13
    lib = ctypes.CDLL(T.LIB_PATH)
    assert not [n for n in sorted(names) if not hasattr(lib, n)]


def test_row_sizes():
    assert [(T.mx4_code_bytes(c), T.mx4_scale_bytes(c)) for c in (0, 1, 32, 33, 4096)] == [(0, 0), (16, 1), (16, 1), (32, 2), (2048, 128)]


def test_quantise_refusals():
    refused(lambda: T.mx4_quantize(A, 3, 1, 32, A, A))
    refused(lambda: T.mx4_quantize(A, T.F32, -1, 32, A, A))
    refused(lambda: T.mx4_quantize(A, T.F32, 1, 0, A, A))
    refused(lambda: T.mx4_quantize(A, T.F32, 1, 32, A, A, ld=31))
    refused(lambda: T.mx4_quantize(0, T.F32, 1, 32, A, A))
    refused(lambda: T.mx4_quantize(A, T.F32, 1, 32, 0, A))
    refused(lambda: T.mx4_quantize(A, T.F32, 1, 32, A, 0))
    refused(lambda: T.mx4_quantize(A, T.F32, 1, 32, A + 8, A))
    refused(lambda: T.mx4_quantize(A + 1, T.BF16, 1, 32, A, A))
    refused(lambda: T.mx4_dequantize(A, A, 1, 32, A, -1))
    refused(lambda: T.mx4_dequantize(A, A, 1, 32, A, T.F16, ld=8))
    refused(lambda: T.mx4_dequantize(A, 0, 1, 32, A, T.F16))
    refused(lambda: T.mx4_dequantize(A + 4, A, 1, 32, A, T.F16))
    refused(lambda: T.mx4_dequantize(A, A, 1, 32, A + 2, T.F32))
    T.mx4_quantize(0, T.F32, 0, 32, 0, 0)  # nothing to do
    T.mx4_dequantize(0, 0, 0, 32, 0, T.F32)


def test_weight_refusals():
    refused(lambda: T.MX4Weights(0, A, 32, 32))
    refused(lambda: T.MX4Weights(A, 0, 32, 32))
    refused(lambda: T.MX4Weights(A + 1, A, 32, 32))
    refused(lambda: T.MX4Weights(A, A, 0, 32))
    refused(lambda: T.MX4Weights(A, A, 32, -1))
    refused(lambda: T.MX4Weights(A, A, 32, 32, experts=0))
    refused(lambda: T.MX4Weights(A, A, 32, 32, experts=1025))
    refused(lambda: T.MX4Weights(A, A, 33, 32, gated=True))
    refused(lambda: T.MX4Weights.quantize(A, 9, 32, 32))
    refused(lambda: T.MX4Weights.quantize(A, T.F32, 32, 32, ld=31))
    refused(lambda: T.MX4Weights.quantize(0, T.F32, 32, 32))
    none = T.MX4Weights.__new__(T.MX4Weights)
    none._h, none.k, none.n = None, 32, 32
    refused(lambda: none.linear(A, A, 1, T.F32))
    refused(lambda: none.prepare(1, T.F32))


def test_router_refusals():
    def route(tokens=1, logits=A, index=A, weight=A, dtype=T.F32, ld=None, **how):
        r = T.Router(how.pop("experts", 16), how.pop("top", 2), **how)
        return lambda: r.route(logits, dtype, tokens, index, weight, ld=ld)

    for call in (route(experts=0), route(experts=1025), route(top=0), route(top=17), route(experts=64, top=33), route(score=2), route(groups=3),
                 route(groups=0), route(experts=130, groups=65), route(groups=4, top_groups=5), route(groups=4, top_groups=0),
                 route(groups=4, top_groups=1, top=5), route(groups=16, top_groups=4, group_by=T.GROUP_TWO), route(group_by=5), route(tokens=-1),
                 route(logits=0), route(index=0), route(weight=0), route(dtype=5), route(ld=15), route(logits=A + 2)):
        refused(call)
    r = T.Router(16, 2)
    refused(lambda: r.backward(A, T.F32, 1, A, A, 0))
    refused(lambda: r.backward(A, T.F32, 1, A, A, A, ld_out=15))
    refused(lambda: r.backward(A, T.BF16, 1, A, A, A + 1))


def test_plain_quantisation_of_worked_numbers():
    x = np.zeros((1, 32))
    x[0, :12] = [7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.01, -0.26, 6.0, -0.0]
    code, scales = P.quantise(x)
    assert scales[0, 0] == 127  # 2^(2 - 2)
    assert list(P.values(code, scales, 12)[0]) == [6, 0, 1, 1, 2, 2, 4, 4, -6, -0.5, 6, 0]
    assert code[0, 0, 11] == 8
    code, scales = P.quantise(np.full((1, 3), 2.0 ** -130))
    assert scales[0, 0] == 0 and list(P.values(code, scales, 3)[0]) == [0, 0, 0]
    assert P.quantise(np.array([[1.0, np.inf]]))[1][0, 0] == 255
    assert np.array_equal(P.unpacked(P.packed(code)), code.reshape(1, -1))


def test_plain_routing_of_worked_numbers():
    x = np.log(np.array([[1.0, 2.0, 4.0, 1.0]]))
    index, weight = P.route(x, 2, renorm=False)
    assert list(index[0]) == [2, 1] and np.allclose(weight, [[0.5, 0.25]])
    index, weight = P.route(x, 2, bias=np.array([1.0, 0, 0, 1.0]))
    assert list(index[0]) == [0, 3] and np.allclose(weight, 0.5)
    index, _ = P.route(x, 1, groups=2, top_groups=1, bias=np.array([0.6, 0, 0, 0]), two=True)
    assert list(index[0]) == [0]


def test_expert_refusals_without_weights():
    none = T.MX4Weights.__new__(T.MX4Weights)
    none._h, none.k, none.n = None, 32, 32
    refused(lambda: T.ExpertLayer(none, none).run(A, A, A, A, 1, 1, T.F32))
    refused(lambda: T.ExpertLayer(none, none).prepare(1, 1, T.F32))
