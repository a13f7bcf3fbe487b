"""Operators on compressed weights (ctypes over include/tetris_mx4.h): 4-bit floating point with shared scales (MX4),
products with MX4 weights, routing of tokens to experts, the experts' products.  Reached as tetris_amd.MX4Weights,
tetris_amd.Router, tetris_amd.ExpertLayer, tetris_amd.mx4_quantize, tetris_amd.mx4_dequantize.

Like the launchers of tetris_amd these take raw device pointers (a torch tensor's .data_ptr()) and a stream handle,
and return as soon as the work is enqueued.  Leading dimensions default to dense rows.
"""
import ctypes as C

from . import _check, _lib

F32, F16, BF16 = range(3)
SCORE_SOFTMAX, SCORE_SIGMOID = range(2)
GROUP_MAX, GROUP_TWO = range(2)


class _Router(C.Structure):
    _fields_ = [("experts", C.c_int32), ("top", C.c_int32), ("score", C.c_int32), ("groups", C.c_int32), ("top_groups", C.c_int32),
                ("group_by", C.c_int32), ("renorm", C.c_int32), ("scale", C.c_float)]


_p, _i, _l = C.c_void_p, C.c_int, C.c_int64
_lib.tetris_mx4_code_bytes.argtypes = _lib.tetris_mx4_scale_bytes.argtypes = [_i]
_lib.tetris_mx4_code_bytes.restype = _lib.tetris_mx4_scale_bytes.restype = C.c_size_t
_lib.tetris_mx4_quantize.argtypes = [_p, _i, _l, _i, _l, _p, _p, _p]
_lib.tetris_mx4_dequantize.argtypes = [_p, _p, _l, _i, _p, _i, _l, _p]
_lib.tetris_mx4_create.argtypes = [_p, _p, _i, _i, _i, _i, _p, C.POINTER(_p)]
_lib.tetris_mx4_create_values.argtypes = [_p, _i, _i, _i, _i, _l, _i, _p, C.POINTER(_p)]
_lib.tetris_mx4_destroy.argtypes = [_p]
_lib.tetris_mx4_destroy.restype = None
_lib.tetris_mx4_prepare.argtypes = [_p, _i, _i, _i, _p]
_lib.tetris_mx4_linear.argtypes = [_p, _p, _i, _i, _l, _p, _l, _p, _i, _p]
_lib.tetris_route.argtypes = [C.POINTER(_Router), _p, _i, _i, _l, _p, _p, _p, _p]
_lib.tetris_route_backward.argtypes = [C.POINTER(_Router), _p, _i, _i, _l, _p, _p, _p, _l, _p]
_lib.tetris_experts_prepare.argtypes = [_p, _p, _i, _i, _i, _p]
_lib.tetris_experts.argtypes = [_p, _p, _p, _i, _i, _l, _i, _p, _p, _p, _l, _p]


def mx4_code_bytes(cols):
    """Bytes of codes in an MX4 row of `cols` values."""
    return _lib.tetris_mx4_code_bytes(cols)


def mx4_scale_bytes(cols):
    """Bytes of scales in an MX4 row of `cols` values."""
    return _lib.tetris_mx4_scale_bytes(cols)


def mx4_quantize(d_x, dtype, rows, cols, d_codes, d_scales, ld=None, stream=0):
    """rows x cols numbers to MX4 rows (tetris_mx4_quantize)."""
    _check(_lib.tetris_mx4_quantize(d_x, dtype, rows, cols, cols if ld is None else ld, d_codes, d_scales, stream))


def mx4_dequantize(d_codes, d_scales, rows, cols, d_y, dtype, ld=None, stream=0):
    """The values that MX4 rows stand for (tetris_mx4_dequantize)."""
    _check(_lib.tetris_mx4_dequantize(d_codes, d_scales, rows, cols, d_y, dtype, cols if ld is None else ld, stream))


class MX4Weights:
    """`experts` matrices of n x k weights in MX4, laid out for the kernels: from MX4 rows, or with MX4Weights.quantize from
    numbers (tetris_mx4_create, tetris_mx4_create_values).  gated: the first half of a matrix's rows gates the second."""

    def __init__(self, d_codes, d_scales, n, k, experts=1, gated=False, stream=0):
        self._h = _p()
        _check(_lib.tetris_mx4_create(d_codes, d_scales, experts, n, k, int(gated), stream, C.byref(self._h)))
        self.n, self.k, self.experts, self.gated = n, k, experts, gated

    @classmethod
    def quantize(cls, d_w, dtype, n, k, experts=1, gated=False, ld=None, stream=0):
        self = cls.__new__(cls)
        self._h = _p()
        _check(_lib.tetris_mx4_create_values(d_w, dtype, experts, n, k, k if ld is None else ld, int(gated), stream, C.byref(self._h)))
        self.n, self.k, self.experts, self.gated = n, k, experts, gated
        return self

    def prepare(self, m, dtype, mx4_input=False, stream=0):
        """Makes the workspace of linear() for up to m rows on `stream`, ahead of a graph capture (tetris_mx4_prepare)."""
        _check(_lib.tetris_mx4_prepare(self._h, m, dtype, int(mx4_input), stream))

    def linear(self, d_x, d_y, m, dtype, d_bias=0, ldx=None, ldy=None, mx4_input=False, stream=0):
        """y = x W^T + bias for m rows (tetris_mx4_linear)."""
        _check(_lib.tetris_mx4_linear(self._h, d_x, dtype, m, self.k if ldx is None else ldx, d_y, self.n if ldy is None else ldy,
                                      d_bias, int(mx4_input), stream))

    def close(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.tetris_mx4_destroy(self._h)
            self._h = None

    __del__ = close


class Router:
    """How tokens are routed (tetris_router): `top` of `experts` experts each, out of the top_groups best of `groups` groups."""

    def __init__(self, experts, top, score=SCORE_SOFTMAX, groups=1, top_groups=1, group_by=GROUP_MAX, renorm=True, scale=1.0):
        self.experts, self.top = experts, top
        self._r = _Router(experts, top, score, groups, top_groups, group_by, int(renorm), scale)

    def route(self, d_logits, dtype, tokens, d_index, d_weight, d_bias=0, ld=None, stream=0):
        """Each token's experts (int32) and weights (float), tokens x top (tetris_route)."""
        _check(_lib.tetris_route(C.byref(self._r), d_logits, dtype, tokens, self.experts if ld is None else ld, d_bias, d_index, d_weight,
                                 stream))

    def backward(self, d_logits, dtype, tokens, d_index, d_dweight, d_dlogits, ld=None, ld_out=None, stream=0):
        """The weights' gradient carried to the logits (tetris_route_backward)."""
        _check(_lib.tetris_route_backward(C.byref(self._r), d_logits, dtype, tokens, self.experts if ld is None else ld, d_index, d_dweight,
                                          d_dlogits, self.experts if ld_out is None else ld_out, stream))


class ExpertLayer:
    """The experts' products (tetris_experts) with `up` (gated, experts x 2 hidden x width) and `down` (experts x width x hidden)."""

    def __init__(self, up, down):
        self.up, self.down = up, down

    def prepare(self, tokens, top, dtype, stream=0):
        """Makes the workspace of run() for up to so many tokens on `stream` (tetris_experts_prepare)."""
        _check(_lib.tetris_experts_prepare(self.up._h, self.down._h, tokens, top, dtype, stream))

    def run(self, d_x, d_index, d_weight, d_y, tokens, top, dtype, ldx=None, ldy=None, stream=0):
        """y[t] = sum_j weight[t, j] expert_{index[t, j]}(x[t])."""
        _check(_lib.tetris_experts(self.up._h, self.down._h, d_x, dtype, tokens, self.up.k if ldx is None else ldx, top, d_index, d_weight,
                                   d_y, self.down.n if ldy is None else ldy, stream))
