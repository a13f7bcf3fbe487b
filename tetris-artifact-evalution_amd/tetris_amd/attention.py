"""The attention half of a served block (ctypes over include/tetris_attention.h): the residual's addition with a
root-mean-square norm, rotary positions, a cache of keys and values in MX4, attention over it.  Reached as
tetris_amd.rms_norm, tetris_amd.Rotary, tetris_amd.MX4Cache, tetris_amd.cache_page_bytes.

Like the launchers of tetris_amd these take raw device pointers (a torch tensor's .data_ptr()) and a stream handle,
and return as soon as the work is enqueued.  Leading dimensions default to dense rows.
"""
import ctypes as C

from . import _check, _lib

PAIR_HALVES, PAIR_NEIGHBOURS = range(2)
RATE_HEAD, RATE_AXIS = range(2)


class _Rotary(C.Structure):
    _fields_ = [("head", C.c_int32), ("dims", C.c_int32), ("axes", C.c_int32), ("sections", C.c_int32 * 4), ("pairing", C.c_int32),
                ("rate", C.c_int32), ("base", C.c_double)]


class _Attention(C.Structure):
    _fields_ = [("heads", C.c_int32), ("sequences", C.c_int32), ("rows", C.c_int32), ("most_rows", C.c_int32), ("most_length", C.c_int32),
                ("window", C.c_int32), ("scale", C.c_float)]


_p, _i, _l, _f = C.c_void_p, C.c_int, C.c_int64, C.c_float
_lib.tetris_rms_norm.argtypes = [_p, _i, _l, _i, _l, _p, _l, _p, _f, _p, _l, _p, _l, _p]
_lib.tetris_rotate.argtypes = [C.POINTER(_Rotary), _p, _i, _i, _i, _l, _p, _l, _i, _p, _l, _p]
_lib.tetris_cache_page_bytes.argtypes = [_i, _i, _i]
_lib.tetris_cache_page_bytes.restype = C.c_size_t
_lib.tetris_cache_create.argtypes = [_i, _i, _i, _l, _p, C.POINTER(_p)]
_lib.tetris_cache_destroy.argtypes = [_p]
_lib.tetris_cache_destroy.restype = None
_lib.tetris_cache_append.argtypes = [_p, _p, _l, _p, _l, _i, _i, _p, _p]
_lib.tetris_cache_read.argtypes = [_p, _p, _i, _p, _l, _p, _l, _i, _p]
_lib.tetris_cache_prepare.argtypes = [_p, C.POINTER(_Attention), _i, _p]
_lib.tetris_cache_attend.argtypes = [_p, C.POINTER(_Attention), _p, _l, _i, _p, _p, _p, _l, _p, _l, _p]


def rms_norm(d_x, d_y, dtype, rows, cols, d_weight=0, eps=1e-6, d_residual=0, d_sum=0, ldx=None, ldy=None, ld_residual=None, ld_sum=None,
             stream=0):
    """s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight, row by row (tetris_rms_norm)."""
    ldx, ldy, ld_residual, ld_sum = (cols if v is None else v for v in (ldx, ldy, ld_residual, ld_sum))
    _check(_lib.tetris_rms_norm(d_x, dtype, rows, cols, ldx, d_residual, ld_residual, d_weight, eps, d_sum, ld_sum, d_y, ldy, stream))


class Rotary:
    """Rotary positions (tetris_rotary): the first `dims` of a head's `head` elements in pairs, the sections' pairs each by their axis."""

    def __init__(self, head, dims=None, base=10000.0, sections=None, pairing=PAIR_HALVES, rate=RATE_HEAD):
        dims = head if dims is None else dims
        sections = [dims // 2] if sections is None else list(sections)
        if not 1 <= len(sections) <= 4:
            raise ValueError("one to four sections, got %d" % len(sections))
        self.head = head
        self._r = _Rotary(head, dims, len(sections), (C.c_int32 * 4)(*sections), pairing, rate, base)

    def rotate(self, d_x, d_y, dtype, tokens, heads, d_position, backward=False, ldx=None, ldy=None, ld_position=None, stream=0):
        """Each token's heads turned by its positions (one row of int32 an axis); backward: the gradient carried through (tetris_rotate)."""
        width = heads * self.head
        _check(_lib.tetris_rotate(C.byref(self._r), d_x, dtype, tokens, heads, width if ldx is None else ldx, d_position,
                                  tokens if ld_position is None else ld_position, int(backward), d_y, width if ldy is None else ldy, stream))


def cache_page_bytes(kv_heads, head, page=64):
    """Bytes of a page of a cache, 0 for sizes that there is none of (tetris_cache_page_bytes)."""
    return _lib.tetris_cache_page_bytes(kv_heads, head, page)


class MX4Cache:
    """Keys and values in MX4 (tetris_cache) in the caller's memory: `pages` pages of `page` tokens, cache_page_bytes bytes each."""

    def __init__(self, d_pages, pages, kv_heads, head, page=64):
        self._h = _p()
        self.pages, self.kv_heads, self.head, self.page = pages, kv_heads, head, page
        _check(_lib.tetris_cache_create(kv_heads, head, page, pages, d_pages, C.byref(self._h)))

    def append(self, d_k, d_v, dtype, tokens, d_slot, ldk=None, ldv=None, stream=0):
        """Keys and values of `tokens` tokens into the slots (int64) page * self.page + place (tetris_cache_append)."""
        width = self.kv_heads * self.head
        _check(_lib.tetris_cache_append(self._h, d_k, width if ldk is None else ldk, d_v, width if ldv is None else ldv, dtype, tokens, d_slot,
                                        stream))

    def read(self, d_slot, d_k, d_v, dtype, tokens, ldk=None, ldv=None, stream=0):
        """The keys and values that slots hold (tetris_cache_read)."""
        width = self.kv_heads * self.head
        _check(_lib.tetris_cache_read(self._h, d_slot, tokens, d_k, width if ldk is None else ldk, d_v, width if ldv is None else ldv, dtype,
                                      stream))

    def prepare(self, heads, sequences, most_length, dtype, rows=None, most_rows=1, window=0, stream=0):
        """Makes the workspace of attend() for calls of these sizes on `stream`, ahead of a graph capture (tetris_cache_prepare)."""
        a = _Attention(heads, sequences, sequences if rows is None else rows, most_rows, most_length, window, 0.0)
        _check(_lib.tetris_cache_prepare(self._h, C.byref(a), dtype, stream))

    def attend(self, d_q, d_y, dtype, heads, sequences, d_length, d_table, most_length, d_first=0, rows=None, most_rows=1, ld_table=None,
               window=0, scale=None, ldq=None, ldy=None, stream=0):
        """Each sequence's newest rows over its cached tokens (tetris_cache_attend).  rows: of all sequences together, one each by default;
        scale: 1 / sqrt(head) by default."""
        width = heads * self.head
        a = _Attention(heads, sequences, sequences if rows is None else rows, most_rows, most_length, window,
                       self.head ** -0.5 if scale is None else scale)
        _check(_lib.tetris_cache_attend(self._h, C.byref(a), d_q, width if ldq is None else ldq, dtype, d_first, d_length, d_table,
                                        -(-most_length // self.page) if ld_table is None else ld_table, d_y, width if ldy is None else ldy,
                                        stream))

    def close(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.tetris_cache_destroy(self._h)
            self._h = None

    __del__ = close
