"""Orthogonalised updates of groups of matrices, and the Muon optimizer step built on them, over the C ABI."""
import ctypes as C

from . import _ffi
from ._ffi import check, lib
from .device import _h
from .group_norm import _at

_LIST = C.POINTER(C.c_void_p)
_ffi._sig("he_muon_create", C.POINTER(C.c_void_p), C.POINTER(C.c_int64), C.c_int, C.c_int, C.c_int, C.c_int)
_ffi._sig("he_muon_destroy", C.c_void_p)
_ffi._sig("he_muon_orthogonalize", C.c_void_p, _LIST, _LIST, C.c_int, C.c_void_p)
_ffi._sig("he_muon_step", C.c_void_p, _LIST, _LIST, _LIST, _LIST, _LIST, C.c_int, C.c_float, C.c_float, C.c_float, C.c_int, C.c_void_p)
_ffi._sig("he_muon_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_muon_describe", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_muon_table", C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.POINTER(C.c_size_t))

PRECISIONS = {"f32_f32": 0, "f16_f32": 3}  # HE_PREC_F32_F32, HE_PREC_F16_F32


def _list(buffers):
    at = [_at(b) for b in buffers]
    return (C.c_void_p * max(len(at), 1))(*[a if isinstance(a, int) else a.value for a in at]), len(at)


class Muon:
    """The optimizer step of a group of matrices, `shapes` as (rows, columns) of each; a convolution's filter [out, kh, kw, in] is
    out x (kh * kw * in).

    Construction generates and compiles the kernels and needs no GPU. Operands are lists of DeviceBuffers, Tensors or raw device addresses,
    one per matrix: gradients (and orthogonalised matrices) of type `dtype`, momenta and weights f32. precision "f32_f32" gives
    the error of f32 products, or some times that where it takes several steps at once (backend.OPT_MUON_SEVERAL_STEPS), "f16_f32" about three digits at a third of the time (f16 matrices, whose results hold more,
    are treated as at "f32_f32").
    """

    def __init__(self, shapes, dtype, precision="f32_f32", steps=5):
        if precision not in PRECISIONS:
            raise ValueError(f"precision {precision!r} is none of {sorted(PRECISIONS)}")
        self.shapes = [(int(r), int(c)) for r, c in shapes]
        self.handle = C.c_void_p()
        check(lib.he_muon_create(C.byref(self.handle), _ffi.arr(C.c_int64, [e for s in self.shapes for e in s]), len(self.shapes),
                                 _ffi.DTYPES[dtype], PRECISIONS[precision], steps))

    @property
    def source(self):
        return lib.he_muon_source(self.handle).decode()

    @property
    def description(self):
        return lib.he_muon_describe(self.handle).decode()

    def table(self, which):
        """The bytes of one of the tables that the kernels read."""
        size = C.c_size_t()
        check(lib.he_muon_table(self.handle, which, None, 0, C.byref(size)))
        data = C.create_string_buffer(max(size.value, 1))
        check(lib.he_muon_table(self.handle, which, data, size.value, C.byref(size)))
        return data.raw[:size.value]

    def orthogonalize(self, matrices, out, stream=None):
        """out[k] becomes the orthogonalised matrices[k]; it may be matrices[k]."""
        (a, n), (b, m) = _list(matrices), _list(out)
        if n != m:
            raise ValueError(f"{n} matrices and {m} results")
        check(lib.he_muon_orthogonalize(self.handle, a, b, n, _h(stream)))

    def step(self, gradients, momenta, weights, new_momenta, new_weights, learning_rate, momentum=0.95, weight_decay=0.0, nesterov=True,
             stream=None):
        """Writes new_momenta and new_weights, which may be momenta and weights."""
        lists = [_list(x) for x in (gradients, momenta, weights, new_momenta, new_weights)]
        if len({n for _, n in lists}) != 1:
            raise ValueError("lists of different lengths: %s" % [n for _, n in lists])
        check(lib.he_muon_step(self.handle, *[a for a, _ in lists], lists[0][1], learning_rate, momentum, weight_decay, int(nesterov), _h(stream)))

    def close(self):
        if self.handle:
            lib.he_muon_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
