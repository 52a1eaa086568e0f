"""Root-mean-square norm over rows with a residual's addition, forward and backward, over the C ABI."""
import ctypes as C

from . import _ffi
from ._ffi import address as _at, check, lib
from .device import _h

_ffi._sig("he_rms_norm_create", C.POINTER(C.c_void_p), C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int, C.c_float)
_ffi._sig("he_rms_norm_destroy", C.c_void_p)
_ffi._sig("he_rms_norm_forward", C.c_void_p, C.c_int64, *[C.c_void_p] * 8)
_ffi._sig("he_rms_norm_backward", C.c_void_p, C.c_int64, *[C.c_void_p] * 9)
_ffi._sig("he_rms_norm_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_rms_norm_describe", C.c_void_p, restype=C.c_char_p)


class RmsNorm:
    """h = x + residual, gamma * h / sqrt(mean(h^2) + epsilon) over rows of `columns` values, whose number each call gives.

    Construction generates and compiles the kernels and needs no GPU. Operands are DeviceBuffers, Tensors or raw device addresses: x, y, dy
    and dx of type `dtype`, the residual, h and their gradients of `residual_dtype` (None: there is no residual, and h is x), gamma of
    `param_dtype`, rstd, scales and gamma's gradient f32. output "i8": y is a quantised matrix (see Int8Matmul) with its scales.
    """

    def __init__(self, columns, dtype, residual_dtype=None, param_dtype="f32", output="same", epsilon=1e-5):
        if output not in ("same", "i8"):
            raise ValueError(f"output {output!r} is neither 'same' nor 'i8'")
        self.columns = int(columns)
        self.handle = C.c_void_p()
        check(lib.he_rms_norm_create(C.byref(self.handle), self.columns, _ffi.DTYPES[dtype], -1 if residual_dtype is None else _ffi.DTYPES[residual_dtype],
                                     _ffi.DTYPES[param_dtype], int(output == "i8"), epsilon))

    @property
    def source(self):
        return lib.he_rms_norm_source(self.handle).decode()

    @property
    def description(self):
        return lib.he_rms_norm_describe(self.handle).decode()

    def forward(self, rows, x, gamma, y, residual=None, new_residual=None, rstd=None, scales=None, stream=None):
        """Writes y, new_residual (h; it may be residual), rstd [rows] where it is asked for, and with output "i8" scales [rows]. y may be x."""
        check(lib.he_rms_norm_forward(self.handle, rows, _at(x), _at(gamma), _at(residual), _at(new_residual), _at(y), _at(rstd), _at(scales), _h(stream)))

    def backward(self, rows, dy, h, gamma, rstd, dx, dgamma, dh=None, dresidual=None, stream=None):
        """Writes the gradient of h, with dh (what reaches h from elsewhere) added, to dx and dresidual (one may be None), and gamma's."""
        check(lib.he_rms_norm_backward(self.handle, rows, _at(dy), _at(h), _at(gamma), _at(rstd), _at(dh), _at(dx), _at(dresidual), _at(dgamma),
                                       _h(stream)))

    def close(self):
        if self.handle:
            lib.he_rms_norm_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
