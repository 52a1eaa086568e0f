"""Group norm with an activation, forward and backward, over the C ABI."""
import ctypes as C

from . import _ffi
from ._ffi import check, lib
from .device import _h

_ffi._sig("he_group_norm_create", C.POINTER(C.c_void_p), C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_float)
_ffi._sig("he_group_norm_destroy", C.c_void_p)
_ffi._sig("he_group_norm_forward", *[C.c_void_p] * 8)
_ffi._sig("he_group_norm_backward", *[C.c_void_p] * 11)
_ffi._sig("he_group_norm_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_group_norm_describe", C.c_void_p, restype=C.c_char_p)

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


def _at(buffer):
    """The address of a DeviceBuffer or Tensor, or a raw one; None stays null."""
    return buffer.ptr if hasattr(buffer, "ptr") else C.c_void_p(buffer)


class GroupNorm:
    """act(gamma * (x - mean) / sqrt(variance + epsilon) + beta) over groups of channels of [batch, pixels, channels] tensors.

    Construction generates and compiles the kernels and needs no GPU. Operands are DeviceBuffers, Tensors or raw device addresses: x, y, dy
    and dx of type `dtype`, gamma and beta of `param_dtype` (f32 unless given), statistics and the parameters' gradients f32.
    """

    def __init__(self, batch, pixels, channels, groups, dtype, param_dtype="f32", activation="none", epsilon=1e-5):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation {activation!r} is none of {sorted(ACTIVATIONS)}")
        self.batch, self.pixels, self.channels, self.groups = int(batch), int(pixels), int(channels), int(groups)
        self.handle = C.c_void_p()
        check(lib.he_group_norm_create(C.byref(self.handle), self.batch, self.pixels, self.channels, self.groups, _ffi.DTYPES[dtype],
                                       _ffi.DTYPES[param_dtype], ACTIVATIONS[activation], epsilon))

    @property
    def source(self):
        return lib.he_group_norm_source(self.handle).decode()

    @property
    def description(self):
        return lib.he_group_norm_describe(self.handle).decode()

    def forward(self, x, gamma, beta, y, mean=None, rstd=None, stream=None):
        """Writes y, and the statistics [batch, groups] where they are asked for. y may be x."""
        check(lib.he_group_norm_forward(self.handle, _at(x), _at(gamma), _at(beta), _at(y), _at(mean), _at(rstd), _h(stream)))

    def backward(self, dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, stream=None):
        """Writes the gradients of x, gamma and beta. dx may be dy or x."""
        check(lib.he_group_norm_backward(self.handle, _at(dy), _at(x), _at(gamma), _at(beta), _at(mean), _at(rstd), _at(dx), _at(dgamma),
                                         _at(dbeta), _h(stream)))

    def close(self):
        if self.handle:
            lib.he_group_norm_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
