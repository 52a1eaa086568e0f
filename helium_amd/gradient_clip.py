"""The norm of all gradients of a model together, and clipping, over the C ABI."""
import ctypes as C

from . import _ffi
from ._ffi import address as _at, addresses as _list, check, lib
from .device import _h

_LIST = C.POINTER(C.c_void_p)
_ffi._sig("he_gradient_clip_create", C.POINTER(C.c_void_p), C.POINTER(C.c_int64), C.POINTER(C.c_int), C.c_int)
_ffi._sig("he_gradient_clip_destroy", C.c_void_p)
_ffi._sig("he_gradient_norm", C.c_void_p, _LIST, C.c_int, C.c_void_p, C.c_void_p)
_ffi._sig("he_gradient_clip", C.c_void_p, _LIST, _LIST, C.c_int, C.c_float, C.c_void_p, C.c_void_p)
_ffi._sig("he_gradient_clip_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_gradient_clip_describe", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_gradient_clip_table", C.c_void_p, C.c_void_p, C.c_size_t, C.POINTER(C.c_size_t))


class GradientClip:
    """Clips the gradients of a model by their norm together: tensors of `sizes` values, all of one type or of a type each (`dtypes`).

    Construction generates and compiles the kernels and needs no GPU. Operands are lists of DeviceBuffers, Tensors or raw device addresses, one
    per tensor; the norm is one f32 value on the device.
    """

    def __init__(self, sizes, dtypes):
        self.sizes = [int(n) for n in sizes]
        each = [dtypes] * len(self.sizes) if isinstance(dtypes, str) else list(dtypes)
        if len(each) != len(self.sizes):
            raise ValueError(f"{len(self.sizes)} sizes and {len(each)} types")
        self.handle = C.c_void_p()
        check(lib.he_gradient_clip_create(C.byref(self.handle), _ffi.arr(C.c_int64, self.sizes), _ffi.arr(C.c_int, [_ffi.DTYPES[d] for d in each]), len(each)))

    @property
    def source(self):
        return lib.he_gradient_clip_source(self.handle).decode()

    @property
    def description(self):
        return lib.he_gradient_clip_describe(self.handle).decode()

    def table(self):
        """The bytes of the table that the kernels read."""
        size = C.c_size_t()
        check(lib.he_gradient_clip_table(self.handle, None, 0, C.byref(size)))
        data = C.create_string_buffer(max(size.value, 1))
        check(lib.he_gradient_clip_table(self.handle, data, size.value, C.byref(size)))
        return data.raw[:size.value]

    def norm(self, gradients, norm, stream=None):
        """Writes the norm of all gradients."""
        a, n = _list(gradients)
        check(lib.he_gradient_norm(self.handle, a, n, _at(norm), _h(stream)))

    def clip(self, gradients, out, most, norm=None, stream=None):
        """out[k] = gradients[k] * min(1, most / (norm + 1e-6)); it may be gradients[k], but results share no memory. norm receives the norm before clipping."""
        (a, n), (b, m) = _list(gradients), _list(out)
        if n != m:
            raise ValueError(f"{n} gradients and {m} results")
        check(lib.he_gradient_clip(self.handle, a, b, n, most, _at(norm), _h(stream)))

    def close(self):
        if self.handle:
            lib.he_gradient_clip_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
