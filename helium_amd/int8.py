"""Quantised matrices, rows of 8-bit whole numbers with an f32 scale each, and their products, over the C ABI."""
import ctypes as C

from . import _ffi
from ._ffi import address as _at, check, lib
from .device import _h

_ffi._sig("he_quantized_pitch", C.c_int64, restype=C.c_int64)
_ffi._sig("he_quantize_rows_create", C.POINTER(C.c_void_p), C.c_int64, C.c_int)
_ffi._sig("he_quantize_rows_destroy", C.c_void_p)
_ffi._sig("he_quantize_rows", C.c_void_p, C.c_int64, *[C.c_void_p] * 4)
_ffi._sig("he_quantize_rows_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_quantize_rows_describe", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_int8_matmul_create", C.POINTER(C.c_void_p), C.c_int64, C.c_int64, C.c_int)
_ffi._sig("he_int8_matmul_destroy", C.c_void_p)
_ffi._sig("he_int8_matmul", C.c_void_p, C.c_int64, *[C.c_void_p] * 7)
_ffi._sig("he_int8_matmul_source", C.c_void_p, restype=C.c_char_p)
_ffi._sig("he_int8_matmul_describe", C.c_void_p, C.c_int64, C.c_char_p, C.c_size_t)


def pitch(columns):
    """Bytes of a quantised matrix' row: its columns, and zeros up to a multiple of 16."""
    return lib.he_quantized_pitch(columns)


class QuantizeRows:
    """q = round(127 x / A), scale = A / 127 with A a row's largest |x|, for rows of `columns` values of type `dtype`."""

    def __init__(self, columns, dtype):
        self.columns = int(columns)
        self.handle = C.c_void_p()
        check(lib.he_quantize_rows_create(C.byref(self.handle), self.columns, _ffi.DTYPES[dtype]))

    @property
    def source(self):
        return lib.he_quantize_rows_source(self.handle).decode()

    @property
    def description(self):
        return lib.he_quantize_rows_describe(self.handle).decode()

    def quantize(self, rows, x, q, scales, stream=None):
        """x [rows, columns] -> q, rows of pitch(columns) bytes, and scales [rows]."""
        check(lib.he_quantize_rows(self.handle, rows, _at(x), _at(q), _at(scales), _h(stream)))

    def close(self):
        if self.handle:
            lib.he_quantize_rows_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Int8Matmul:
    """y = x weights^T of quantised matrices: tokens of `inputs` values, a row of weights for each of `channels`, results of type `dtype`.

    A quantised matrix has rows of pitch(columns) bytes, whole numbers from -127 to 127 and zeros behind the columns, and an f32 scale for
    each: QuantizeRows makes them of weights and activations, RmsNorm(output="i8") of a normalised residual stream.
    """

    def __init__(self, inputs, channels, dtype):
        self.inputs, self.channels = int(inputs), int(channels)
        self.handle = C.c_void_p()
        check(lib.he_int8_matmul_create(C.byref(self.handle), self.inputs, self.channels, _ffi.DTYPES[dtype]))

    @property
    def source(self):
        return lib.he_int8_matmul_source(self.handle).decode()

    def describe(self, tokens):
        """How a call with so many tokens is cut."""
        text = C.create_string_buffer(256)
        check(lib.he_int8_matmul_describe(self.handle, tokens, text, len(text)))
        return text.value.decode()

    def multiply(self, tokens, x, x_scales, weights, weight_scales, y, bias=None, stream=None):
        """y[t][n] = x_scales[t] weight_scales[n] (x[t] . weights[n]) + bias[n]"""
        check(lib.he_int8_matmul(self.handle, tokens, _at(x), _at(x_scales), _at(weights), _at(weight_scales), _at(bias), _at(y), _h(stream)))

    def close(self):
        if self.handle:
            lib.he_int8_matmul_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
