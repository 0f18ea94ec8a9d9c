"""Microscaled 4-bit floating point (MXFP4 of the OCP Microscaling Formats specification 1.0):
quantisation and products with 4-bit weights (stt_mxfp4_* of include/stt_mi355x.h).

32 consecutive elements of a row share a power-of-two scale, every element is one of 0, 0.5, 1, 1.5, 2,
3, 4, 6 with a sign: 4.25 bits an element.  `WhisperEngine(decoder_format = 'mxfp4')` runs its token
steps on these products; `quantize` / `matmul` work on any matrices.  No counterpart in the reference.

Every call runs on the current stream of the tensors' device and returns without waiting for it.
"""
import ctypes as C
import struct

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GELU = {None: 0, "tanh": 1, "erf": 2}


class MatmulArgs(C.Structure):
    _fields_ = [("d_x", C.c_void_p), ("d_x_scales", C.c_void_p), ("x_row", C.c_int64), ("d_w", C.c_void_p),
                ("d_bias", C.c_void_p), ("d_out", C.c_void_p), ("out_row", C.c_int64), ("out_dtype", C.c_int32),
                ("gelu", C.c_int32), ("accumulate", C.c_int32), ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64)]


# the same layout as bytes, which the host packs faster than it fills the structure
_PACKED = struct.Struct("@2Pq3Pq3i4x3q")
assert _PACKED.size == C.sizeof(MatmulArgs)


def _gpu(t):
    if not t.is_cuda:
        raise ValueError("tensors must be on a GPU, got %s" % t.device)
    return t.device


class Mxfp4Tensor(object):
    """A matrix [rows, k] in MXFP4: `codes` uint8 [rows, k / 2] (element 2 i in the low half of byte i) and
    `scales` uint8 [rows, k / 32] (2 ** (byte - 127), 255: the block is NaN)."""

    def __init__(self, codes, scales):
        for name, t in (("codes", codes), ("scales", scales)):
            if t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous():
                raise ValueError("%s must be a contiguous uint8 matrix, got %s %s" % (name, t.dtype, list(t.shape)))
        if codes.shape[0] != scales.shape[0] or codes.shape[1] != 16 * scales.shape[1]:
            raise ValueError("codes %s and scales %s do not describe blocks of 32" % (list(codes.shape), list(scales.shape)))
        if codes.device != scales.device:
            raise ValueError("tensors on %s and %s" % (codes.device, scales.device))
        if codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], 2 * self.codes.shape[1]))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """The values the codes stand for, float32 or bfloat16 (both hold them exactly)."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("float32 or bfloat16, got %s" % dtype)
        dev = _gpu(self.codes)
        rows, k = self.shape
        lib = _library()
        with _lib.on(dev):
            out = torch.empty((rows, k), dtype=dtype, device=dev)
            _lib.check(lib.stt_mxfp4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), rows, k, out.data_ptr(),
                                                _TYPES[dtype], _lib.stream(dev)))
        return out


def quantize(x):
    """x [rows, k] (float32, bfloat16 or float16, k a multiple of 32, rows contiguous) as an Mxfp4Tensor.
    The scale of a block is 2 ** (floor(log2(max |x|)) - 2), at least 2 ** -127; elements round to the
    nearest code, ties to the even one, and saturate at 6 times the scale.  A block that holds a NaN or
    an infinity becomes NaN."""
    if x.dtype not in _TYPES or x.dim() != 2:
        raise ValueError("x must be a float32, bfloat16 or float16 matrix, got %s %s" % (x.dtype, list(x.shape)))
    rows, k = x.shape
    if k % 32:
        raise ValueError("rows of %d elements: a multiple of 32 is needed" % k)
    if x.numel() and (x.stride(1) != 1 or x.data_ptr() % 16 or (rows > 1 and (x.stride(0) < k or x.stride(0) * x.element_size() % 16))):
        raise ValueError("rows must be contiguous, 16-byte aligned and must not overlap (strides %s)" % (x.stride(),))
    dev = _gpu(x)
    lib = _library()
    with _lib.on(dev):
        codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((rows, k // 32), dtype=torch.uint8, device=dev)
        _lib.check(lib.stt_mxfp4_quantize(x.data_ptr(), _TYPES[x.dtype], rows, k, x.stride(0), codes.data_ptr(),
                                          scales.data_ptr(), _lib.stream(dev)))
    made = Mxfp4Tensor.__new__(Mxfp4Tensor)     # what its constructor checks holds already
    made.codes, made.scales = codes, scales
    return made


class Mxfp4Weight(object):
    """A weight matrix [n, k] (output features first) laid out once for `matmul`: from an Mxfp4Tensor or
    from a float matrix, which is quantised."""

    def __init__(self, w):
        if not isinstance(w, Mxfp4Tensor):
            w = quantize(w)
        self.shape = w.shape
        n, k = w.shape
        if n < 1 or k < 1:
            raise ValueError("empty weight matrix %s" % (list(w.shape),))
        dev = _gpu(w.codes)
        lib = _library()
        with _lib.on(dev):
            self.packed = torch.empty(lib.stt_mxfp4_packed_bytes(n, k), dtype=torch.uint8, device=dev)
            _lib.check(lib.stt_mxfp4_pack(w.codes.data_ptr(), w.scales.data_ptr(), n, k, self.packed.data_ptr(),
                                          _lib.stream(dev)))

    @property
    def device(self):
        return self.packed.device


def matmul(x, weight, bias=None, gelu=None, out_dtype=None, out=None, accumulate=False):
    """act(x @ weight.T + bias) -> [m, n].

    x: bfloat16 [m, k] (rows contiguous; products with the exact weight values) or an Mxfp4Tensor (4-bit
    activations); weight: Mxfp4Weight; bias float32 [n]; gelu: None, 'tanh' or 'erf'.  Sums are float32,
    rounded once to `out_dtype` (bfloat16, the default, or float32).  `out`: a matrix [m, n] to write to
    (not overlapping the inputs), with `accumulate` (float32, no gelu) one to add to."""
    if not isinstance(weight, Mxfp4Weight):
        raise ValueError("weight must be an Mxfp4Weight, got %s" % type(weight).__name__)
    if gelu not in _GELU:
        raise ValueError("gelu must be None, 'tanh' or 'erf', got %r" % (gelu,))
    n, k = weight.shape
    four = isinstance(x, Mxfp4Tensor)
    if not four and (x.dtype != torch.bfloat16 or x.dim() != 2):
        raise ValueError("x must be a bfloat16 matrix or an Mxfp4Tensor, got %s %s" % (x.dtype, list(x.shape)))
    m = x.shape[0]
    if x.shape[1] != k:
        raise ValueError("x has %d columns, the weight %d" % (x.shape[1], k))
    if not four and x.numel() and (x.stride(1) != 1 or x.data_ptr() % 16 or (m > 1 and (x.stride(0) < k or x.stride(0) % 8))):
        raise ValueError("rows of x must be contiguous, 16-byte aligned and must not overlap (strides %s)" % (x.stride(),))
    if out is not None and out_dtype is None:
        out_dtype = out.dtype
    out_dtype = out_dtype or torch.bfloat16
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("output float32 or bfloat16, got %s" % out_dtype)
    if out is not None and (out.dtype != out_dtype or tuple(out.shape) != (m, n) or (
            out.numel() and (out.stride(1) != 1 or (m > 1 and out.stride(0) < n)))):
        raise ValueError("out must be %s [%d, %d] with contiguous rows, got %s %s" % (out_dtype, m, n, out.dtype, list(out.shape)))
    if accumulate and (out is None or out_dtype != torch.float32 or gelu is not None):
        raise ValueError("accumulate needs a float32 `out` and no gelu")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (n,) or not bias.is_contiguous()):
        raise ValueError("bias must be float32 [%d], got %s %s" % (n, bias.dtype, list(bias.shape)))
    dev = weight.device
    for t in (x, bias, out):
        if t is not None and t.device != dev:
            raise ValueError("tensors on %s and %s" % (dev, t.device))
    lib = _library()
    with _lib.on(dev):
        if out is None:
            out = torch.empty((m, n), dtype=out_dtype, device=dev)
        a = _PACKED.pack(x.codes.data_ptr() if four else x.data_ptr(), x.scales.data_ptr() if four else 0,
                         0 if four else x.stride(0), weight.packed.data_ptr(), bias.data_ptr() if bias is not None else 0,
                         out.data_ptr(), out.stride(0), _TYPES[out_dtype], _GELU[gelu], 1 if accumulate else 0, m, n, k)
        _lib.check(lib.stt_mxfp4_matmul(a, _lib.stream(dev)))
    return out


SYMBOLS = ("stt_mxfp4_quantize", "stt_mxfp4_dequantize", "stt_mxfp4_packed_bytes", "stt_mxfp4_pack", "stt_mxfp4_matmul")
_declared = False


def _library():
    global _declared
    lib = _lib.load()
    if not _declared:
        vp, i32, i64 = C.c_void_p, C.c_int, C.c_int64
        lib.stt_mxfp4_quantize.restype = i32
        lib.stt_mxfp4_quantize.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp]
        lib.stt_mxfp4_dequantize.restype = i32
        lib.stt_mxfp4_dequantize.argtypes = [vp, vp, i64, i64, vp, i32, vp]
        lib.stt_mxfp4_packed_bytes.restype = C.c_size_t
        lib.stt_mxfp4_packed_bytes.argtypes = [i64, i64]
        lib.stt_mxfp4_pack.restype = i32
        lib.stt_mxfp4_pack.argtypes = [vp, vp, i64, i64, vp, vp]
        lib.stt_mxfp4_matmul.restype = i32
        lib.stt_mxfp4_matmul.argtypes = [vp, vp]
        _declared = True
    return lib
