"""The 4-bit operators beside the requantised weights, over the C ABI of include/llmini_b200_fp4.h.

Activations and gradients quantised to NVFP4 by rows or by columns, the product of NVFP4 operands, the linear layer and its
gradients, reading 4-bit tensors back, and a paged cache of keys and values.  Tensors are torch CUDA tensors used purely as
device buffers; every call enqueues its work on the current stream of the current device, which has to hold all of them.
"""
from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass, field

import torch

from . import _ffi
from ._ffi import SCALES_RAW, SCALES_SM100, check
from .nvfp4 import Nvfp4Tensor, _raw_stream

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
NVFP4_MAXIMA = 1024
_TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}


class Matrix(C.Structure):
    _fields_ = [("data", C.c_void_p), ("ld", C.c_uint64), ("rows", C.c_uint32), ("cols", C.c_uint32), ("type", C.c_uint32),
                ("reserved", C.c_uint32)]


class Operand(C.Structure):
    _fields_ = [("bytes", C.c_void_p), ("scales", C.c_void_p), ("scale", C.c_void_p), ("row_bytes", C.c_uint64), ("rows", C.c_uint32),
                ("cols", C.c_uint32), ("scale_count", C.c_uint32), ("reserved", C.c_uint32)]


class LinearGradients(C.Structure):
    _fields_ = [("grad", Matrix), ("x", Matrix), ("weight_t", Operand), ("grad_x", Matrix), ("grad_weight", Matrix), ("grad_rows", Operand),
                ("grad_columns", Operand), ("x_columns", Operand), ("d_maxima", C.c_void_p), ("accumulate", C.c_uint32), ("reserved", C.c_uint32)]


class Cache(C.Structure):
    _fields_ = [("bytes", C.c_void_p), ("scales", C.c_void_p), ("exponents", C.c_void_p), ("pages", C.c_uint32), ("page_size", C.c_uint32),
                ("heads", C.c_uint32), ("dim", C.c_uint32)]


class Vectors(C.Structure):
    _fields_ = [("data", C.c_void_p), ("sequence_stride", C.c_uint64), ("token_stride", C.c_uint64), ("head_stride", C.c_uint64),
                ("type", C.c_uint32), ("reserved", C.c_uint32)]


# The bytes of a Matrix and of a Vectors, which a call takes as they are: a fifth of the time that such an object takes.
_matrix_bytes, _vectors_bytes = struct.Struct("@PQIIII").pack, struct.Struct("@PQQQII").pack
_NO_MATRIX, _NO_OPERAND = bytes(C.sizeof(Matrix)), bytes(C.sizeof(Operand))
_declared = False


def _lib() -> C.CDLL:
    global _declared
    L = _ffi.lib()
    if not _declared:
        vp, u32, i = C.c_void_p, C.c_uint32, C.c_int
        sig = {
            "b2_nvfp4_quantize_rows": [vp, vp, vp],
            "b2_nvfp4_quantize_columns": [vp, vp, vp, vp],
            "b2_nvfp4_decode": [vp, u32, vp, vp],
            "b2_nvfp4_matmul": [vp, vp, vp, vp, u32, vp],
            "b2_nvfp4_linear_forward": [vp, vp, vp, vp, vp, vp],
            "b2_nvfp4_linear_backward": [vp, vp],
            "b2_nvfp4_status": [vp],
            "b2_nvfp4_cache_write": [vp, vp, u32, vp, u32, vp],
            "b2_nvfp4_cache_read": [vp, vp, u32, vp, u32, vp, u32, u32, vp],
        }
        for name, args in sig.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = i, args
        _declared = True
    return L


def _refuse(what: str):
    raise ValueError(what)


# The current device, and its current stream's handle, without the objects around them: of the 4 to 5 us that a call on small
# tensors takes on the host, the launch itself is 2.5.
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream_of(device: int) -> int:
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _here(t: torch.Tensor, device: int) -> int:
    """The address of a tensor of the current device."""
    if t.get_device() != device:
        _refuse(f"a tensor on {t.device}: the call works on the current CUDA device")
    return t.data_ptr()


def _matrix(t: torch.Tensor, device: int) -> bytes:
    kind = _TYPES.get(t.dtype)
    if kind is None or t.dim() != 2:
        _refuse(f"a matrix of FP32, BF16 or F16 is wanted, not {tuple(t.shape)} of {t.dtype}")
    (rows, cols), (ld, step) = t.shape, t.stride()
    if step != 1 and cols > 1:
        _refuse("a row's values have to lie side by side")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        _refuse("rows overlap")
    if t.get_device() != device:
        _refuse(f"a tensor on {t.device}: the call works on the current CUDA device")
    try:
        return _matrix_bytes(t.data_ptr(), ld, rows, cols, kind, 0)
    except struct.error:
        _refuse("rows and columns are 32-bit numbers")


def _overlaps(t: torch.Tensor) -> bool:
    """Whether values of a tensor lie in one place: whether a dimension's step is shorter than what the smaller steps reach over."""
    reach = 1
    for step, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1):
        if step < reach and t.numel():
            return True
        reach += step * (n - 1)
    return False


def _floats(t: torch.Tensor, count: int, what: str, device: int) -> int:
    if t.dtype != torch.float32 or t.numel() < count or not t.is_contiguous():
        _refuse(f"{what}: {count} contiguous FP32 values are wanted")
    return _here(t, device)


def _operand(o: "Nvfp4Operand", device: int):
    if o.device_index != device:
        _refuse("an operand of another device than the current one")
    return o.ref


def _csf_bytes(rows: int, k: int) -> int:
    return int(_ffi.lib().b2_csf_encoded_len(rows, k))


def _up(n: int, step: int) -> int:
    return -(-n // step) * step


class _Described:
    """An object whose tensors' addresses calls take from a structure made once (`_describe`: what follows from the fields).  Fields
    are looked over before they are stored, together with what follows from them; a field that is refused changes nothing."""

    def __post_init__(self):
        self.replace()

    def __setattr__(self, name, value):
        if name in self._FIELDS and "c" in self.__dict__:
            self.replace(**{name: value})
        else:
            object.__setattr__(self, name, value)

    def replace(self, **fields) -> None:
        """Other values for some fields at once, as another size needs."""
        if not fields.keys() <= set(self._FIELDS):
            raise TypeError(f"fields are {self._FIELDS}")
        self.__dict__.update(self._describe(**{n: fields.get(n, self.__dict__[n]) for n in self._FIELDS}))


def _tensors(*tensors) -> bool:
    return all(isinstance(t, torch.Tensor) for t in tensors)


@dataclass
class Nvfp4Operand(_Described):
    """A matrix in NVFP4 as the product reads it: codes [rows, row_bytes] (two a byte, k / 2 of a row's bytes), block scales in the
    tensor cores' layout (SCALES_SM100), and the scale on top, one or one a row.  k: the values of a row, a multiple of 16."""
    bytes: torch.Tensor
    scales: torch.Tensor
    scale: torch.Tensor
    rows: int
    k: int
    c: Operand = field(init=False, repr=False)
    _FIELDS = ("bytes", "scales", "scale", "rows", "k")

    @staticmethod
    def _describe(bytes, scales, scale, rows, k):
        b = bytes
        if not _tensors(b, scales, scale) or b.dtype != torch.uint8 or b.dim() != 2 or b.shape[0] != rows or (b.shape[1] > 1 and b.stride(1) != 1):
            _refuse("codes: uint8 [rows, bytes of a row]")
        row_bytes = b.stride(0) if rows > 1 else _up(b.shape[1], 16)
        if k % 16 or k <= 0 or b.shape[1] < k // 2 or row_bytes % 16:
            _refuse("a row: k values, a multiple of 16, on a 16-byte boundary")
        if scales.dtype != torch.uint8 or not scales.is_contiguous() or scales.numel() < _up(rows, 128) * _up(k // 16, 4):
            _refuse("scales: a contiguous buffer of sm100_scales_bytes(rows, k) bytes")
        n = scale.numel()
        if scale.dtype != torch.float32 or not scale.is_contiguous() or n not in (1, rows):
            _refuse("scale: FP32, one or one a row")
        if rows and (b.data_ptr() % 16 or scales.data_ptr() % 16):
            _refuse("codes and scales start on 16-byte boundaries")
        if not (b.device == scales.device == scale.device) or not b.is_cuda:
            _refuse("an operand lies on one CUDA device")
        c = Operand(b.data_ptr(), scales.data_ptr(), scale.data_ptr(), row_bytes, rows, k, n, 0)
        return dict(bytes=bytes, scales=scales, scale=scale, rows=rows, k=k, device_index=b.device.index, c=c, ref=C.byref(c))

    @staticmethod
    def empty(rows: int, k: int, per_row: bool = True, device="cuda") -> "Nvfp4Operand":
        """Memory for `rows` rows of k values, rounded up to a multiple of 16: what the quantisers write."""
        k = max(_up(k, 16), 16)
        return Nvfp4Operand(torch.empty(rows, _up(k // 2, 16), dtype=torch.uint8, device=device),
                            torch.zeros(max(_up(rows, 128) * _up(k // 16, 4), 16), dtype=torch.uint8, device=device),
                            torch.empty(rows if per_row else 1, dtype=torch.float32, device=device), rows, k)

    @staticmethod
    def from_tensor(t: Nvfp4Tensor) -> "Nvfp4Operand":
        """A requantised weight [rows][k] as it lies, its scales in SCALES_SM100 (a plan of that layout, or `scales_to_sm100`);
        k has to be a multiple of 32, so that rows start on 16-byte boundaries."""
        if t.scale_layout != SCALES_SM100:
            _refuse("scales in SCALES_SM100 are wanted: see scales_to_sm100")
        return Nvfp4Operand(t.bytes.view(t.rows, t.k // 2), t.scales, t.global_scale, t.rows, t.k)


class Nvfp4LinearScratch:
    """Memory of a linear layer's calls on `tokens` rows: its quantised activations, with `backward` also what the gradients
    need.  Calls that may run at the same time, captured ones too, each need their own."""

    def __init__(self, tokens: int, inputs: int, outputs: int, backward: bool = False, device="cuda"):
        self.rows = None if backward else Nvfp4Operand.empty(tokens, inputs, device=device)
        self.backward = backward
        if backward:
            self.grad_rows = Nvfp4Operand.empty(tokens, outputs, device=device)
            self.grad_columns = Nvfp4Operand.empty(outputs, tokens, per_row=False, device=device)
            self.x_columns = Nvfp4Operand.empty(inputs, tokens, per_row=False, device=device)
            self.maxima = torch.empty(2 * NVFP4_MAXIMA, dtype=torch.float32, device=device)


@dataclass
class Nvfp4PagedCache(_Described):
    """Keys and values in pages: for each, codes [pages, page_size, heads, dim / 2], block scales [.., dim / 16] and exponents
    [pages, page_size, heads], all uint8 and contiguous.  `value` may be None: a cache of one tensor.  Sides are kept as tuples."""
    key: tuple
    value: tuple | None = None
    c: object = field(init=False, repr=False)
    _FIELDS = ("key", "value")

    @staticmethod
    def _describe(key, value):
        sides = []
        for side in (key,) if value is None else (key, value):
            side = tuple(side) if isinstance(side, (tuple, list)) else ()
            if len(side) != 3 or not _tensors(*side) or side[0].dim() != 4:
                _refuse("a side of a cache: codes, scales and exponents")
            codes, scales, exponents = side
            pages, page_size, heads, half = codes.shape
            shapes = (codes.shape, scales.shape, exponents.shape) == ((pages, page_size, heads, half), (pages, page_size, heads, half // 8), (pages, page_size, heads))
            if half % 8 or not shapes or any(t.dtype != torch.uint8 or not t.is_contiguous() for t in side):
                _refuse("a cache: uint8 [pages, page_size, heads, dim / 2], [.., dim / 16], [pages, page_size, heads]")
            sides.append(side)
        first = sides[0][0]
        if any(not t.is_cuda or t.device != first.device for side in sides for t in side):
            _refuse("a cache lies on one CUDA device")
        c = (Cache * len(sides))(*(Cache(*(t.data_ptr() for t in side), *side[2].shape, side[0].shape[3] * 2) for side in sides))
        return dict(key=sides[0], value=sides[1] if len(sides) > 1 else None, device_index=first.device.index, c=c,
                    sizes=[(side[2].shape[2], side[0].shape[3] * 2) for side in sides])

    @staticmethod
    def empty(pages: int, page_size: int, heads: int, dim: int, value_dim: int | None = None, device="cuda") -> "Nvfp4PagedCache":
        def side(d):
            return tuple(torch.zeros(pages, page_size, heads, *more, dtype=torch.uint8, device=device) for more in ((d // 2,), (d // 16,), ()))
        return Nvfp4PagedCache(side(dim), side(value_dim or dim))


class Nvfp4LinearModule:
    """The entry points, named after those of the library."""

    def __init__(self):
        self._lib = _lib()

    def quantize_rows(self, x: torch.Tensor, out: Nvfp4Operand) -> None:
        d = _device()
        check(self._lib.b2_nvfp4_quantize_rows(_matrix(x, d), _operand(out, d), _stream_of(d)), "nvfp4_quantize_rows")

    def quantize_columns(self, x: torch.Tensor, out: Nvfp4Operand, maxima: torch.Tensor) -> None:
        """The transpose of x; `maxima`: scratch of NVFP4_MAXIMA FP32 values."""
        d = _device()
        check(self._lib.b2_nvfp4_quantize_columns(_matrix(x, d), _operand(out, d), _floats(maxima, NVFP4_MAXIMA, "maxima", d), _stream_of(d)),
              "nvfp4_quantize_columns")

    def decode(self, operand, out: torch.Tensor) -> None:
        """The values of an Nvfp4Operand, or of an Nvfp4Tensor of any scale layout, in out's type."""
        d = _device()
        if isinstance(operand, Nvfp4Tensor):
            t, layout = operand, operand.scale_layout
            if (t.k // 2) % 16 and t.rows > 1:
                _refuse("rows of k values start on 16-byte boundaries where k is a multiple of 32")
            need = _up(t.rows, 128) * _up(t.k // 16, 4) if layout == SCALES_SM100 else t.rows * t.k // 16 if layout == SCALES_RAW else _csf_bytes(t.rows, t.k)
            if t.bytes.numel() < t.rows * t.k // 2 or t.scales.numel() < need or not (t.bytes.is_contiguous() and t.scales.is_contiguous()):
                _refuse("an Nvfp4Tensor with too little memory for its rows and k, or with gaps in it")
            c = C.byref(Operand(_here(t.bytes, d), _here(t.scales, d), _floats(t.global_scale, 1, "global_scale", d), _up(t.k // 2, 16), t.rows, t.k, 1, 0))
        else:
            c, layout = _operand(operand, d), SCALES_SM100
        check(self._lib.b2_nvfp4_decode(c, layout, _matrix(out, d), _stream_of(d)), "nvfp4_decode")

    def matmul(self, a: Nvfp4Operand, b: Nvfp4Operand, out: torch.Tensor, bias: torch.Tensor | None = None, accumulate: bool = False) -> None:
        """out [a.rows, b.rows] = a b^T (+ bias) (+ out, FP32 only)."""
        d = _device()
        check(self._lib.b2_nvfp4_matmul(_operand(a, d), _operand(b, d), _matrix(out, d),
                                        None if bias is None else _floats(bias, b.rows, "bias", d), int(accumulate), _stream_of(d)), "nvfp4_matmul")

    def linear_forward(self, x: torch.Tensor, weight: Nvfp4Operand, out: torch.Tensor, scratch: Nvfp4LinearScratch,
                       bias: torch.Tensor | None = None) -> None:
        """out [tokens, outputs] = Q(x) weight^T (+ bias)."""
        d = _device()
        if scratch.rows is None:
            _refuse("scratch of the backward pass")
        check(self._lib.b2_nvfp4_linear_forward(_matrix(x, d), _operand(weight, d), _matrix(out, d),
                                                None if bias is None else _floats(bias, weight.rows, "bias", d), _operand(scratch.rows, d),
                                                _stream_of(d)), "nvfp4_linear_forward")

    def linear_backward(self, grad: torch.Tensor, x: torch.Tensor | None, weight_t: Nvfp4Operand | None, grad_x: torch.Tensor | None,
                        grad_weight: torch.Tensor | None, scratch: Nvfp4LinearScratch, accumulate: bool = False) -> None:
        """grad_x [tokens, inputs] and grad_weight [outputs, inputs] (FP32) of linear_forward; either may be None.  weight_t: the
        transposed weight, quantised along the outputs (quantize_columns of the master weights)."""
        d = _device()
        if not scratch.backward:
            _refuse("scratch of the forward pass")
        if (grad_x is not None and weight_t is None) or (grad_weight is not None and x is None):
            _refuse("grad_x wants weight_t, grad_weight wants x")
        kept = (scratch.grad_rows, scratch.grad_columns, scratch.x_columns)
        for o in kept if grad_x is None else kept + (weight_t,):
            _operand(o, d)
        # a LinearGradients
        args = b"".join((_matrix(grad, d), _matrix(x, d) if grad_weight is not None else _NO_MATRIX,
                         bytes(weight_t.c) if grad_x is not None else _NO_OPERAND, _matrix(grad_x, d) if grad_x is not None else _NO_MATRIX,
                         _matrix(grad_weight, d) if grad_weight is not None else _NO_MATRIX, *(bytes(o.c) for o in kept),
                         struct.pack("@PII", _floats(scratch.maxima, 2 * NVFP4_MAXIMA, "maxima", d), int(accumulate), 0)))
        check(self._lib.b2_nvfp4_linear_backward(args, _stream_of(d)), "nvfp4_linear_backward")

    def status(self) -> int:
        """0, or ERROR_LAUNCH_TIMEOUT if a bounded device wait of a product ran out since the last call (synchronises)."""
        return int(self._lib.b2_nvfp4_status(_stream_of(_device())))

    @staticmethod
    def _sides(cache: Nvfp4PagedCache, tensors, dims: int, d: int):
        if cache.device_index != d:
            _refuse("a cache of another device than the current one")
        if (tensors[1] is None) != (len(cache.c) == 1):
            _refuse("one tensor for each side of the cache")
        v, first, n = b"", tensors[0], len(cache.c)
        kind = _TYPES.get(first.dtype)
        if kind is None or first.dim() != dims:
            _refuse(f"vectors of FP32, BF16 or F16 are wanted, not {tuple(first.shape)} of {first.dtype}")
        for i in range(n):
            t, shape, stride = tensors[i], tensors[i].shape, tensors[i].stride()
            if shape[-2:] != cache.sizes[i] or stride[-1] != 1:
                _refuse("vectors of the cache's heads and size, their values side by side")
            if dims == 4 and not t.is_contiguous() and _overlaps(t):
                _refuse("vectors that are written lie apart")
            if i and (t.dtype != first.dtype or shape[:-2] != first.shape[:-2]):
                _refuse("keys and values: tensors of one type and length")
            at = _here(t, d)
            if dims == 4 and i and at == first.data_ptr() and t.numel():
                _refuse("keys and values go to places of their own")
            v += _vectors_bytes(at, stride[0] if dims == 4 else 0, stride[-3], stride[-2], kind, 0)
        return v, n, first.shape

    def cache_write(self, cache: Nvfp4PagedCache, slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor | None = None) -> None:
        """key, value [tokens, heads, dim] into slots int64 [tokens] (page * page_size + place; others leave a token out)."""
        d = _device()
        v, n, shape = self._sides(cache, (key, value), 3, d)
        if slots.dtype != torch.int64 or slots.shape != shape[:1] or not slots.is_contiguous():
            _refuse("slots: int64 [tokens]")
        check(self._lib.b2_nvfp4_cache_write(cache.c, v, n, _here(slots, d), shape[0], _stream_of(d)), "nvfp4_cache_write")

    def cache_read(self, cache: Nvfp4PagedCache, table: torch.Tensor, lengths: torch.Tensor, key: torch.Tensor,
                   value: torch.Tensor | None = None) -> None:
        """The first lengths[b] tokens of every sequence b, whose pages table [sequences, pages of a sequence] lists, into key,
        value [sequences, tokens, heads, dim]; what lies behind them is left as it is.  table, lengths: int32."""
        d = _device()
        v, n, shape = self._sides(cache, (key, value), 4, d)
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.shape[0] != shape[0]:
            _refuse("table: int32 [sequences, pages of a sequence]")
        if lengths.dtype != torch.int32 or lengths.shape != shape[:1] or not lengths.is_contiguous():
            _refuse("lengths: int32 [sequences]")
        check(self._lib.b2_nvfp4_cache_read(cache.c, v, n, _here(table, d), table.shape[1], _here(lengths, d), shape[0], shape[1],
                                            _stream_of(d)), "nvfp4_cache_read")
