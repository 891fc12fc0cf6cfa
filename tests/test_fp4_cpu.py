"""The 4-bit operators without a GPU: what the header declares is exported and mirrored, what is wrong is refused before anything
is launched, and the plain definition that the kernels are tested against does what it says."""
import ctypes as C
import os
import re
import struct

import numpy as np
import pytest
import torch

import llmini_b200 as b2
from llmini_b200 import _ffi, fp4
from tests import fp4_plain as plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "llmini_b200_fp4.h")).read(), flags=re.S)
SHIM = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "rust-shim", "src", "fp4.rs")).read())
INVALID = _ffi.ERROR_INVALID_VALUE
AT = 4096   # an address that is never looked at


def structs(text):
    return {m.group(1): [re.findall(r"(\w+)\s*$", part.strip())[0] for decl in m.group(2).split(";") if decl.strip() for part in decl.split(",")]
            for m in re.finditer(r"typedef\s+struct\s+(b2_\w+)\s*\{(.*?)\}\s*\1\s*;", text, flags=re.S)}


def test_exports_and_mirrors():
    declared = {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"\b(b2_nvfp4_\w+)\s*\(([^;{}]*?)\)\s*;", HEADER, flags=re.S)}
    assert len(declared) == 9
    for name in declared:
        fn = getattr(fp4._lib(), name)
        assert len(fn.argtypes) == declared[name], name
    bound = {m.group(1): len([a for a in m.group(2).split(",") if a.strip()]) for m in re.finditer(r"pub fn (b2_nvfp4_\w+)\s*\((.*?)\)\s*->", SHIM, flags=re.S)}
    assert bound == declared
    mirrors = {"b2_matrix": fp4.Matrix, "b2_nvfp4_operand": fp4.Operand, "b2_nvfp4_linear_gradients": fp4.LinearGradients, "b2_nvfp4_cache": fp4.Cache,
               "b2_vectors": fp4.Vectors}
    h = structs(HEADER)
    assert set(h) == set(mirrors)
    for name, fields in h.items():
        assert [f for f, _ in mirrors[name]._fields_] == fields, name
        body = re.search(rf"#\[repr\(C\)\][^{{;]*?pub struct {name}\s*\{{(.*?)\n\}}", SHIM, flags=re.S).group(1)
        assert re.findall(r"pub (?:r#)?(\w+)\s*:", body) == fields, name
    assert [C.sizeof(t) for t in mirrors.values()] == [32, 48, 336, 40, 40]
    assert int(re.search(r"#define B2_NVFP4_MAXIMA (\d+)", HEADER).group(1)) == b2.NVFP4_MAXIMA == int(re.search(r"B2_NVFP4_MAXIMA: usize = (\d+)", SHIM).group(1))
    for name, value in re.findall(r"(B2_TYPE_\w+) = (\d)", HEADER):
        assert re.search(rf"pub const {name}: u32 = {value};", SHIM), name


def matrix(rows, cols, ld=None, type=fp4.TYPE_BF16, data=AT):
    return fp4.Matrix(data, cols if ld is None else ld, rows, cols, type, 0)


def operand(rows, cols, count=None, row_bytes=None, data=AT):
    return fp4.Operand(data, data, data, -(-cols // 32) * 16 if row_bytes is None else row_bytes, rows, cols, rows if count is None else count, 0)


def with_field(struct, **fields):
    for name, v in fields.items():
        setattr(struct, name, v)
    return struct


BAD_MATRICES = [matrix(4, 64, data=None), matrix(4, 64, ld=63), matrix(4, 64, type=3), matrix(4, 64, data=AT + 1), with_field(matrix(4, 64), reserved=1),
                matrix(4, 64, ld=1 << 40), matrix(65535 * 128 + 1, 64)]
BAD_OPERANDS = [operand(4, 64, data=None), operand(4, 64, data=AT + 8), operand(4, 64, row_bytes=40), operand(4, 64, row_bytes=16), operand(4, 64, count=3),
                operand(4, 72), with_field(operand(4, 64), reserved=7), operand(4, 64, row_bytes=1 << 40)]


def test_bytes_of_the_mirrors():
    """What the Python calls pass in a structure's place is that structure."""
    assert bytes(fp4.Matrix(1 << 40, 1 << 35, 3, 4, 2, 0)) == fp4._matrix_bytes(1 << 40, 1 << 35, 3, 4, 2, 0)
    assert bytes(fp4.Vectors(1 << 40, 1 << 35, 1 << 34, 64, 1, 0)) == fp4._vectors_bytes(1 << 40, 1 << 35, 1 << 34, 64, 1, 0)
    m, o = C.sizeof(fp4.Matrix), C.sizeof(fp4.Operand)
    g = fp4.LinearGradients
    assert [f.offset for f in (g.x, g.weight_t, g.grad_x, g.grad_weight, g.grad_rows, g.grad_columns, g.x_columns, g.d_maxima)] == \
        [m, 2 * m, 2 * m + o, 3 * m + o, 4 * m + o, 4 * m + 2 * o, 4 * m + 3 * o, 4 * m + 4 * o]
    assert C.sizeof(g) == 4 * m + 4 * o + struct.calcsize("@PII") and len(fp4._NO_MATRIX) == m and len(fp4._NO_OPERAND) == o
    with pytest.raises(ValueError):
        fp4._matrix(torch.empty(1, dtype=torch.float32).expand(1 << 33, 1), -1)


def test_quantisers_refuse():
    L = fp4._lib()
    rows = lambda x, o: L.b2_nvfp4_quantize_rows(C.byref(x) if x else None, C.byref(o) if o else None, None)
    columns = lambda x, o, maxima=AT: L.b2_nvfp4_quantize_columns(C.byref(x) if x else None, C.byref(o) if o else None, maxima, None)
    good = (matrix(4, 64), operand(4, 64))
    assert rows(None, good[1]) == rows(good[0], None) == INVALID
    for bad in BAD_MATRICES:
        assert rows(bad, good[1]) == INVALID, bad.ld
        assert columns(bad, operand(64, 16, 1)) == INVALID
    for bad in BAD_OPERANDS:
        assert rows(good[0], bad) == INVALID
    for o in (operand(5, 64), operand(4, 80), operand(4, 64, 1)):
        assert rows(good[0], o) == INVALID
    for o in (operand(64, 32, 1), operand(63, 16, 1), operand(64, 16), operand(64, 16, 1, data=None)):
        assert columns(good[0], o) == INVALID
    assert columns(good[0], operand(64, 16, 1), None) == columns(good[0], operand(64, 16, 1), AT + 2) == INVALID
    assert columns(matrix(0, 64), operand(64, 16, 1)) == INVALID
    assert rows(matrix(0, 64), operand(0, 64)) == 0


def test_products_refuse():
    L = fp4._lib()
    mm = lambda a, b, c, bias=None, acc=0: L.b2_nvfp4_matmul(C.byref(a), C.byref(b), C.byref(c), bias, acc, None)
    a, b, c = operand(4, 64), operand(8, 64, 1), matrix(4, 8, type=fp4.TYPE_F32)
    for bad in BAD_OPERANDS:
        assert mm(bad, b, c) == INVALID and mm(a, bad, matrix(4, bad.rows)) == INVALID
    for bad in BAD_MATRICES:
        assert mm(operand(4, 64), operand(64, 64, 1), bad) == INVALID
    assert mm(a, operand(8, 48, 1), c) == mm(a, b, matrix(4, 9)) == mm(a, b, matrix(5, 8)) == INVALID
    assert mm(a, b, c, bias=AT + 2) == mm(a, b, c, acc=2) == mm(a, b, matrix(4, 8), acc=1) == INVALID
    assert mm(operand(0, 64), b, matrix(0, 8)) == mm(a, operand(0, 64, 1), matrix(4, 0)) == 0
    fw = lambda x, w, y, s: L.b2_nvfp4_linear_forward(C.byref(x), C.byref(w), C.byref(y), None, C.byref(s), None)
    assert fw(matrix(4, 64), b, matrix(4, 8), operand(4, 64, 1)) == INVALID
    assert fw(matrix(4, 60), b, matrix(4, 8), operand(4, 80)) == fw(matrix(4, 80), b, matrix(4, 8), operand(4, 80)) == INVALID
    assert fw(matrix(0, 64), b, matrix(0, 8), operand(0, 64)) == 0

    def bw(**fields):
        g = fp4.LinearGradients(matrix(20, 8), matrix(20, 64), operand(64, 16, 1), matrix(20, 64), matrix(8, 64, type=fp4.TYPE_F32), operand(20, 16),
                                operand(8, 32, 1), operand(64, 32, 1), AT, 0, 0)
        return L.b2_nvfp4_linear_backward(C.byref(with_field(g, **fields)), None)
    for fields in (dict(grad=matrix(20, 0)), dict(x=matrix(19, 64)), dict(weight_t=operand(64, 32, 1)), dict(grad_x=matrix(20, 63)), dict(d_maxima=None),
                   dict(grad_weight=matrix(8, 64)), dict(grad_weight=matrix(64, 8, type=fp4.TYPE_F32)), dict(grad_rows=operand(20, 16, 1)),
                   dict(grad_columns=operand(8, 32)), dict(x_columns=operand(64, 16, 1)), dict(accumulate=2), dict(reserved=1)):
        assert bw(**fields) == INVALID, fields


def test_decode_refuses():
    L = fp4._lib()
    dec = lambda o, m, layout=2: L.b2_nvfp4_decode(C.byref(o), layout, C.byref(m), None)
    for bad in BAD_OPERANDS:
        assert dec(bad, matrix(4, 64)) == INVALID
    for bad in BAD_MATRICES:
        assert dec(operand(4, 64), bad) == INVALID
    assert dec(operand(4, 64), matrix(4, 48)) == dec(operand(4, 64), matrix(3, 64)) == dec(operand(4, 64), matrix(4, 64), 3) == INVALID
    assert dec(operand(4, 64), matrix(4, 64), 0) == INVALID                                   # CSF: whole 128-value pieces
    assert dec(operand(65536, 1 << 21, 1), matrix(65536, 1 << 21), 0) == INVALID              # and 32-bit group numbers


def test_cache_refuses():
    L = fp4._lib()
    cache = lambda **f: (fp4.Cache * 1)(with_field(fp4.Cache(AT, AT, AT, 4, 16, 2, 64), **f))
    vectors = lambda **f: (fp4.Vectors * 1)(with_field(fp4.Vectors(AT, 4096, 128, 64, fp4.TYPE_BF16, 0), **f))
    write = lambda c, v, count=1, slots=AT, n=5: L.b2_nvfp4_cache_write(c, v, count, slots, n, None)
    read = lambda c, v, count=1, table=AT, lengths=AT, b=2, n=30: L.b2_nvfp4_cache_read(c, v, count, table, 2, lengths, b, n, None)
    for f in (dict(bytes=None), dict(bytes=AT + 4), dict(scales=None), dict(exponents=None), dict(page_size=0), dict(heads=0), dict(dim=40), dict(dim=0),
              dict(dim=1040), dict(heads=65536)):
        assert write(cache(**f), vectors()) == read(cache(**f), vectors()) == INVALID, f
    for f in (dict(data=None), dict(data=AT + 1), dict(type=3), dict(reserved=1), dict(token_stride=1 << 40)):
        assert write(cache(), vectors(**f)) == read(cache(), vectors(**f)) == INVALID, f
    assert write(cache(), vectors(), 0) == write(cache(), vectors(), 3) == write(cache(), vectors(), slots=None) == write(cache(), vectors(), slots=AT + 4) == INVALID
    assert read(cache(), vectors(), 0) == read(cache(), vectors(), table=None) == read(cache(), vectors(), lengths=AT + 2) == read(cache(), vectors(), b=65536) == INVALID
    two = (fp4.Vectors * 2)(vectors()[0], vectors(type=fp4.TYPE_F16)[0])
    assert write((fp4.Cache * 2)(cache()[0], cache()[0]), two, 2) == INVALID
    assert write(cache(), vectors(), n=0) == read(cache(), vectors(), b=0) == read(cache(), vectors(), n=0) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_calls_fail_loudly_without_a_gpu():
    L = fp4._lib()
    assert L.b2_nvfp4_quantize_rows(C.byref(matrix(4, 64)), C.byref(operand(4, 64)), None) not in (0, INVALID)
    assert L.b2_nvfp4_matmul(C.byref(operand(4, 64)), C.byref(operand(8, 64, 1)), C.byref(matrix(4, 8)), None, 0, None) not in (0, INVALID)
    with pytest.raises((ValueError, RuntimeError)):
        b2.Nvfp4LinearModule().quantize_rows(torch.zeros(4, 64), None)


def test_plain_definition():
    x = np.array([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0] + [0.0] * 8])
    codes, s, g = plain.quantise(x)
    assert g[0] == 2.0 ** -8 and s[0, 0] == 0x78 and plain.e4m3_grid()[0x78] == 256 and codes.shape == (1, 32)   # 1 / 2^-8
    assert codes[0, :10].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 14]
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 100)) * np.exp2(rng.integers(-20, 20, (5, 1)))
    codes, s, g = plain.quantise(x)
    err = np.abs(plain.values(codes, s, g)[:, :100] - x)
    step = np.repeat(plain.e4m3_grid()[s] * g[:, None], 16, 1)[:, :100]
    assert (err <= 1.4 * step).all()   # half the widest step, and what saturates: 6 (1 + 1/16) - 6
    assert np.array_equal(plain.untiled(plain.tiled(s), 5, 7)[0], s) and np.array_equal(plain.unpack(plain.pack(codes), 112), codes)


def test_every_kernel_waits_before_it_touches_memory():
    """All kernels of these operators are launched so that they may begin while the launch in front still runs."""
    csrc = os.path.join(ROOT, "llmini_b200", "csrc")
    text = "".join(re.sub(r"//[^\n]*", "", open(os.path.join(csrc, n)).read()) for n in ("fp4_kernels.cu", "fp4_gemm_sm100.cu"))
    kernels = re.findall(r"__global__[^;{]*?\b(k_fp4_\w+)\(([^{]*)\)\s*\{(.*?)\n\}", text, flags=re.S)
    assert len(kernels) >= 7
    for name, _, body in kernels:
        assert body.count("stream_enter();") == 1, name
        before = body.split("stream_enter();")[0]
        assert "return" not in re.sub(r"\{ return [^}]*\}", "", before), name
        assert "ld.global" not in before and "tma_load" not in before, name
    for form in ("__ldg(", "ld.global.nc", "const float *__restrict__"):
        assert form not in text, form


class OnDevice(torch.Tensor):
    """Host memory that passes for memory of a CUDA device: what is described and refused needs no GPU."""
    is_cuda = property(lambda self: True)


def on_device(*shape, dtype=torch.uint8):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def whole_operand(rows, k):
    return dict(bytes=on_device(rows, -(-k // 32) * 16), scales=on_device(-(-rows // 128) * -(-k // 64) * 512), scale=on_device(rows, dtype=torch.float32), rows=rows,
                k=k)


def test_a_refused_field_changes_nothing():
    """An operand and a cache refuse a field before they take it: what calls read (c) is what the fields hold, before and after."""
    kept = whole_operand(40, 64)
    o = b2.Nvfp4Operand(**kept)

    def agrees():
        assert (o.c.bytes, o.c.scales, o.c.scale) == (o.bytes.data_ptr(), o.scales.data_ptr(), o.scale.data_ptr())
        assert (o.c.rows, o.c.cols, o.c.row_bytes, o.c.scale_count) == (o.rows, o.k, o.bytes.stride(0), o.scale.numel())
        assert o.ref._obj is o.c
    agrees()
    for name, bad in (("bytes", on_device(39, 32)), ("bytes", torch.zeros(40, 32, dtype=torch.uint8)), ("bytes", on_device(40, 24)), ("bytes", None),
                      ("scales", on_device(511)), ("scale", on_device(39, dtype=torch.float32)), ("scale", on_device(40)), ("rows", 39), ("rows", 41),
                      ("k", 80), ("k", 72), ("k", 0), ("rows", "40"), ("rows", 1 << 32)):
        with pytest.raises(ValueError):
            setattr(o, name, bad)
        assert all(getattr(o, n) is v for n, v in kept.items()), name
        agrees()
    o.bytes, o.k = on_device(40, 48), 48
    agrees()
    larger = whole_operand(300, 160)
    with pytest.raises(ValueError):
        o.replace(**{**larger, "scale": on_device(299, dtype=torch.float32)})
    assert o.rows == 40
    agrees()
    o.replace(**larger)
    assert o.rows == 300 and o.bytes is larger["bytes"]
    agrees()

    def side(pages, page, heads, dim):
        return tuple(on_device(pages, page, heads, *more) for more in ((dim // 2,), (dim // 16,), ()))
    key, value = side(4, 8, 2, 32), side(4, 8, 2, 48)
    cache = b2.Nvfp4PagedCache(key, value)

    def follows(n=2):
        assert len(cache.c) == len(cache.sizes) == n and (cache.value is None) == (n == 1)
        for c, s, size in zip(cache.c, (cache.key, cache.value), cache.sizes):
            assert [c.bytes, c.scales, c.exponents] == [t.data_ptr() for t in s]
            assert (c.pages, c.page_size, c.heads, c.dim) == (*s[2].shape, s[0].shape[-1] * 2) and size == (c.heads, c.dim)
    follows()
    before = cache.key, cache.value, cache.c
    for bad in (side(4, 8, 2, 40), side(4, 8, 2, 32)[:2], [torch.zeros(4, 8, 2, n, dtype=torch.uint8) for n in (16, 2)] + [torch.zeros(4, 8, 2, dtype=torch.uint8)],
                side(4, 8, 2, 32)[::-1], [t[:, :, :1] for t in side(4, 8, 2, 32)], None, 7):
        for name in ("key",) if bad is None else ("key", "value"):
            with pytest.raises(ValueError):
                setattr(cache, name, bad)
            assert (cache.key, cache.value, cache.c) == before
            follows()
    cache.key = side(9, 8, 3, 64)
    follows()
    cache.value = None
    follows(1)


def test_a_cache_keeps_its_own_tuples():
    """Sides may be given as lists; what happens to these later is not half followed."""
    def side():
        return [on_device(4, 8, 2, *more) for more in ((16,), (2,), ())]
    key, value = side(), side()
    cache = b2.Nvfp4PagedCache(key, value)
    kept = tuple(key), tuple(value)
    key[0], value[1] = on_device(4, 8, 2, 16), on_device(4, 8, 2, 2)

    def holds(key, value):
        assert isinstance(cache.key, tuple) and all(a is b for a, b in zip(cache.key + cache.value, key + value))
        assert [(c.bytes, c.scales, c.exponents) for c in cache.c] == [tuple(t.data_ptr() for t in s) for s in (key, value)]
    holds(*kept)
    with pytest.raises(TypeError):
        cache.key[0] = on_device(4, 8, 2, 16)
    holds(*kept)
    cache.key = key
    key.reverse()
    holds(tuple(key[::-1]), kept[1])


def test_plain_rounding():
    x = np.random.default_rng(0).standard_normal(4000).astype(np.float32) * np.exp2(np.arange(4000) % 60 - 30).astype(np.float32)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):   # one rounding of FP32 values, which torch does too
        assert np.array_equal(plain.rounded_once(x, dtype), torch.from_numpy(x).to(dtype).double().numpy())
    big = torch.finfo(torch.float16).max
    assert plain.rounded_once([big + 15.9, big + 16, -big - 16, 2.0 ** -25, 2.0 ** -24 * 1.5, -0.0], torch.float16).tolist() == [big, np.inf, -np.inf, 0, 2.0 ** -23, 0]
    assert plain.rounded_once([1 + 2.0 ** -8 + 2.0 ** -40], torch.bfloat16).tolist() == [1 + 2.0 ** -7]   # in two steps it would be 1


@pytest.mark.parametrize("rows,k", [(1, 16), (33, 48), (128, 64), (130, 1600), (1000, 384)])
def test_memory_of_a_tensor_in_every_scale_layout(rows, k):
    """Nvfp4Tensor.empty has room for the scales in the layout that it is asked for."""
    sizes = {b2.SCALES_RAW: rows * k // 16, b2.SCALES_SM100: -(-rows // 128) * -(-k // 64) * 512}
    if k % 128 == 0:
        sizes[b2.SCALES_CSF] = b2.csf_encoded_len(rows, k)
    for layout, size in sizes.items():
        t = b2.Nvfp4Tensor.empty(rows, k, layout, device="cpu")
        assert (t.bytes.numel(), t.scales.numel(), t.scale_layout) == (rows * k // 2, size, layout)
        assert layout == b2.SCALES_CSF or not t.scales.any()


def test_results_of_a_cache_lie_apart():
    """Vectors that are read into may be in any order and at any distance, but not over one another."""
    n = 4096
    memory = torch.zeros(n).as_subclass(OnDevice)
    shapes = [((2, 3, 4, 16), s) for s in ((192, 64, 16, 1), (192, 16, 48, 1), (64, 128, 16, 1), (16, 32, 96, 1), (500, 100, 17, 1), (1024, 64, 16, 1))]
    shapes += [((1, 3, 4, 16), (0, 64, 16, 1)), ((2, 1, 1, 16), (16, 0, 0, 1)), ((1, 1, 1, 16), (5, 5, 5, 1)), ((0, 3, 4, 16), (0, 0, 0, 1))]
    for shape, stride in shapes:
        assert not fp4._overlaps(memory.as_strided(shape, stride)), stride
    for shape, stride in (((2, 3, 4, 16), (191, 64, 16, 1)), ((2, 3, 4, 16), (192, 63, 16, 1)), ((2, 3, 4, 16), (192, 64, 15, 1)), ((2, 3, 4, 16), (64, 64, 16, 1)),
                          ((2, 3, 4, 16), (0, 64, 16, 1)), ((5, 1, 1, 16), (8, 0, 0, 1)), ((2, 3, 4, 16), (16, 64, 16, 1))):
        t = memory.as_strided(shape, stride)
        assert fp4._overlaps(t), stride
        places = torch.arange(n).as_strided(shape, stride).flatten()
        assert len(places.unique()) < len(places)
