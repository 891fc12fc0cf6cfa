"""The 4-bit operators against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import llmini_b200 as b2
from tests import fp4_plain as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def module():
    return b2.Nvfp4LinearModule()


def activations(rng, rows, cols, dtype):
    """Values with outlier columns, blocks of zeros, and many that lie exactly between two codes."""
    x = rng.standard_normal((rows, cols))
    x[:, rng.random(cols) < 0.02] *= 30
    # multiples of the row maximum that are borders of the E2M1 grid times a power of two
    ties = rng.random((rows, cols)) < 0.2
    top = np.exp2(np.floor(np.log2(np.abs(x).max(1, keepdims=True))))
    x = np.where(ties, top * rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], (rows, cols)) * np.exp2(rng.integers(-6, 1, (rows, cols))) / 8, x)
    if cols > 40:
        x[:, 16:32] = 0
    return torch.from_numpy(x).float().to(TYPES[dtype])


def check_operand(out, x64, whole=False):
    codes, s, g = plain.quantise(x64, whole)
    rows, k = codes.shape
    assert (out.rows, out.k) == (rows, k)
    got_g = out.scale.cpu().numpy().astype(np.float64)
    np.testing.assert_array_equal(got_g, g[:1] if whole else g)
    got_s, padding = plain.untiled(out.scales.cpu().numpy(), rows, k // 16)
    np.testing.assert_array_equal(got_s, s)
    assert not padding.any()
    got = plain.unpack(out.bytes.cpu().numpy(), k)
    # a code of zero may have either sign
    np.testing.assert_array_equal(np.where(got == 8, 0, got), np.where(codes == 8, 0, codes))


SHAPES = [(1, 16), (1, 1), (7, 17), (33, 1000), (130, 2048), (5, 2050), (129, 1600), (3, 8208), (2, 33000), (300, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_rows(module, rows, cols, dtype):
    x = activations(np.random.default_rng(rows * 7 + cols), rows, cols, dtype)
    out = b2.Nvfp4Operand.empty(rows, cols)
    out.scales.fill_(0x7f)   # padding behind the blocks of a row is written
    module.quantize_rows(x.cuda(), out)
    check_operand(out, plain.to_double(x))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 1), (1, 130), (17, 7), (777, 100), (128, 128), (300, 1600), (1000, 33), (40, 2050)])
def test_quantize_columns(module, rows, cols, dtype):
    x = activations(np.random.default_rng(rows * 5 + cols), rows, cols, dtype)
    out = b2.Nvfp4Operand.empty(cols, rows, per_row=False)
    out.scales.fill_(0x7f)
    module.quantize_columns(x.cuda(), out, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    check_operand(out, plain.to_double(x).T, whole=True)


@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (1, 3), (4, 4), (8, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_views(module, offset, pad, dtype):
    """Rows with gaps and starts on every kind of boundary."""
    rows, cols = 70, 200
    x = activations(np.random.default_rng(3), rows, cols, dtype)
    memory = torch.full((rows * (cols + pad) + offset,), float("nan"), dtype=x.dtype, device="cuda")
    view = memory[offset:].view(rows, cols + pad)[:, :cols]
    view.copy_(x)
    out = b2.Nvfp4Operand.empty(rows, cols)
    module.quantize_rows(view, out)
    check_operand(out, plain.to_double(x))
    out = b2.Nvfp4Operand.empty(cols, rows, per_row=False)
    module.quantize_columns(view, out, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    check_operand(out, plain.to_double(x).T, whole=True)


def test_rows_at_the_ends_of_the_range(module):
    """Rows of zeros, of the type's smallest and largest values, and rows that are not finite."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 70)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(2.0 ** -126)
    x[2] = np.float32(2.0 ** -149)
    x[3] *= np.float32(2.0 ** 125)
    x[4] = np.finfo(np.float32).max
    x[5, 3] = np.inf
    x[6, 69] = np.nan
    x[7, 16:32] = -np.inf
    x[8] *= np.float32(2.0 ** -101)
    x[9] = -0.0
    x[10, 1:] *= np.float32(2.0 ** -20)
    out = b2.Nvfp4Operand.empty(12, 70)
    module.quantize_rows(torch.from_numpy(x).cuda(), out)
    check_operand(out, x)
    columns = b2.Nvfp4Operand.empty(70, 12, per_row=False)
    module.quantize_columns(torch.from_numpy(x).cuda(), columns, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    assert torch.isnan(columns.scale).all() and not columns.bytes[:, :8].any()
    tame = x[[0, 1, 2, 8, 9]]
    columns = b2.Nvfp4Operand.empty(70, 5, per_row=False)
    module.quantize_columns(torch.from_numpy(tame).cuda(), columns, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    check_operand(columns, tame.T, whole=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,whole", [(1, 1, False), (7, 100, False), (130, 1600, True), (3, 5000, False)])
def test_decode_gives_the_values_that_codes_stand_for(module, rows, cols, whole, dtype):
    rng = np.random.default_rng(rows)
    k = -(-cols // 16) * 16
    v, packed, s, g = plain.random_operand(rng, rows, k, not whole, -(-k // 32) * 16)
    o = b2.Nvfp4Operand(torch.from_numpy(packed).cuda(), torch.from_numpy(plain.tiled(s)).cuda(), torch.from_numpy(g).cuda(), rows, k)
    out = torch.full((rows, cols + 3), -7.0, dtype=TYPES[dtype], device="cuda")
    module.decode(o, out[:, :cols])
    got, want = plain.to_double(out), v[:, :cols]
    assert (got[:, cols:] == -7).all()
    # a product in FP32 and one rounding to the type (exact where g is a power of two and the value in range)
    bound = np.abs(want) * (2.0 ** -24 + plain.half_step(TYPES[dtype])) * 1.001 + (2.0 ** -25 if dtype == "f16" else 0)
    assert (np.abs(got[:, :cols] - want) <= bound).all()


@pytest.mark.parametrize("layout", [b2.SCALES_CSF, b2.SCALES_RAW, b2.SCALES_SM100])
def test_decode_reads_the_optimizers_weights(module, layout):
    rows, k = 130, 384
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((rows, k)).astype(np.float32) * 0.02).cuda()
    raw = b2.Nvfp4Tensor.empty(rows, k, b2.SCALES_RAW)
    b2.Nvfp4QuantModule().fp32_to_nvfp4_four_six(x, x.abs().max().reshape(1), raw.bytes, raw.scales, raw.global_scale, rows * k // 16, b2.SCALES_RAW)
    s = raw.scales.cpu().numpy().reshape(rows, -1)
    t = raw
    if layout == b2.SCALES_CSF:
        t = b2.Nvfp4Tensor(raw.bytes, torch.from_numpy(b2.csf_encode_host(s.reshape(-1), rows, k)).cuda(), raw.global_scale, rows, k, layout)
    elif layout == b2.SCALES_SM100:
        t = b2.Nvfp4Tensor(raw.bytes, b2.scales_to_sm100(raw.scales, b2.SCALES_RAW, rows, k), raw.global_scale, rows, k, layout)
    out = torch.empty(rows, k, device="cuda")
    module.decode(t, out)
    want = plain.values(plain.unpack(raw.bytes.cpu().numpy().reshape(rows, -1), k), s, raw.global_scale.item())
    assert (np.abs(plain.to_double(out) - want) <= np.abs(want) * 2.0 ** -24).all()
    # the quantiser's own error: half a step of the code grid (1, of values up to 6), and what saturates of a block scale rounded
    # down by 2^-4
    step = np.repeat(plain.e4m3_grid()[s] * raw.global_scale.item(), 16, 1)
    assert (np.abs(plain.to_double(out) - plain.to_double(x)) <= 1.001 * step).all()


# ---- the product ------------------------------------------------------------------------------------------------------------
def operand(rng, rows, k, per_row, spare=0):
    """(values, Nvfp4Operand) with `spare` bytes behind every row, which are not the product's to read."""
    v, packed, s, g = plain.random_operand(rng, rows, k, per_row, -(-k // 32) * 16 + spare)
    packed[:, k // 2:] = 0x77
    t = plain.tiled(s)
    o = b2.Nvfp4Operand(torch.from_numpy(packed).cuda(), torch.from_numpy(t).cuda(), torch.from_numpy(g).cuda(), rows, k)
    return v, o


def product_bound(a, b, want, dtype):
    """FP32 sums: every addition of a product is off by at most 2^-23 of what has been added up by then (a truncated sum), scaling
    and bias by 2^-24 each; then half a step of the type."""
    terms = np.abs(a) @ np.abs(b).T
    return terms * (a.shape[1] * 2.0 ** -23 + 2.0 ** -22) + np.abs(want) * (2.0 ** -22 + plain.half_step(dtype)) + (2.0 ** -25 if dtype == torch.float16 else 0)


PRODUCTS = [(1, 1, 16), (1, 4800, 1600), (3, 40, 48), (16, 128, 256), (24, 1600, 6400), (33, 257, 64), (64, 1000, 320), (65, 300, 96), (127, 129, 784),
            (128, 128, 64), (129, 127, 1616), (200, 1000, 512), (257, 511, 1040), (777, 1600, 1600), (1000, 2304, 768), (300, 5025, 160),
            (2048, 2304, 768), (2100, 4000, 400)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(module, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, oa = operand(rng, m, k, True)
    b, ob = operand(rng, n, k, False, 16)
    want = a @ b.T
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        module.matmul(oa, ob, out)
        assert module.status() == 0
        err = np.abs(plain.to_double(out) - want)
        assert (err <= product_bound(a, b, want, dtype)).all(), (dtype, np.argwhere(~(err <= product_bound(a, b, want, dtype)))[:5])


@pytest.mark.parametrize("m,n,k", [(5, 70, 64), (140, 300, 272), (600, 1000, 512), (1100, 523, 144), (1100, 790, 64), (40, 67, 48), (130, 1, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (0, 3), (8, 8), (5, 1)])
def test_matmul_epilogue(module, m, n, k, dtype, offset, pad):
    """Scales for rows of both sides, a bias, rows of c with gaps and starts on every boundary: nothing else of c's memory changes."""
    rng = np.random.default_rng(m * n)
    a, oa = operand(rng, m, k, True)
    b, ob = operand(rng, n, k, True)
    a, b = a / 64, b / 64
    oa.scale /= 64
    ob.scale /= 64
    bias = rng.standard_normal(n).astype(np.float32)
    memory = torch.full((offset + m * (n + pad) + 64,), -3.0, dtype=TYPES[dtype], device="cuda")
    c = memory[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n]
    module.matmul(oa, ob, c, bias=torch.from_numpy(bias).cuda())
    want = a @ b.T + bias.astype(np.float64)
    assert (np.abs(plain.to_double(c) - want) <= product_bound(a, b, want, TYPES[dtype]) + np.abs(bias) * 2.0 ** -22).all()
    c.fill_(-3.0)
    assert (memory == -3.0).all()


# rows of c on no boundary in the kernels of both tile shapes; last units of 1, 64, 67, 71, 72, 73, 127 and 128 columns
ODD_ROWS = [(64, 65), (129, 127), (300, 1031), (161, 200), (257, 455), (33, 521), (1100, 2643), (2049, 2631), (700, 4168), (1000, 4169), (2000, 2751), (2016, 2689)]


@pytest.mark.parametrize("m,n", ODD_ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (2, 3), (4, 2), (7, 5), (3, 12)])
def test_matmul_into_odd_rows(module, m, n, dtype, offset, pad):
    """Every value of c, in rows that are 0 .. 7 places off a boundary, and nothing between or around them; the same bits twice."""
    rng = np.random.default_rng(m + n)
    k = 336 if m < 400 else 80
    a, oa = operand(rng, m, k, True)
    b, ob = operand(rng, n, k, False)
    bias = rng.standard_normal(n).astype(np.float32)
    a, oa.scale = a / 64, oa.scale.div_(64)
    outs = []
    for _ in range(2):
        memory = torch.full((offset + m * (n + pad) + 64,), -3.0, dtype=TYPES[dtype], device="cuda")
        c = memory[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n]
        module.matmul(oa, ob, c, bias=torch.from_numpy(bias).cuda())
        assert module.status() == 0
        outs.append(c.clone())
        c.fill_(-3.0)
        assert (memory == -3.0).all()
    want = a @ b.T + bias.astype(np.float64)
    bound = product_bound(a, b, want, TYPES[dtype]) + np.abs(bias) * 2.0 ** -22
    wrong = ~(np.abs(plain.to_double(outs[0]) - want) <= bound)
    assert not wrong.any(), np.argwhere(wrong)[:5]
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("m,n,k", [(5, 70, 64), (140, 300, 272), (600, 1000, 512), (1100, 523, 144), (1100, 788, 64)])
@pytest.mark.parametrize("pad", [0, 1])
def test_matmul_accumulates(module, m, n, k, pad):
    rng = np.random.default_rng(m + 1)
    a, oa = operand(rng, m, k, False)
    b, ob = operand(rng, n, k, False)
    start = rng.standard_normal((m, n + pad)).astype(np.float32)
    c = torch.from_numpy(start).cuda()
    module.matmul(oa, ob, c[:, :n], accumulate=True)
    want = a @ b.T + start[:, :n]
    assert (np.abs(plain.to_double(c)[:, :n] - want) <= product_bound(a, b, want, torch.float32) + np.abs(start[:, :n]) * 2.0 ** -22).all()
    assert (plain.to_double(c)[:, n:] == start[:, n:]).all()


def test_matmul_keeps_rows_apart(module):
    """A row that is not finite makes its own results NaN and no others; scales behind the last row of an operand do not matter."""
    rng = np.random.default_rng(9)
    for m, n in ((40, 300), (300, 500)):
        a, oa = operand(rng, m, 160, True)
        b, ob = operand(rng, n, 160, False)
        for o, rows in ((oa, m), (ob, n)):
            full = o.scales.view(-(-rows // 128), 3, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, 12).clone()
            full[rows:] = 0x7f
            o.scales.copy_(full.view(-1, 4, 32, 3, 4).permute(0, 3, 2, 1, 4).reshape(-1))
        oa.scale[7] = float("nan")
        out = torch.empty(m, n, device="cuda")
        module.matmul(oa, ob, out)
        want = a @ b.T
        bad = np.arange(m) == 7
        got = plain.to_double(out)
        assert np.isnan(got[bad]).all()
        assert (np.abs(got - want)[~bad] <= product_bound(a, b, want, torch.float32)[~bad]).all()


def test_matmul_does_not_depend_on_the_launch(module):
    """The same bits again, and on another stream."""
    rng = np.random.default_rng(2)
    for m, n, k in ((1, 4800, 1600), (24, 1600, 6400), (600, 1000, 512), (2100, 4000, 400)):
        _, oa = operand(rng, m, k, True)
        _, ob = operand(rng, n, k, False)
        outs = [torch.empty(m, n, device="cuda") for _ in range(3)]
        module.matmul(oa, ob, outs[0])
        module.matmul(oa, ob, outs[1])
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            module.matmul(oa, ob, outs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- the linear layer ---------------------------------------------------------------------------------------------------------
def rounded(x, whole=False):
    codes, s, g = plain.quantise(x, whole)
    return plain.values(codes, s, g)[:, : x.shape[1]]


def within(got, a, b, dtype, extra=0.0):
    """got = a b^T (+ extra) to the product's bound"""
    want = a @ b.T + extra
    assert (np.abs(plain.to_double(got) - want) <= product_bound(a, b, want, dtype) + np.abs(extra) * 2.0 ** -22).all()


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 64, 40), (1, 1600, 4800), (7, 96, 33), (24, 6400, 1600), (200, 768, 1000), (1030, 160, 300)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_linear_forward(module, tokens, inputs, outputs, dtype):
    rng = np.random.default_rng(tokens + outputs)
    x = activations(rng, tokens, inputs, dtype) / 64
    w, ow = operand(rng, outputs, inputs, False)
    bias = rng.standard_normal(outputs).astype(np.float32)
    out = torch.empty(tokens, outputs, dtype=TYPES[dtype], device="cuda")
    module.linear_forward(x.cuda(), ow, out, b2.Nvfp4LinearScratch(tokens, inputs, outputs), bias=torch.from_numpy(bias).cuda())
    within(out, rounded(plain.to_double(x)), w, TYPES[dtype], bias.astype(np.float64))


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 16, 16), (7, 100, 33), (130, 272, 496), (777, 160, 320), (300, 1000, 770)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_linear_backward(module, tokens, inputs, outputs, dtype):
    rng = np.random.default_rng(tokens + outputs)
    x, grad = activations(rng, tokens, inputs, dtype), activations(rng, tokens, outputs, dtype) / 64
    x64, grad64 = plain.to_double(x), plain.to_double(grad)
    wt, owt = operand(rng, inputs, -(-outputs // 16) * 16, False)
    args = dict(device="cuda", dtype=TYPES[dtype])
    scratch = b2.Nvfp4LinearScratch(tokens, inputs, outputs, backward=True)
    k = wt.shape[1]
    gr = np.zeros((tokens, k))
    gr[:, :outputs] = rounded(grad64)
    gc, xc = rounded(grad64.T, True), rounded(x64.T, True)
    for want_x, want_w, accumulate in ((True, True, False), (True, False, False), (False, True, False), (True, True, True)):
        start = rng.standard_normal((outputs, inputs)).astype(np.float32)
        grad_x = torch.full((tokens, inputs), -3.0, **args) if want_x else None
        grad_w = torch.from_numpy(start).cuda() if want_w else None
        module.linear_backward(grad.cuda(), x.cuda(), owt, grad_x, grad_w, scratch, accumulate=accumulate)
        if want_x:
            within(grad_x, gr, wt, TYPES[dtype])
        if want_w:
            within(grad_w, gc, xc, torch.float32, start.astype(np.float64) if accumulate else 0.0)


@pytest.mark.parametrize("tokens,inputs,outputs", [(20, 48, 9000), (3, 64, 33008), (5000, 48, 64), (4096, 80, 2064), (4097, 1600, 32), (600, 5000, 16)])
@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("gap", [0, 5])
def test_linear_backward_is_its_parts(module, tokens, inputs, outputs, types, gap):
    """Bit for bit what the quantisers and the product give one by one: rows of every length, many and few of them, with gaps."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    x = torch.randn(tokens, inputs + gap, device="cuda", generator=gen).to(TYPES[types[0]])[:, :inputs]
    grad = torch.randn(tokens, outputs + gap, device="cuda", generator=gen).to(TYPES[types[1]])[:, :outputs]
    x[tokens // 2, inputs // 3] = 100.0       # the maxima, each in one place
    grad[tokens - 1, outputs - 1] = -70.0
    wt = b2.Nvfp4Operand.empty(inputs, outputs)
    module.quantize_rows(torch.randn(inputs, outputs, device="cuda", generator=gen), wt)
    got = torch.empty(tokens, inputs, device="cuda"), torch.empty(outputs, inputs, device="cuda")
    module.linear_backward(grad, x, wt, *got, b2.Nvfp4LinearScratch(tokens, inputs, outputs, backward=True))
    maxima = torch.empty(b2.NVFP4_MAXIMA, device="cuda")
    rows, columns, x_columns = (b2.Nvfp4Operand.empty(r, k, per_row=p) for r, k, p in ((tokens, outputs, True), (outputs, tokens, False), (inputs, tokens, False)))
    module.quantize_rows(grad, rows)
    module.quantize_columns(grad, columns, maxima)
    module.quantize_columns(x, x_columns, maxima)
    assert x_columns.scale.item() == 2.0 ** (6 - 10) and columns.scale.item() == 2.0 ** (6 - 10)
    want = torch.empty_like(got[0]), torch.empty_like(got[1])
    module.matmul(rows, wt, want[0])
    module.matmul(columns, x_columns, want[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_linear_gradients_are_those_of_the_layer(module):
    """Against differences of sum(grad * (x W^T)): the gradients are off by what the rounding of their operands to 4 bits is.  A
    block's values are off by half a step of E2M1, 1/2 of values 4 .. 6 down to 1/4 of those below 2, in units of max / 6; normal
    values by 0.10 of their size together.  Three sigma above the two operands' 0.14, for sums over 256 or more."""
    rng = np.random.default_rng(4)
    tokens, inputs, outputs = 256, 320, 384
    x, grad, w = (torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda() for s in ((tokens, inputs), (tokens, outputs), (outputs, inputs)))
    owt = b2.Nvfp4Operand.empty(inputs, outputs, per_row=False)
    module.quantize_columns(w, owt, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    grad_x, grad_w = torch.empty_like(x), torch.empty_like(w)
    module.linear_backward(grad, x, owt, grad_x, grad_w, b2.Nvfp4LinearScratch(tokens, inputs, outputs, backward=True))
    loss = lambda x, w: (grad.double() * (x.double() @ w.double().T)).sum()
    for got, at, other in ((grad_x, x, 0), (grad_w, w, 1)):
        for _ in range(4):
            d = torch.randn(at.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(_)) * 0.5
            ends = [loss(*((at + s * d, w) if other == 0 else (x, at + s * d))) for s in (1, -1)]
            slope = ((ends[0] - ends[1]) / 2).item()
            scale = (torch.linalg.vector_norm((grad.double() @ w.double() if other == 0 else grad.double().T @ x.double())) * torch.linalg.vector_norm(d.double()) / d.numel() ** 0.5).item()
            assert abs((got.double() * d.double()).sum().item() - slope) <= 3 * 0.15 * scale


def test_linear_backward_of_no_tokens(module):
    w = torch.full((40, 24), 5.0, device="cuda")
    s = b2.Nvfp4LinearScratch(0, 24, 40, backward=True)
    x, grad = torch.empty(0, 24, device="cuda"), torch.empty(0, 40, device="cuda")
    module.linear_backward(grad, x, None, None, w, s, accumulate=True)
    assert (w == 5).all()
    module.linear_backward(grad, x, None, None, w, s)
    assert (w == 0).all()


def test_a_training_step_together(module):
    """The optimizer's weights through the layer and back: a plan that leaves its scales in SCALES_SM100, forward, backward from
    the quantised transpose of the masters, the weight gradient added up over two micro-batches into the plan's gradient buffer,
    and the next optimizer step on it; then the same as a captured graph."""
    from tests.gpu_util import host
    rng = np.random.default_rng(8)
    tokens, inputs, outputs = 96, 256, 384
    slot = b2.MuonSlot.allocate(outputs, inputs, scale_layout=b2.SCALES_SM100)
    master = torch.from_numpy(rng.standard_normal((outputs, inputs)).astype(np.float32) * 0.02).cuda()
    slot.z_master.copy_(master.view_as(slot.z_master))
    slot.x_master.copy_(master.view_as(slot.x_master))
    slot.grad.copy_(torch.from_numpy(rng.standard_normal((outputs, inputs)).astype(np.float32) * 1e-3).view_as(slot.grad))
    plan = b2.MuonPlan([(outputs, inputs)], scale_layout=b2.SCALES_SM100)
    opt, table, step = b2.OptimizerModule(), b2.slot_table([slot]), b2.MuonMegaUpdateArgs(learning_rate=0.02)
    opt.muon_mega_update(plan, table, step)
    weight = b2.Nvfp4Operand(slot.bytes.view(outputs, inputs // 2), slot.scales, slot.global_scale, outputs, inputs)
    weight_t = b2.Nvfp4Operand.empty(inputs, outputs, per_row=False)
    maxima = torch.empty(b2.NVFP4_MAXIMA, device="cuda")
    x = [torch.randn(tokens, inputs, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    grad = [torch.randn(tokens, outputs, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    y, grad_x = torch.empty(tokens, outputs, device="cuda", dtype=torch.bfloat16), torch.empty(tokens, inputs, device="cuda", dtype=torch.bfloat16)
    forward, backward = b2.Nvfp4LinearScratch(tokens, inputs, outputs), b2.Nvfp4LinearScratch(tokens, inputs, outputs, backward=True)
    grad_w = slot.grad.view(outputs, inputs)

    def layer():
        module.quantize_columns(slot.x_master.view(outputs, inputs), weight_t, maxima)
        for i in range(2):
            module.linear_forward(x[i], weight, y, forward)
            module.linear_backward(grad[i], x[i], weight_t, grad_x, grad_w, backward, accumulate=i > 0)

    layer()
    torch.cuda.synchronize()
    w64 = plain.values(plain.unpack(host(weight.bytes), inputs), plain.untiled(host(slot.scales), outputs, inputs // 16)[0], slot.global_scale.item())
    wt64 = rounded(plain.to_double(slot.x_master.view(outputs, inputs)).T, True)
    within(y, rounded(plain.to_double(x[1])), w64, torch.bfloat16)
    within(grad_x, rounded(plain.to_double(grad[1])), wt64, torch.bfloat16)
    sides = [(rounded(plain.to_double(grad[i]).T, True), rounded(plain.to_double(x[i]).T, True)) for i in range(2)]
    want = sum(g @ xx.T for g, xx in sides)
    assert (np.abs(plain.to_double(grad_w) - want) <= sum(product_bound(g, xx, want, torch.float32) for g, xx in sides)).all()
    eager = [t.clone() for t in (y, grad_x, grad_w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for t in (y, grad_x, grad_w):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, (y, grad_x, grad_w)))
    for t in x + grad:
        t.mul_(2.0)   # the graph reads its inputs anew; scales are powers of two, so everything is exactly twice (four times) as large
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, 2 * eager[0]) and torch.equal(grad_x, 2 * eager[1]) and torch.equal(grad_w, 4 * eager[2])
    before = slot.x_master.clone()
    opt.muon_mega_update(plan, table, step)
    assert plan.status() == 0 and module.status() == 0
    assert torch.isfinite(slot.x_master).all() and not torch.equal(before, slot.x_master)
    plan.close()


# ---- the cache ------------------------------------------------------------------------------------------------------------------
def cache_values(side, dim):
    """[pages, page_size, heads, dim] values of one side of a cache, in 64 bits."""
    codes, s, e = (t.cpu().numpy() for t in side)
    n = int(np.prod(e.shape))
    g = np.where(e.reshape(-1) == 255, np.nan, np.exp2(e.reshape(-1).astype(np.float64) - 127))
    return plain.values(plain.unpack(codes.reshape(n, -1), dim), s.reshape(n, -1), g).reshape(*e.shape, dim)


@pytest.mark.parametrize("heads,dim,value_dim,page", [(1, 16, 16, 1), (4, 64, 64, 16), (25, 64, 64, 32), (3, 96, 128, 7), (2, 576, 512, 64), (1, 1024, 16, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_cache(module, heads, dim, value_dim, page, dtype):
    """Tokens written to scattered slots out of a fused projection, some left out; sequences of every length read back."""
    rng = np.random.default_rng(dim + page)
    pages, sequences, width = 40, 6, 6
    longest = width * page + 3
    cache = b2.Nvfp4PagedCache.empty(pages, page, heads, dim, value_dim)
    for side in (cache.key, cache.value):
        for t in side:
            t.random_(0, 120)
    before = [t.clone() for side in (cache.key, cache.value) for t in side]
    tokens = min(pages * page, 50)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    leave = [0, tokens // 2] if tokens > 4 else []
    for i, bad in zip(leave, (-1, pages * page)):
        slots[i] = bad
    fused = activations(rng, tokens, heads * (dim + value_dim) + 8, dtype).cuda()
    if tokens > 3:
        fused[3, 1] = float("inf")   # one vector
    key = fused[:, : heads * dim].unflatten(1, (heads, dim))
    value = fused[:, heads * dim: heads * (dim + value_dim)].unflatten(1, (heads, value_dim))
    module.cache_write(cache, torch.from_numpy(slots).cuda(), key, value)
    kept = np.ones(pages * page, bool)
    for i, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            kept[slot] = False
    for j, (side, new, d) in enumerate(((cache.key, key, dim), (cache.value, value, value_dim))):
        codes, s, g = plain.quantise(plain.to_double(new).reshape(-1, d))
        got = cache_values(side, d).reshape(pages * page, heads, d)
        want = plain.values(codes, s, g).reshape(tokens, heads, d)
        for i, slot in enumerate(slots):
            if 0 <= slot < pages * page:
                np.testing.assert_array_equal(got[slot], want[i])
        for t, old in zip(side, before[3 * j: 3 * j + 3]):   # slots that no token went to
            assert torch.equal(t.view(pages * page, -1)[torch.from_numpy(kept)], old.view(pages * page, -1)[torch.from_numpy(kept)])
    # the old slots of random bytes hold numbers too
    table = rng.integers(0, pages, (sequences, width)).astype(np.int32)
    table[1, 0], table[2, width - 1] = -1, pages
    lengths = np.array([width * page, 1, width * page + 2, 0, -5, page], np.int32)
    outs = [torch.full((sequences, longest, heads, d + 8), -3.0, dtype=TYPES[dtype], device="cuda")[..., :d] for d in (dim, value_dim)]
    module.cache_read(cache, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(), *outs)
    for side, out, d in ((cache.key, outs[0], dim), (cache.value, outs[1], value_dim)):
        v = cache_values(side, d)
        got = plain.to_double(out)
        for b in range(sequences):
            n = int(np.clip(lengths[b], 0, width * page))
            for t in range(n):
                p = table[b, t // page]
                want = v[p, t % page] if 0 <= p < pages else np.full((heads, d), np.nan)
                want = torch.from_numpy(want).to(TYPES[dtype]).double().numpy()
                np.testing.assert_array_equal(got[b, t], want)
            assert (got[b, n:] == -3).all()
        assert (out._base[..., d:] == -3).all()


def test_cache_beyond_32_bits(module):
    """A cache of more than 2^32 bytes of codes: the last page's, and the same tokens' near the start."""
    pages, page, heads, dim = 33000, 64, 16, 256
    codes = torch.empty(pages, page, heads, dim // 2, dtype=torch.uint8, device="cuda")
    cache = b2.Nvfp4PagedCache((codes, torch.empty(pages, page, heads, dim // 16, dtype=torch.uint8, device="cuda"),
                                torch.empty(pages, page, heads, dtype=torch.uint8, device="cuda")))
    assert codes.numel() > 1 << 32
    key = torch.randn(2 * page, heads, dim, device="cuda", dtype=torch.bfloat16)
    place = torch.arange(page, device="cuda")
    module.cache_write(cache, torch.cat([place + page, place + (pages - 1) * page]), key)
    out = torch.zeros(2, page, heads, dim, device="cuda", dtype=torch.bfloat16)
    module.cache_read(cache, torch.tensor([[1], [pages - 1]], dtype=torch.int32, device="cuda"), torch.full((2,), page, dtype=torch.int32, device="cuda"), out)
    want = rounded(plain.to_double(key).reshape(-1, dim)).reshape(2, page, heads, dim)
    np.testing.assert_array_equal(plain.to_double(out), torch.from_numpy(want).bfloat16().double().numpy())


def test_tensors_beyond_32_bits(module):
    """More than 2^32 values: the last rows come out as they do by themselves."""
    rows, cols = 66000, 65600
    x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[:256].normal_()
    for r in range(256, rows, 256):
        x[r:r + 256] = x[:min(256, rows - r)]
    x[-1].mul_(3.0)
    big = b2.Nvfp4Operand.empty(rows, cols)
    module.quantize_rows(x, big)
    tail = b2.Nvfp4Operand.empty(5, cols)
    module.quantize_rows(x[-5:].clone(), tail)
    assert torch.equal(big.bytes[-5:, : cols // 2], tail.bytes[:, : cols // 2]) and torch.equal(big.scale[-5:], tail.scale)
    back, part = torch.empty_like(x), torch.empty(5, cols, device="cuda", dtype=torch.bfloat16)
    module.decode(big, back)
    module.decode(tail, part)
    assert torch.equal(back[-5:], part)
    del back, big
    columns = b2.Nvfp4Operand.empty(cols, rows, per_row=False)
    module.quantize_columns(x, columns, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    some = b2.Nvfp4Operand.empty(16, rows, per_row=False)
    module.quantize_columns(torch.cat([x[:, -15:], torch.full((rows, 1), x.abs().max().item(), device="cuda", dtype=x.dtype)], 1), some,
                            torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
    assert torch.equal(columns.bytes[-15:, : rows // 2], some.bytes[:15, : rows // 2]) and torch.equal(columns.scale, some.scale)
    del columns, some
    rng = np.random.default_rng(0)
    a, oa = operand(rng, rows, 64, True)
    b, ob = operand(rng, cols, 64, False)
    module.matmul(oa, ob, x)
    want = a[-300:] @ b[-300:].T
    assert (np.abs(plain.to_double(x[-300:, -300:]) - want) <= product_bound(a[-300:], b[-300:], want, torch.bfloat16)).all()


# ---- what is refused --------------------------------------------------------------------------------------------------------------
def test_refusals(module):
    f = lambda *s, dtype=torch.float32, device="cuda": torch.zeros(*s, dtype=dtype, device=device)
    o = b2.Nvfp4Operand.empty
    with pytest.raises(ValueError):
        module.quantize_rows(f(4, 32, device="cpu"), o(4, 32))
    with pytest.raises(ValueError):
        module.quantize_rows(f(4, 32, dtype=torch.float64), o(4, 32))
    with pytest.raises(ValueError):
        module.quantize_rows(f(32, 4).T, o(4, 32))
    with pytest.raises(ValueError):
        module.quantize_rows(f(1, 32).expand(4, 32), o(4, 32))
    for x, out in ((f(4, 32), o(5, 32)), (f(4, 32), o(4, 48)), (f(4, 32), o(4, 32, per_row=False))):
        with pytest.raises(b2.B2Error):
            module.quantize_rows(x, out)
    with pytest.raises(ValueError):
        module.quantize_columns(f(4, 32), o(32, 4, per_row=False), f(10))
    with pytest.raises(b2.B2Error):
        module.quantize_columns(f(4, 32), o(4, 32, per_row=False), f(1024))
    for a, b, c in ((o(4, 32), o(5, 48), f(4, 5)), (o(4, 32), o(5, 32), f(5, 4)), (o(4, 32), o(5, 32), f(4, 6))):
        with pytest.raises(b2.B2Error):
            module.matmul(a, b, c)
    with pytest.raises(b2.B2Error):
        module.matmul(o(4, 32), o(5, 32), f(4, 5, dtype=torch.bfloat16), accumulate=True)
    with pytest.raises(ValueError):
        module.matmul(o(4, 32), o(5, 32), f(4, 5), bias=f(4))
    with pytest.raises(ValueError):
        module.linear_forward(f(4, 32), o(5, 32), f(4, 5), b2.Nvfp4LinearScratch(4, 32, 5, backward=True))
    with pytest.raises(ValueError):
        b2.Nvfp4Operand(f(4, 8, dtype=torch.uint8), f(512, dtype=torch.uint8), f(4), 4, 16)   # rows on 8-byte boundaries
    with pytest.raises(ValueError):
        b2.Nvfp4Operand(f(4, 16, dtype=torch.uint8), f(100, dtype=torch.uint8), f(4), 4, 32)  # too few scales
    cache = b2.Nvfp4PagedCache.empty(4, 2, 3, 32)
    slots = torch.zeros(5, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        module.cache_write(cache, slots, f(5, 3, 32))
    with pytest.raises(ValueError):
        module.cache_write(cache, slots, f(5, 3, 48), f(5, 3, 48))
    with pytest.raises(ValueError):
        module.cache_write(cache, slots.int(), f(5, 3, 32), f(5, 3, 32))
    with pytest.raises(ValueError):
        module.cache_write(cache, slots, f(5, 3, 32), f(5, 3, 32, dtype=torch.bfloat16))
    with pytest.raises(b2.B2Error):
        b2.Nvfp4LinearModule().cache_write(b2.Nvfp4PagedCache.empty(4, 2, 3, 1040), slots, f(5, 3, 1040), f(5, 3, 1040))
    # nothing to do is no error
    module.quantize_rows(f(0, 32), o(0, 32))
    module.matmul(o(0, 32), o(5, 32), f(0, 5))
    module.matmul(o(4, 32), o(0, 32, per_row=False), f(4, 0))
    module.cache_write(cache, slots[:0], f(0, 3, 32), f(0, 3, 32))


def test_fields_may_be_replaced(module):
    """Calls see the tensors that an operand and a cache have now, not those that they were made with."""
    x = torch.randn(40, 64, device="cuda")
    o = b2.Nvfp4Operand.empty(40, 64)
    first = o.bytes
    first.fill_(0x55)
    o.bytes, o.scale = torch.zeros(40, 48, dtype=torch.uint8, device="cuda"), torch.zeros(40, device="cuda")
    module.quantize_rows(x, o)
    assert (first == 0x55).all() and o.scale.all()
    assert (o.bytes[:, 32:] == 0).all() and o.bytes.any()
    with pytest.raises(ValueError):
        o.bytes = torch.zeros(39, 32, dtype=torch.uint8, device="cuda")
    cache, other = (b2.Nvfp4PagedCache.empty(4, 8, 2, 32) for _ in range(2))
    before = cache.key
    cache.key = other.key
    key = torch.randn(3, 2, 32, device="cuda")
    module.cache_write(cache, torch.arange(3, device="cuda"), key, key)
    assert not before[0].any() and other.key[0].any() and cache.value[0].any()


def test_results_do_not_overlap(module):
    cache = b2.Nvfp4PagedCache.empty(4, 8, 2, 32)
    table, lengths = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    good = torch.zeros(3, 8, 2, 32, device="cuda")
    for bad in (good[:1].expand(3, 8, 2, 32), good[:, :1].expand(3, 8, 2, 32), good[:, :, :1].expand(3, 8, 2, 32)):
        with pytest.raises(ValueError):
            module.cache_read(cache, table, lengths, bad, good)
    # what is read may: one vector for every head and token
    one = torch.randn(1, 1, 32, device="cuda").expand(5, 2, 32)
    module.cache_write(cache, torch.arange(5, device="cuda"), one, one)
    module.cache_read(cache, table, torch.full_like(lengths, 5), good, good.clone())
    assert torch.equal(good[0, :5], good[1, :5]) and (good[0, :5] == good[0, 0, 0]).all() and good[0, 0, 0].any()


FIRST_CALLS = """
import torch, llmini_b200 as b2
m = b2.Nvfp4LinearModule()
x, w = torch.randn(%d, 160, device="cuda"), b2.Nvfp4Operand.empty(96, 160, per_row=False)
y, s, maxima = torch.empty(%d, 96, device="cuda"), b2.Nvfp4LinearScratch(%d, 160, 96), torch.empty(1024, device="cuda")
master = torch.randn(160, 96, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    m.quantize_columns(master, w, maxima)
    m.linear_forward(x, w, y, s)
graph.replay()
torch.cuda.synchronize()
first = y.clone()
m.quantize_columns(master, w, maxima)
m.linear_forward(x, w, y, s)
assert torch.equal(first, y) and y.any() and m.status() == 0
"""


@pytest.mark.parametrize("tokens", [2, 30, 300])
def test_the_first_calls_of_a_process_are_captured(tokens):
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS % (tokens, tokens, tokens)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_calls_on_two_streams(module):
    """Products of every kernel at the same time, each with its own scratch: what they give one after the other."""
    rng = np.random.default_rng(5)
    jobs = []
    for tokens, inputs, outputs in ((1, 1600, 4800), (24, 6400, 1600), (300, 768, 1000), (2100, 400, 4000)):
        _, w = operand(rng, outputs, inputs, False)
        x = torch.randn(tokens, inputs, device="cuda", dtype=torch.bfloat16)
        jobs.append((x, w, [torch.empty(tokens, outputs, device="cuda") for _ in range(3)], [b2.Nvfp4LinearScratch(tokens, inputs, outputs) for _ in range(2)]))
    for x, w, y, s in jobs:
        module.linear_forward(x, w, y[2], s[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for x, w, y, s in (jobs if i == 0 else reversed(jobs)):
                    module.linear_forward(x, w, y[i], s[i])
    torch.cuda.synchronize()
    assert module.status() == 0
    for x, w, y, s in jobs:
        assert torch.equal(y[0], y[2]) and torch.equal(y[1], y[2])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offset,spare", [(0, 0), (8, 8), (4, 4), (1, 3), (16, 0)])
def test_cache_of_vectors_on_any_boundary(module, dtype, offset, spare):
    heads, dim, tokens = 3, 48, 10
    cache = b2.Nvfp4PagedCache.empty(5, 4, heads, dim)
    memory = torch.randn(tokens, heads, offset + dim + spare, device="cuda").to(TYPES[dtype])
    key, value = memory[..., offset:offset + dim], torch.randn(tokens, heads, dim, device="cuda").to(TYPES[dtype])
    module.cache_write(cache, torch.arange(tokens, device="cuda") + 4, key, value)
    out = torch.full((1, tokens, heads, offset + dim + spare), -3.0, device="cuda", dtype=TYPES[dtype])
    other = torch.empty(1, tokens, heads, dim, device="cuda", dtype=TYPES[dtype])
    module.cache_read(cache, torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda"), torch.tensor([tokens], dtype=torch.int32, device="cuda"),
                      out[..., offset:offset + dim], other)
    for got, given in ((out[0, ..., offset:offset + dim], key), (other[0], value)):
        want = rounded(plain.to_double(given).reshape(-1, dim)).reshape(tokens, heads, dim)
        np.testing.assert_array_equal(plain.to_double(got), torch.from_numpy(want).to(TYPES[dtype]).double().numpy())
    assert (out[..., :offset] == -3).all() and (out[..., offset + dim:] == -3).all()


def test_after_a_refused_field_calls_use_what_was_there(module):
    """An operand and a cache that refused a field work on, on the memory that they still hold."""
    x = torch.randn(40, 64, device="cuda")
    o, want = b2.Nvfp4Operand.empty(40, 64), b2.Nvfp4Operand.empty(40, 64)
    module.quantize_rows(x, want)
    kept = o.bytes
    for name, bad in (("bytes", torch.zeros(39, 32, dtype=torch.uint8, device="cuda")), ("rows", 20), ("scale", torch.zeros(20, device="cuda"))):
        with pytest.raises(ValueError):
            setattr(o, name, bad)
    module.quantize_rows(x, o)
    assert o.bytes is kept and torch.equal(kept, want.bytes) and torch.equal(o.scale, want.scale) and torch.equal(o.scales, want.scales)
    with pytest.raises(ValueError):   # a bias for the rows that there are
        module.matmul(o, o, torch.empty(40, 40, device="cuda"), bias=torch.zeros(20, device="cuda"))
    more = b2.Nvfp4Operand.empty(130, 160)
    o.replace(bytes=more.bytes, scales=more.scales, scale=more.scale, rows=130, k=160)
    y = torch.randn(130, 160, device="cuda")
    module.quantize_rows(y, o)
    back = torch.empty_like(y)
    module.decode(more, back)
    assert (plain.to_double(back) == rounded(plain.to_double(y))).all()
    cache = b2.Nvfp4PagedCache.empty(4, 8, 2, 32)
    key = cache.key
    with pytest.raises(ValueError):
        cache.key = tuple(t.cpu() for t in key)
    v = torch.randn(3, 2, 32, device="cuda")
    module.cache_write(cache, torch.arange(3, device="cuda"), v, v)
    assert cache.key is key and key[0].view(32, -1)[:3].any() and torch.equal(key[0], cache.value[0])


def scales_next_to_borders(dtype, rng):
    """FP32 scales whose products with some code * s lie so close to the middle between two values of `dtype` that FP32 has that middle
    for them, below it or above, where it is the other value that is nearest."""
    products = np.array([a * b for a in (1, 3) for b in range(8, 16)], np.float64)
    bits = {torch.bfloat16: 7, torch.float16: 10}[dtype]
    found = []
    for a in products:
        middles = (2 * rng.integers(1 << bits, 2 << bits, 4000) + 1) / 2.0
        g = (middles / a).astype(np.float32)
        exact = a * g.astype(np.float64)
        near = (exact != middles) & (exact.astype(np.float32) == middles)
        even = np.floor(middles) % 2 == 0   # the second rounding would go to the even one
        found += list(g[near & ((exact > middles) == even)][:12])
    return np.array(found, np.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_decode_rounds_once(module, dtype):
    """Every code with every scale: the nearest value of the type, whatever the scale on top."""
    rng = np.random.default_rng(11)
    t = TYPES[dtype]
    near = scales_next_to_borders(torch.bfloat16 if dtype == "f32" else t, rng)
    assert len(near) > 40
    g = np.concatenate([near * np.float32(2.0) ** rng.integers(-14, 4, len(near)).astype(np.float32), [0.13489583134651184, 2.0 ** -8, 1.0 / 3, 2.0 ** 120 * 1.3,
                       2.0 ** -126 * 1.7, 2.0 ** -135 * 1.37, 2.0 ** -149, 2.0 ** -30 * 1.1], rng.random(40)]).astype(np.float32)
    rows, k = len(g), 16 * 127
    codes = np.tile(np.arange(16, dtype=np.uint8), (rows, k // 16))
    s = np.tile(np.arange(127, dtype=np.uint8), (rows, 1))
    v = plain.values(codes, s, g)
    o = b2.Nvfp4Operand(torch.from_numpy(plain.pack(codes, -(-k // 32) * 16)).cuda(), torch.from_numpy(plain.tiled(s)).cuda(), torch.from_numpy(g).cuda(), rows, k)
    out = torch.empty(rows, k, dtype=t, device="cuda")
    module.decode(o, out)
    np.testing.assert_array_equal(plain.to_double(out), plain.rounded_once(v, t))
    if dtype != "f32":   # and rounding twice is something else here
        with np.errstate(all="ignore"):
            assert (plain.rounded_once(v.astype(np.float32), t) != plain.rounded_once(v, t)).sum() > 20


# (exponent of A's scales, of B's, the codes of the block scales): the scales' product is subnormal, out of range below or above, or in
# range with one of them far out
ENDS = [(-110, -24, (0x28, 0x79)), (-60, -86, (0x28, 0x79)), (117, 13, (1, 2)), (126, -140, (0x28, 0x79)), (-110, 100, (0x28, 0x79)), (-149, 110, (0x40, 0x79)),
        (127, 127, (0x28, 0x79)), (-149, -149, (0x28, 0x79)), (-70, -79, (0x70, 0x79))]


def operand_at(rng, rows, k, per_row, exponent, s_range, zero_row):
    codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    if zero_row is not None:
        codes[zero_row] = 8 * rng.integers(0, 2, k)
    s = rng.integers(*s_range, (rows, k // 16)).astype(np.uint8)
    g = np.ldexp(rng.uniform(1, 1.9, rows if per_row else 1), exponent).astype(np.float32)
    o = b2.Nvfp4Operand(torch.from_numpy(plain.pack(codes, -(-k // 32) * 16)).cuda(), torch.from_numpy(plain.tiled(s)).cuda(), torch.from_numpy(g).cuda(), rows, k)
    return plain.values(codes, s, g), o


def check_at_the_ends(got, want, terms, k, dtype):
    got = plain.to_double(got)
    bound = terms * (k * 2.0 ** -23 + 2.0 ** -22) + np.abs(want) * (2.0 ** -22 + plain.half_step(dtype)) + {torch.float32: 2.0 ** -148, torch.bfloat16: 2.0 ** -134}[dtype]
    over = np.abs(want) + bound >= torch.finfo(dtype).max
    assert not np.isnan(got).any()
    assert (np.abs(got - want) <= bound)[~over].all()
    sure = np.abs(want) - bound > 2.0 ** 128
    assert (got[sure] == np.copysign(np.inf, want[sure])).all()


@pytest.mark.parametrize("m,n,k", [(5, 70, 64), (60, 200, 4112), (140, 300, 272), (140, 301, 272), (1100, 2100, 64), (1100, 2101, 64)])
@pytest.mark.parametrize("per_row", [(True, False), (True, True), (False, True)])
def test_products_of_scales_at_the_ends_of_the_range(module, m, n, k, per_row):
    """Results that FP32 has come out as they are, whatever the product of the two scales on top alone would be."""
    rng = np.random.default_rng(m + n)
    for ea, eb, s_range in ENDS:
        a, oa = operand_at(rng, m, k, per_row[0], ea, s_range, 3)
        b, ob = operand_at(rng, n, k, per_row[1], eb, s_range, None)
        want, terms = a @ b.T, np.abs(a) @ np.abs(b).T
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
            module.matmul(oa, ob, out)
            check_at_the_ends(out, want, terms, k, dtype)
            assert (out[3] == 0).all()
    zero = b2.Nvfp4Operand(ob.bytes, ob.scales, torch.zeros_like(ob.scale), n, k)   # the scale of a tensor of zeros
    out = torch.full((m, n), float("nan"), device="cuda")
    module.matmul(oa, zero, out)
    assert (out == 0).all()


@pytest.mark.parametrize("tokens,inputs", [(1, 256), (5, 1008), (12, 1008), (200, 256)])
def test_small_activations_times_small_weights(module, tokens, inputs):
    rng = np.random.default_rng(tokens)
    x = torch.from_numpy((rng.standard_normal((tokens, inputs)) * 2.0 ** -101).astype(np.float32))
    w, ow = operand_at(rng, 300, inputs, False, -22, (0x28, 0x79), None)
    out = torch.empty(tokens, 300, device="cuda")
    module.linear_forward(x.cuda(), ow, out, b2.Nvfp4LinearScratch(tokens, inputs, 300))
    q = rounded(plain.to_double(x))
    check_at_the_ends(out, q @ w.T, np.abs(q) @ np.abs(w).T, inputs, torch.float32)


@pytest.mark.parametrize("rows,k", [(7, 40), (33, 100), (96, 128), (127, 250), (130, 70), (256, 64)])
def test_quantisers_leave_rows_behind_the_last_one_alone(module, rows, k):
    """Of a band of 128 rows a tensor owns the scales of its own; all 64-value tiles of these are written."""
    x = torch.randn(rows, k, device="cuda")
    for columns in (False, True):
        o = b2.Nvfp4Operand.empty(rows, k, per_row=not columns)
        o.scales.fill_(0x7f)
        o.bytes.fill_(0x55)
        if columns:
            module.quantize_columns(x.T.contiguous(), o, torch.empty(b2.NVFP4_MAXIMA, device="cuda"))
        else:
            module.quantize_rows(x, o)
        bands, chunks = -(-rows // 128), -(-o.k // 64)
        all_rows, _ = plain.untiled(o.scales.cpu().numpy(), bands * 128, chunks * 4)
        assert (all_rows[rows:] == 0x7f).all() and (all_rows[:rows, o.k // 16:] == 0).all()
        assert (all_rows[:rows, :o.k // 16] < 0x7f).all() and (o.bytes[:, o.k // 2:] == 0x55).all()
        check_operand(o, plain.to_double(x), whole=columns)


@pytest.mark.parametrize("tokens,size", [(3, 96), (300, 320), (5000, 64)])
@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "bf16")])
def test_gradients_over_their_inputs(module, tokens, size, types):
    """grad_x in the place of x or of grad: both gradients are those of what lay there."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    x, grad = (torch.randn(tokens, size, device="cuda", generator=gen).to(TYPES[t]) for t in types)
    wt = b2.Nvfp4Operand.empty(size, size)
    module.quantize_rows(torch.randn(size, size, device="cuda", generator=gen), wt)
    scratch = b2.Nvfp4LinearScratch(tokens, size, size, backward=True)
    for place in (0, 1):
        want = torch.empty_like((x, grad)[place]), torch.empty(size, size, device="cuda")
        module.linear_backward(grad, x, wt, *want, scratch)
        both = [x.clone(), grad.clone()]
        got = both[place], torch.empty(size, size, device="cuda")
        module.linear_backward(both[1], both[0], wt, *got, scratch)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(both[1 - place], (x, grad)[1 - place])


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 4800, 4800), (4, 1600, 1600), (3, 768, 2304), (1, 64, 200001), (5, 1600, 100000), (12, 1600, 1600), (300, 768, 512)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_over_its_input(module, tokens, inputs, outputs, dtype):
    """y in the place of x, at its start or some rows on: what a call with a place of its own gives, time and again."""
    rng = np.random.default_rng(tokens)
    x = activations(rng, tokens, inputs, dtype).cuda()
    _, w = operand(rng, outputs, inputs, False)
    scratch, want = b2.Nvfp4LinearScratch(tokens, inputs, outputs), torch.empty(tokens, outputs, dtype=TYPES[dtype], device="cuda")
    module.linear_forward(x, w, want, scratch)
    for offset in (0, 7, (tokens - 1) * inputs):
        memory = torch.empty(offset + tokens * max(inputs, outputs), dtype=TYPES[dtype], device="cuda")
        for _ in range(10):
            memory[:tokens * inputs].view_as(x).copy_(x)
            y = memory[offset:offset + tokens * outputs].view(tokens, outputs)
            module.linear_forward(memory[:tokens * inputs].view_as(x), w, y, scratch)
            assert torch.equal(y, want)


@pytest.mark.parametrize("rows", [1, 5, 130])
def test_decode_of_csf_storage_goes_by_its_header(module, rows):
    """A header that is missing, of a smaller tensor or of no record size reads as NaN; the same scales under another shape are the same."""
    k = 256
    x = torch.randn(rows, k, device="cuda") * 0.02
    raw = b2.Nvfp4Tensor.empty(rows, k, b2.SCALES_RAW)
    b2.Nvfp4QuantModule().fp32_to_nvfp4_four_six(x, x.abs().max().reshape(1), raw.bytes, raw.scales, raw.global_scale, rows * k // 16, b2.SCALES_RAW)
    want, out = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda")
    module.decode(raw, want)
    good = torch.from_numpy(b2.csf_encode_host(raw.scales.cpu().numpy(), rows, k)).cuda()

    def read(scales, rows=rows, k=k):
        out.zero_()
        module.decode(b2.Nvfp4Tensor(raw.bytes, scales, raw.global_scale, rows, k, b2.SCALES_CSF), out.view(rows, k))
        return out
    assert torch.equal(read(good), want)
    if rows > 1:
        assert torch.equal(read(good, rows * 2, k // 2), want)
    for at, values in ((0, [0, 0, 0, 0]), (0, [128, 0, 0, 0]), (0, [255, 255, 255, 255]), (0, [16, 1, 0, 0]), (4, [0, 0, 0, 0]), (4, [(rows - 1) % 256, 0, 0, 0]),
                       (8, [255 if rows > 1 else 4]), (9, [6 if rows > 1 else 8])):
        bad = good.clone()
        bad[at:at + len(values)] = torch.tensor(values, dtype=torch.uint8, device="cuda")
        if torch.equal(bad, good):
            continue
        assert torch.isnan(read(bad)).all(), (at, values)
    assert torch.isnan(read(torch.zeros_like(good))).all()


@pytest.mark.parametrize("rows,k", [(1, 32), (33, 96), (128, 64), (130, 1600), (300, 160)])
def test_operands_out_of_requantised_weights(module, rows, k):
    """What the flat quantiser leaves, as the product's operand, by way of the converter or of memory that empty() gives."""
    x = torch.randn(rows, k, device="cuda") * 0.02
    raw = b2.Nvfp4Tensor.empty(rows, k, b2.SCALES_RAW)
    b2.Nvfp4QuantModule().fp32_to_nvfp4_four_six(x, x.abs().max().reshape(1), raw.bytes, raw.scales, raw.global_scale, rows * k // 16, b2.SCALES_RAW)
    tiled = b2.scales_to_sm100(raw.scales, b2.SCALES_RAW, rows, k)
    t = b2.Nvfp4Tensor.empty(rows, k, b2.SCALES_SM100)
    t.bytes.copy_(raw.bytes)
    t.scales.copy_(tiled)
    t.global_scale.copy_(raw.global_scale)
    w = plain.values(plain.unpack(raw.bytes.cpu().numpy().reshape(rows, -1), k), raw.scales.cpu().numpy().reshape(rows, -1), raw.global_scale.item())
    a = torch.randn(50, k, device="cuda")
    for tensor in (b2.Nvfp4Tensor(raw.bytes, tiled, raw.global_scale, rows, k, b2.SCALES_SM100), t):
        o = b2.Nvfp4Operand.from_tensor(tensor)
        assert o.bytes.data_ptr() == tensor.bytes.data_ptr() and (o.rows, o.k) == (rows, k)
        out = torch.empty(50, rows, device="cuda")
        module.linear_forward(a, o, out, b2.Nvfp4LinearScratch(50, k, rows))
        within(out, rounded(plain.to_double(a)), w, torch.float32)
        back = torch.empty(rows, k, device="cuda")
        module.decode(tensor, back)
        np.testing.assert_array_equal(plain.to_double(back), plain.rounded_once(w, torch.float32))
    for bad in (raw, b2.Nvfp4Tensor(raw.bytes, tiled[:-1], raw.global_scale, rows, k, b2.SCALES_SM100)):
        with pytest.raises(ValueError):
            b2.Nvfp4Operand.from_tensor(bad)
    if rows > 1:
        with pytest.raises(ValueError):
            b2.Nvfp4Operand.from_tensor(b2.Nvfp4Tensor.empty(rows, 48, b2.SCALES_SM100))


# few rows over more tiles of columns than there are SMs (pipelines shorter than K, several CTAs an SM), over a long K, and the 33 .. 64
# rows that take the few rows' way where K is long
FEW_ROWS = [(1, 50257, 1600), (8, 50257, 1600), (32, 50257, 1600), (33, 1600, 6400), (40, 1600, 6400), (64, 1600, 6400), (64, 48, 4112), (3, 64, 33008),
            (64, 20000, 4096), (17, 129, 70000)]


@pytest.mark.parametrize("m,n,k", FEW_ROWS)
def test_matmul_of_few_rows(module, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, oa = operand(rng, m, k, True)
    b, ob = operand(rng, n, k, False, 16)
    want, bound = a @ b.T, None
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        module.matmul(oa, ob, out)
        assert module.status() == 0
        bound = product_bound(a, b, want, dtype)
        assert (np.abs(plain.to_double(out) - want) <= bound).all()


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 1600, 50257), (8, 1000, 20000), (1, 1001, 50257), (1, 7, 33), (3, 1001, 300), (8, 1024, 19000), (2, 4095, 64), (8, 33, 129)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offset,gap", [(0, 0), (1, 0), (8, 8), (3, 5)])
def test_linear_of_few_rows(module, tokens, inputs, outputs, dtype, offset, gap):
    """Rows quantised inside the product: of any length, with gaps, on any boundary; what is around them is not read into them."""
    rng = np.random.default_rng(tokens + outputs + offset)
    x = activations(rng, tokens, inputs, dtype) / 64
    memory = torch.full((offset + tokens * (inputs + gap),), float("nan"), dtype=x.dtype, device="cuda")
    view = memory[offset:].view(tokens, inputs + gap)[:, :inputs]
    view.copy_(x)
    k = -(-inputs // 16) * 16
    w, ow = operand(rng, outputs, k, False)
    out = torch.empty(tokens, outputs, device="cuda")
    module.linear_forward(view, ow, out, b2.Nvfp4LinearScratch(tokens, inputs, outputs))
    q = np.zeros((tokens, k))
    q[:, :inputs] = rounded(plain.to_double(x))
    within(out, q, w, torch.float32)


@pytest.mark.parametrize("m,n,k", [(1, 300, 6400), (5, 20000, 1600), (64, 130, 6400), (24, 1600, 6400), (3, 64, 33008), (300, 500, 6400), (140, 301, 16400), (1100, 2100, 1616),
                                   (1100, 2101, 4000)])
def test_matmul_of_exact_sums(module, m, n, k):
    """Products that are multiples of 1/4 and add up to less than 2^22: FP32 has every sum, in any order, so nothing may be missing."""
    rng = np.random.default_rng(k + m)
    s_range = (1,) if k > 6400 else (1, 2, 4)   # 6 6 s s 6400 < 2^22
    sides = []
    for rows in (m, n):
        codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
        s = rng.choice([0x38 + 8 * int(np.log2(v)) for v in s_range], (rows, k // 16)).astype(np.uint8)
        sides.append((plain.values(codes, s, [1.0]), b2.Nvfp4Operand(torch.from_numpy(plain.pack(codes, -(-k // 32) * 16)).cuda(),
                                                                     torch.from_numpy(plain.tiled(s)).cuda(), torch.ones(1, device="cuda"), rows, k)))
    (a, oa), (b, ob) = sides
    assert (np.abs(a).max() * np.abs(b).max()) * k < 2 ** 22
    out = torch.empty(m, n, device="cuda")
    module.matmul(oa, ob, out)
    np.testing.assert_array_equal(plain.to_double(out), a @ b.T)


def test_a_cache_is_not_read_into_the_same_place_twice(module):
    cache = b2.Nvfp4PagedCache.empty(4, 8, 2, 32)
    table, lengths = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    good, memory = torch.zeros(3, 8, 2, 32, device="cuda"), torch.zeros(4096, device="cuda")
    for strides in ((256, 64, 32, 1), (511, 32, 256, 1)):
        for bad in (memory.as_strided((3, 8, 2, 32), strides), good):
            with pytest.raises(ValueError):
                module.cache_read(cache, table, lengths, bad, good)
    both = torch.zeros(3, 8, 2, 2, 32, device="cuda")
    module.cache_read(cache, table, lengths, both[:, :, 0], both[:, :, 1])
    module.cache_read(cache, table, lengths, memory.as_strided((3, 8, 2, 32), (512, 32, 256, 1)), good)   # head by head


def test_decode_refuses_another_scale_type(module):
    out = torch.empty(4, 32, device="cuda")
    for bad in (torch.ones(1, dtype=torch.float64, device="cuda"), torch.ones(1, dtype=torch.bfloat16, device="cuda"), torch.ones(0, device="cuda"), torch.ones(1)):
        t = b2.Nvfp4Tensor.empty(4, 32, b2.SCALES_RAW)
        t.global_scale = bad
        with pytest.raises(ValueError):
            module.decode(t, out)


@pytest.mark.parametrize("m,n,k", [(40, 300, 64), (140, 300, 272), (140, 301, 272), (1100, 2101, 64)])
def test_rows_of_zeros_beside_small_weights(module, m, n, k):
    """The scale of a row of zeros is the least that there is, and its product with a small weight's is subnormal: the row stays zero and the
    others are what they are without it, bit for bit, with tiny rows among them too."""
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, k)).astype(np.float32)
    w, ow = operand_at(rng, n, k, False, -20, (0x28, 0x79), None)
    bias = torch.randn(n, device="cuda")
    outs = []
    for zeros in (False, True):
        x[1::3] *= not zeros
        x[5] *= np.float32(2.0 ** -102) if zeros else 1
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
            module.linear_forward(torch.from_numpy(x).cuda(), ow, out, b2.Nvfp4LinearScratch(m, k, n), bias=bias)
            outs.append(out)
    kept = np.setdiff1d(np.arange(m), np.r_[1:m:3, 5])
    for whole, some in zip(outs[:2], outs[2:]):
        assert torch.equal(whole[kept], some[kept])
        assert (some[1::3] == bias.to(some.dtype)).all()
    q = rounded(x.astype(np.float64))
    out = torch.empty(m, n, device="cuda")
    module.linear_forward(torch.from_numpy(x).cuda(), ow, out, b2.Nvfp4LinearScratch(m, k, n))
    check_at_the_ends(out, q @ w.T, np.abs(q) @ np.abs(w).T, k, torch.float32)


@pytest.mark.parametrize("tokens,inputs", [(2, 160), (8, 1008), (20, 6400), (60, 4160), (300, 160)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_that_are_not_finite_stay_apart(module, tokens, inputs, dtype):
    rng = np.random.default_rng(tokens)
    x = activations(rng, tokens, inputs, dtype) / 64
    good = x.clone()
    x[1, 3], x[-1, inputs - 1] = float("inf"), float("nan")
    w, ow = operand(rng, 200, inputs, False)
    out = torch.zeros(tokens, 200, device="cuda")
    module.linear_forward(x.cuda(), ow, out, b2.Nvfp4LinearScratch(tokens, inputs, 200))
    bad = np.isin(np.arange(tokens), [1, tokens - 1])
    got, q = plain.to_double(out), rounded(plain.to_double(good))
    want = q @ w.T
    assert np.isnan(got[bad]).all()
    assert (np.abs(got - want) <= product_bound(q, w, want, torch.float32))[~bad].all()
