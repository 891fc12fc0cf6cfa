"""NVFP4 quantisation and products in 64 bits, from the definition: what the 4-bit operators are tested against (CPU)."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _nearest_even(v, grid):
    """Index of the value of the ascending `grid` nearest to each v >= 0, the even index between two; the last one beyond."""
    v = np.minimum(v, grid[-1])
    hi = np.minimum(np.searchsorted(grid, v), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = v - grid[lo], grid[hi] - v
    return np.where(below < above, lo, np.where(above < below, hi, np.where(lo % 2 == 0, lo, hi)))


def e4m3_grid():
    """The values of the E4M3 codes 0 .. 126."""
    c = np.arange(127)
    e, f = c >> 3, c & 7
    return np.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7.0), f * 2.0 ** -9)


def top_scale(amax):
    """2^(floor(log2 amax) - 10) with amax >= 2^-100; NaN where amax is not finite."""
    with np.errstate(all="ignore"):
        g = 2.0 ** (np.floor(np.log2(np.maximum(amax, 2.0 ** -100))) - 10)
    return np.where(np.isfinite(amax), g, np.nan)


def quantise(x, whole=False):
    """x [rows, k] -> codes [rows, k16] (sign in bit 3), E4M3 codes [rows, k16 / 16], g [rows] (one for all with `whole`)."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    k16 = -(-k // 16) * 16
    pad = np.zeros((rows, k16))
    pad[:, :k] = x
    amax = np.abs(pad).max(1) if rows else np.zeros(0)
    bad = ~np.isfinite(amax)
    if whole:
        amax = np.full(rows, np.nan if bad.any() else amax.max())
        bad = np.full(rows, bad.any())
    g = top_scale(np.where(bad, np.nan, amax))
    blocks = np.where(bad[:, None], 0.0, pad).reshape(rows, -1, 16)
    g1 = np.where(bad, 1.0, g)
    s = _nearest_even(np.abs(blocks).max(2) / 6 / g1[:, None], e4m3_grid())
    step = (e4m3_grid()[s] * g1[:, None])[:, :, None]
    q = np.where(step > 0, np.abs(blocks) / np.where(step > 0, step, 1), 0.0)
    codes = _nearest_even(q, GRID) + 8 * (blocks < 0)
    return codes.reshape(rows, k16).astype(np.uint8), s.astype(np.uint8), g


def values(codes, s, g):
    """What codes stand for, in 64 bits; g: one a row, or one."""
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    rows, k = codes.shape
    return (v.reshape(rows, -1, 16) * e4m3_grid()[s][:, :, None]).reshape(rows, k) * np.asarray(g, np.float64).reshape(-1, 1)


def pack(codes, row_bytes=None):
    p = codes[:, 0::2] | (codes[:, 1::2] << 4)
    if row_bytes is None:
        return p
    out = np.zeros((len(p), row_bytes), np.uint8)
    out[:, : p.shape[1]] = p
    return out


def unpack(p, k):
    p = p[:, : k // 2]
    return np.stack([p & 15, p >> 4], -1).reshape(len(p), k)


def tiled(s):
    """[rows, blocks] scales -> 128 x 4 tiles, zeros behind the ends."""
    rows, blocks = s.shape
    r, b = -(-rows // 128), -(-blocks // 4)
    full = np.zeros((r * 128, b * 4), np.uint8)
    full[:rows, :blocks] = s
    return full.reshape(r, 4, 32, b, 4).transpose(0, 3, 2, 1, 4).reshape(-1)


def untiled(t, rows, blocks):
    """The same back; also the padding behind the blocks of the rows that there are."""
    r, b = -(-rows // 128), -(-blocks // 4)
    full = np.asarray(t)[: r * b * 512].reshape(r, b, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(r * 128, b * 4)
    return full[:rows, :blocks], full[:rows, blocks:]


def random_operand(rng, rows, k, per_row, row_bytes=None):
    """A random NVFP4 operand: (values in 64 bits, packed codes, scales [rows, blocks], g)."""
    codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    s = rng.integers(0x28, 0x79, (rows, k // 16)).astype(np.uint8)
    g = (np.exp2(rng.integers(-8, -3, rows if per_row else 1)) * (1.0 if per_row else 1.37)).astype(np.float32)
    return values(codes, s, g), pack(codes, row_bytes), s, g


def to_double(t):
    return t.detach().double().cpu().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded_once(v, dtype):
    """Numbers in 64 bits to the nearest ones of `dtype` (still in 64 bits), the even one between two; beyond the range infinity."""
    bits, least = {torch.float32: (23, -126), torch.bfloat16: (7, -126), torch.float16: (10, -14)}[dtype]
    v = np.asarray(v, np.float64)
    with np.errstate(all="ignore"):
        unit = np.exp2(np.maximum(np.floor(np.log2(np.abs(v))), least) - bits)
        r = np.where(v == 0, v, np.rint(v / unit) * unit)
    return np.where(np.abs(r) > torch.finfo(dtype).max, np.copysign(np.inf, v), r)
