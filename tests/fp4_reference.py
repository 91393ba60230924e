"""4-bit microscaled tables in numpy FP64, from the definition: the checker of
gat_b200_fp4_quantize and gat_b200_fp4_product."""
import numpy as np

MX, NV = 2, 3
BLOCK = {MX: 32, NV: 16}
VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


def bf16_round(x):
    """FP32 values rounded to BF16 (nearest even), as FP32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
    return r.view(np.float32)


def _nearest_even(y, grid):
    """Index of the nearest grid point; halfway cases take the even index."""
    hi = np.clip(np.searchsorted(grid, y, side="left"), 1, len(grid) - 1)
    lo = hi - 1
    a, b = y - grid[lo], grid[hi] - y
    return np.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)


def _e4m3_grid():
    g = [m * 2.0 ** -9 for m in range(8)]
    g += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return np.array(g[:-1])  # the last code is NaN


E4M3 = _e4m3_grid()


def quantize(x, fmt):
    """(codes 0..15 [n][w], scale bytes [n][blocks], scale values, row scales)."""
    x = np.asarray(x, np.float64)
    n, w = x.shape
    b = BLOCK[fmt]
    nb = -(-w // b)
    xp = np.zeros((n, nb * b))
    xp[:, :w] = x
    xb = xp.reshape(n, nb, b)
    amax = np.abs(xb).max(-1)  # NaN wins
    row = np.ones(n)
    if fmt == MX:
        with np.errstate(divide="ignore", invalid="ignore"):
            _, e = np.frexp(np.where(np.isfinite(amax), amax, 1.0))
        e = np.where(amax > 0, np.clip(e - 3, -127, 127), -127)
        byte = np.where(np.isfinite(amax), e + 127, 255).astype(np.uint8)
        scale = np.where(np.isfinite(amax), np.exp2(e.astype(np.float64)), np.nan)
    else:
        top = amax.max(-1)
        fin = np.isfinite(top)
        m, e = np.frexp(np.where(fin, top, 1.0) / 2688.0)
        j = np.where(m == 0.5, e - 1, e)  # smallest j with top / 2688 <= 2^j
        row = np.where(top == 0, 1.0, np.exp2(np.maximum(j, -100).astype(np.float64)))
        want = np.where(fin[:, None], np.where(np.isfinite(amax), amax, 0.0) / (6.0 * row[:, None]), 0.0)
        byte = _nearest_even(want, E4M3).astype(np.uint8)
        scale = E4M3[byte]
        row = np.where(fin, row, np.nan)
    full = (scale * row[:, None])[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(full > 0, np.abs(xb) / full, 0.0)
    code = _nearest_even(np.minimum(np.where(np.isnan(y), 0, y), 6.0), VALUES)
    code = np.where((xb < 0), code + 8, code)
    return code.reshape(n, nb * b)[:, :w], byte, scale, row


def values(code, scale, row, fmt):
    w = code.shape[1]
    v = np.where(code >= 8, -VALUES[code % 8], VALUES[code % 8])
    return v * np.repeat(scale, BLOCK[fmt], 1)[:, :w] * row[:, None]


def scale_offset(r, blk, tiles):
    """Byte of row r, block blk in the tiled scales of a table with `tiles` tiles a row."""
    return ((r // 128) * tiles + blk // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + blk % 4


def tables(code, byte, fmt):
    """(codes as bytes [n][ld], tiled scales) in the library's layout, padding zero."""
    n, w = code.shape
    ld = (w + 31) // 32 * 16
    c = np.zeros((n, 2 * ld), np.uint8)
    c[:, :w] = code
    nb = byte.shape[1]
    tiles = -(-nb // 4)
    flat = np.zeros(-(-n // 128) * tiles * 512, np.uint8)
    r, k = np.meshgrid(np.arange(n), np.arange(nb), indexing="ij")
    flat[scale_offset(r, k, tiles)] = byte
    return c[:, 0::2] | (c[:, 1::2] << 4), flat
