"""4-bit tables on the GPU against the FP64 definition (fp4_reference.py)."""
import numpy as np
import pytest

import fp4_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
FORMATS = [R.MX, R.NV]


@pytest.fixture(scope="module")
def G():
    import gatb200
    return gatb200


def features(n, w, seed, dtype):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, w)) * np.exp(2 * rng.standard_normal((n, 1)))
    x[rng.random((n, w)) < 0.02] = 0
    x[:, rng.random(w) < 0.05] *= 30
    if n > 3:
        x[3] = 0  # a row of zeros
    if n > 4:
        x[4, : w // 2] *= 1e-6  # blocks far below the row's largest
    x = x.astype(np.float32)
    return R.bf16_round(x) if dtype == "bf16" else x


def to_dev(x, dtype, ld, dev):
    t = torch.full((max(x.shape[0], 1), ld), float("nan"), dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device=dev)
    t[: x.shape[0], : x.shape[1]] = torch.from_numpy(np.ascontiguousarray(x)).to(dev).to(t.dtype)
    return t


def quantize(G, x, fmt, dtype, dev, ldx=None, extra_ldc=0, v_dtype=None, extra_ldv=0, offset=0, stream=None):
    """Runs the library: dict of host arrays, buffers prefilled with 0xA5 / -7."""
    n, w = x.shape
    ldx = ldx or w
    base = torch.zeros(max(n, 1) * ldx + offset, dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device=dev)
    xt = base[offset:]
    xt[: n * ldx].view(n, ldx).copy_(to_dev(x, dtype, ldx, dev)[:n])
    ldc = G.fp4_ld(w) + extra_ldc
    codes = torch.full((max(n, 1), ldc), 0xA5, dtype=torch.uint8, device=dev)
    scales = torch.full((max(G.fp4_scale_bytes(fmt, n, w), 16),), 0xA5, dtype=torch.uint8, device=dev)
    row = torch.full((max(n, 1),), -7.0, device=dev)
    ldv = w + extra_ldv
    vals = None if v_dtype is None else torch.full((max(n, 1), ldv), -7.0, device=dev,
                                                   dtype=torch.float32 if v_dtype == G.F32 else torch.bfloat16)
    G.fp4_quantize(fmt, n, w, xt, G.F32 if dtype == "f32" else G.BF16, ldx, codes, ldc, scales,
                   row if fmt == R.NV else None, values=vals, v_dtype=v_dtype or 0, ldv=ldv, stream=stream)
    torch.cuda.synchronize()
    return dict(codes=codes, scales=scales, row=row, values=vals, ldc=ldc)


def check(G, got, x, fmt, v=True):
    n, w = x.shape
    code, byte, scale, row = R.quantize(x, fmt)
    want_c, want_s = R.tables(code, byte, fmt)
    ld = G.fp4_ld(w)
    c = got["codes"].cpu().numpy()
    lo, hi = c[:n, :ld] & 15, c[:n, :ld] >> 4
    wl, wh = want_c & 15, want_c >> 4
    ok_row = np.isfinite(row)
    same = lambda a, b: (a == b) | ((a % 8 == 0) & (b % 8 == 0))  # noqa: E731  (both zeros)
    blocks_ok = np.repeat(np.isfinite(scale), R.BLOCK[fmt], 1)
    full = np.zeros((n, 2 * ld), bool)
    full[:, :] = True
    k = min(2 * ld, blocks_ok.shape[1])
    full[:, :k] = blocks_ok[:, :k]
    full &= ok_row[:, None]
    assert (same(lo, wl) | ~full[:, 0::2]).all()
    assert (same(hi, wh) | ~full[:, 1::2]).all()
    assert (c[:n, ld:] == 0xA5).all()  # behind the code row: untouched
    nb = byte.shape[1]
    tiles = -(-nb // 4)
    r, b = np.meshgrid(np.arange(n), np.arange(4 * tiles), indexing="ij")
    s = got["scales"].cpu().numpy()
    want = np.zeros((n, 4 * tiles), np.uint8)
    want[:, :nb] = byte
    assert (s[R.scale_offset(r, b, tiles)] == want).all()
    if fmt == R.NV:
        rs = got["row"].cpu().numpy()[:n].astype(np.float64)
        assert np.array_equal(np.isnan(rs), np.isnan(row)) and (rs[ok_row] == row[ok_row]).all()
    if got["values"] is not None:
        vals = got["values"].float().cpu().numpy().astype(np.float64)
        want_v = R.values(code, scale, row, fmt)
        assert np.array_equal(np.isnan(vals[:n, :w]), np.isnan(want_v))
        fin = np.isfinite(want_v)
        assert (vals[:n, :w][fin] == want_v[fin]).all()
        assert (vals[:n, w:] == -7).all()


SHAPES = [(1, 1), (1, 4096), (3, 15), (5, 16), (7, 17), (33, 31), (130, 32), (129, 33), (64, 100), (257, 128), (40, 129),
          (20, 250), (9, 256), (11, 257), (6, 513), (5, 1000), (4, 1024), (3, 1025), (2, 2049), (2, 5000), (2, 8200),
          (1, 20000)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,w", SHAPES)
def test_quantize_matches_the_definition(G, dev, fmt, dtype, n, w):
    x = features(n, w, n * 7919 + w, dtype)
    check(G, quantize(G, x, fmt, dtype, dev, v_dtype=G.BF16), x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,offset,v32", [(1, 0, True), (2, 2, False), (3, 1, True), (4, 4, False), (8, 8, True)])
def test_quantize_strides_and_alignment(G, dev, fmt, dtype, pad, offset, v32):
    x = features(37, 100, 5, dtype)
    got = quantize(G, x, fmt, dtype, dev, ldx=100 + pad, extra_ldc=16, v_dtype=G.F32 if v32 else G.BF16, extra_ldv=pad,
                   offset=offset)
    check(G, got, x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad,vpad,v32", [(1, 0, 3, False), (3, 2, 1, True), (0, 5, 2, False), (2, 3, 0, True)])
@pytest.mark.parametrize("n,w", [(150, 1), (70, 2), (67, 30), (40, 63), (35, 126), (19, 129), (9, 255), (6, 509),
                                 (5, 1023), (3, 2045), (3, 4001), (2, 8190), (2, 8203)])
def test_quantize_rows_that_begin_and_end_anywhere(G, dev, fmt, dtype, n, w, offset, pad, vpad, v32):
    x = features(n, w, 31 * n + w, dtype)
    got = quantize(G, x, fmt, dtype, dev, ldx=w + pad, extra_ldc=0, v_dtype=G.F32 if v32 else G.BF16, extra_ldv=vpad,
                   offset=offset)
    check(G, got, x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_borders_and_ties(G, dev, fmt):
    # every rounding border of E2M1 at every block scale, with its neighbours in FP32
    borders = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    pts = np.concatenate([borders, np.nextafter(borders, np.float32(0)), np.nextafter(borders, np.float32(9)),
                          -borders, [6, 0, 1e-30]]).astype(np.float32)
    rows = []
    if fmt == R.MX:
        for e in (-120, -30, 0, 7, 100):
            for part in (pts[:16], pts[16:]):
                blk = np.zeros(32, np.float64)
                blk[: len(part)] = part
                blk[31] = 4.0
                rows.append((blk * 2.0 ** e).astype(np.float32))
    else:
        for s in R.E4M3[R.E4M3 >= 1]:  # block scale s with row scale 1: a row holds 2688 = 6 * 448
            for i in range(0, len(pts), 14):
                part = pts[i:i + 14].astype(np.float64) * s
                blk = np.zeros(32, np.float64)
                blk[: len(part)] = part
                blk[15] = 6 * s
                blk[16] = 2688
                rows.append(blk.astype(np.float32))
    x = np.stack(rows)
    check(G, quantize(G, x, fmt, "f32", dev, v_dtype=G.F32), x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_extremes(G, dev, fmt):
    x = features(12, 96, 3, "f32")
    x[0] *= np.float32(1e30)
    x[1, 0] = np.float32(3.4e38)
    x[2] = np.float32(1e-40)      # subnormal rows
    x[5, 40] = np.inf
    x[6, 70] = -np.nan
    x[7, 95] = np.nan
    x[8] = np.float32(2.0 ** -149)
    x[9, :] = np.float32(2.0 ** -101) * 2688
    # FP32 values below 2^-126 keep fewer bits: only the codes, scales and row scales are exact there
    got = quantize(G, x, fmt, "f32", dev)
    check(G, got, x, fmt)


def test_quantize_no_rows_and_streams(G, dev):
    got = quantize(G, np.zeros((0, 64), np.float32), R.NV, "f32", dev)
    assert (got["codes"] == 0xA5).all() and (got["scales"] == 0xA5).all()
    st = torch.cuda.Stream()
    x = features(50, 64, 9, "f32")
    check(G, quantize(G, x, R.MX, "f32", dev, stream=st), x, R.MX)


# -------------------------------------------------------------------- product
def table(x, fmt, dev, extra=0):
    code, byte, scale, row = R.quantize(x, fmt)
    c, s = R.tables(code, byte, fmt)
    cp = np.full((c.shape[0], c.shape[1] + extra), 0xA5, np.uint8)
    cp[:, : c.shape[1]] = c
    return dict(codes=torch.from_numpy(cp).to(dev), ld=cp.shape[1], scales=torch.from_numpy(s).to(dev),
                row=torch.from_numpy(row.astype(np.float32)).to(dev) if fmt == R.NV else None,
                values=R.values(code, scale, row, fmt))


def product(G, fmt, a, b, m, n, k, out_dtype, ldo=None, stream=None, dev=None):
    ldo = ldo or n
    out = torch.full((max(m, 1), ldo), -7.0, device=dev, dtype=torch.bfloat16 if out_dtype == G.BF16 else torch.float32)
    G.fp4_product(fmt, m, n, k, a["codes"], a["ld"], a["scales"], a["row"], b["codes"], b["ld"], b["scales"], b["row"],
                  out, out_dtype, ldo, stream=stream)
    torch.cuda.synchronize()
    G.check_device()
    return out


def check_product(got, a, b, bf16):
    want = a["values"] @ b["values"].T
    # FP32 sums of k products, at most k half steps of the sum of magnitudes, and the rounding of the output
    k = a["values"].shape[1]
    mag = np.abs(a["values"]) @ np.abs(b["values"]).T
    tol = mag * k * 2.0 ** -24 + (np.abs(want) * 2.0 ** -8 if bf16 else np.abs(want) * 3 * 2.0 ** -24)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol + 1e-300).all(), float((err / (tol + 1e-300)).max())


PRODUCTS = [(1, 1, 1), (1, 16, 32), (1, 100, 64), (2, 129, 65), (3, 8, 33), (8, 512, 1024), (9, 300, 129), (16, 257, 4096),
            (17, 64, 300), (37, 203, 744), (64, 1000, 512), (65, 40, 200), (100, 128, 256), (128, 128, 256), (129, 130, 257),
            (200, 47, 256), (255, 256, 100), (256, 256, 512), (300, 384, 1111), (513, 200, 31), (1000, 700, 2000),
            (4000, 256, 256), (3, 5003, 2744), (4900, 1000, 300), (19000, 130, 520), (260, 18950, 77), (5001, 1025, 1500)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_matches_fp64(G, dev, fmt, bf16, m, n, k):
    a = table(features(m, k, m + 3 * n + 7 * k, "f32"), fmt, dev)
    b = table(features(n, k, m + 5 * n + 11 * k, "f32"), fmt, dev)
    out = product(G, fmt, a, b, m, n, k, G.BF16 if bf16 else G.F32, dev=dev)
    check_product(out.float().cpu().numpy(), a, b, bf16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,ldo", [(5, 50, 53), (140, 99, 100), (300, 260, 264), (1, 33, 40), (19001, 70, 71),
                                      (18990, 100, 136)])
def test_product_strides_leave_the_rest_alone(G, dev, fmt, m, n, ldo):
    k = 200
    a = table(features(m, k, 1, "f32"), fmt, dev, extra=32)
    b = table(features(n, k, 2, "f32"), fmt, dev, extra=16)
    for dt in (G.F32, G.BF16):
        out = product(G, fmt, a, b, m, n, k, dt, ldo=ldo, dev=dev).float().cpu().numpy()
        check_product(out[:, :n], a, b, dt == G.BF16)
        assert (out[:, n:] == -7).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_product_nan_stays_in_its_row(G, dev, fmt):
    m, n, k = 70, 90, 256
    xa = features(m, k, 1, "f32")
    xa[20, 100] = np.nan
    a, b = table(xa, fmt, dev), table(features(n, k, 2, "f32"), fmt, dev)
    out = product(G, fmt, a, b, m, n, k, G.F32, dev=dev).cpu().numpy()
    assert np.isnan(out[20]).all() and np.isfinite(np.delete(out, 20, 0)).all()


def test_product_is_the_same_every_time_and_replays(G, dev):
    m, n, k = 5, 700, 4096
    a, b = table(features(m, k, 1, "f32"), R.NV, dev), table(features(n, k, 2, "f32"), R.NV, dev)
    first = product(G, R.NV, a, b, m, n, k, G.F32, dev=dev)
    for _ in range(3):
        assert torch.equal(first, product(G, R.NV, a, b, m, n, k, G.F32, dev=dev))
    out = torch.zeros(m, n, device=dev)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        G.fp4_product(R.NV, m, n, k, a["codes"], a["ld"], a["scales"], a["row"], b["codes"], b["ld"], b["scales"],
                      b["row"], out, G.F32, n, stream=st)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)


def test_quantize_then_product(G, dev):
    """The projection as a user runs it: features quantised, multiplied with weights laid out once."""
    n, k, w = 300, 256, 256
    x = features(n, k, 4, "bf16")
    wt = (np.random.default_rng(1).standard_normal((w, k)) / 16).astype(np.float32)
    for fmt in FORMATS:
        qa, qb = quantize(G, x, fmt, "bf16", dev), quantize(G, wt, fmt, "f32", dev)
        out = torch.empty(n, w, device=dev)
        G.fp4_product(fmt, n, w, k, qa["codes"], qa["ldc"], qa["scales"], qa["row"] if fmt == R.NV else None,
                      qb["codes"], qb["ldc"], qb["scales"], qb["row"] if fmt == R.NV else None, out, G.F32, w)
        torch.cuda.synchronize()
        av, bv = (R.values(*(lambda c, _, s, r: (c, s, r))(*R.quantize(t, fmt)), fmt) for t in (x, wt))
        check_product(out.cpu().numpy(), dict(values=av), dict(values=bv), False)


def test_host_pointers_are_refused(G, dev):
    x = torch.zeros(4, 32)
    c = torch.zeros(4, 16, dtype=torch.uint8, device=dev)
    s = torch.zeros(512, dtype=torch.uint8, device=dev)
    with pytest.raises(G.GatError, match="not memory of the current device"):
        G.fp4_quantize(R.MX, 4, 32, x, G.F32, 32, c, 16, s)
