"""4-bit products whose row scales lie far apart, against the FP64 definition (fp4_reference.py)."""
import numpy as np
import pytest

import fp4_reference as R

torch = pytest.importorskip("torch")
from test_gpu_fp4 import check_product, features, product, table  # noqa: E402

pytestmark = pytest.mark.gpu
SHAPES = [(5, 40, 128), (100, 70, 256), (300, 300, 128)]  # few rows, many rows of one tile, CTA pairs


@pytest.fixture(scope="module")
def G():
    import gatb200
    return gatb200


def rescale(t, row):
    """The same codes and block scales under other row scales."""
    before = t["row"].cpu().numpy().astype(np.float64)
    t["values"] = t["values"] / before[:, None] * row.astype(np.float64)[:, None]
    t["row"] = torch.from_numpy(row.astype(np.float32)).to(t["row"].device)
    return t


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_rows_of_a_few_huge_elements(G, dev, m, n, k):
    """Row scales whose product is no FP32 number, while the products are: a huge element meets zeros."""
    xa, xb = features(m, k, 1, "f32"), features(n, k, 2, "f32")
    xa[:, :16], xb[:, :16] = 0, 0
    xa[::3], xb[::2] = 0, 0
    xa[::3, 0], xb[::2, 1] = 3e38, 1e9
    xb[1::2, 0] = 1e-9
    for bf16 in (False, True):
        a, b = table(xa, R.NV, dev), table(xb, R.NV, dev)
        out = product(G, R.NV, a, b, m, n, k, G.BF16 if bf16 else G.F32, dev=dev)
        assert torch.isfinite(out).all()
        check_product(out.float().cpu().numpy(), a, b, bf16)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("ea,eb", [(-100, -49), (-75, -76), (100, -149), (-140, 127), (120, 8), (-126, 20), (0, 0)])
def test_row_scales_of_any_size(G, dev, m, n, k, ea, eb):
    """Row scales of both signs around 2^ea and 2^eb whose product leaves FP32's normal range or passes near its ends."""
    rng = np.random.default_rng(m + n)
    a, b = table(features(m, k, 3, "f32"), R.NV, dev), table(features(n, k, 4, "f32"), R.NV, dev)

    def scales(size, e):
        x = rng.uniform(1, 2, size) * rng.choice([-1.0, 1.0], size) if e > -127 else np.ones(size)
        return (x * 2.0 ** e).astype(np.float32)
    rescale(a, scales(m, ea))
    rescale(b, scales(n, eb))
    out = product(G, R.NV, a, b, m, n, k, G.F32, dev=dev).double().cpu().numpy()
    want = a["values"] @ b["values"].T
    mag = np.abs(a["values"]) @ np.abs(b["values"]).T
    # the sums, one rounding of the result (two where the scales' product is rounded first), a step of the subnormals
    tol = mag * k * 2.0 ** -24 + np.abs(want) * 3 * 2.0 ** -24 + 2.0 ** -149
    over = np.abs(want) + tol >= float(np.finfo(np.float32).max)
    assert (np.abs(out - want)[~over] <= tol[~over]).all()
    assert not np.isnan(out).any() and (np.abs(want) + tol).min() < float(np.finfo(np.float32).max)
