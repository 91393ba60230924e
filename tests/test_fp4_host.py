"""4-bit tables: sizes and refused calls (no GPU needed), and the checker's own grids."""
import numpy as np
import pytest

import fp4_reference as R
import gatb200 as G


def test_sizes():
    assert [G.fp4_ld(w) for w in (1, 32, 33, 100, 256)] == [16, 16, 32, 64, 128]
    assert G.fp4_ld(0) == 0 and G.fp4_scale_bytes(1, 5, 32) == 0
    assert G.fp4_scale_bytes(G.MXFP4, 128, 128) == 512
    assert G.fp4_scale_bytes(G.NVFP4, 129, 128) == 2048
    assert G.fp4_scale_bytes(G.MXFP4, 0, 128) == 0


def test_reference_grids():
    assert len(R.E4M3) == 127 and R.E4M3[-1] == 448 and R.E4M3[1] == 2.0 ** -9 and (np.diff(R.E4M3) > 0).all()
    c, byte, scale, row = R.quantize(np.array([[6.0, 0.25, 0.75, -5.0] + [0.0] * 28]), R.MX)
    assert byte[0, 0] == 127 and list(c[0, :4]) == [7, 0, 2, 14]


BAD_QUANTIZE = [
    (dict(fmt=1), "bad format"),
    (dict(x_dtype=2), "bad input dtype"),
    (dict(width=0), "bad width"),
    (dict(ldx=31), "row stride smaller"),
    (dict(ldc=8), "16-byte aligned"),
    (dict(ldc=24), "16-byte aligned"),
    (dict(n=1 << 40), "too many rows"),
    (dict(x=None), "null argument"),
    (dict(scales=None), "null argument"),
    (dict(fmt=3, row=None), "needs the row scales"),
    (dict(x=0x1001), "misaligned"),
    (dict(codes=0x1008), "16-byte aligned"),
    (dict(values=0x1000, v_dtype=5), "bad values dtype"),
    (dict(values=0x1000, ldv=31), "values row stride"),
]


@pytest.mark.parametrize("change,message", BAD_QUANTIZE)
def test_quantize_refusals(change, message):
    a = dict(fmt=2, n=4, width=32, x=0x1000, x_dtype=0, ldx=32, codes=0x2000, ldc=16, scales=0x3000, row=None, values=None,
             v_dtype=1, ldv=32)
    a.update(change)
    with pytest.raises(G.GatError, match=message) as e:
        G.fp4_quantize(a["fmt"], a["n"], a["width"], a["x"], a["x_dtype"], a["ldx"], a["codes"], a["ldc"], a["scales"],
                       a["row"], a["values"], a["v_dtype"], a["ldv"])
    assert e.value.code == G.EINVAL


BAD_PRODUCT = [
    (dict(fmt=0), "bad format"),
    (dict(out_dtype=2), "bad output dtype"),
    (dict(k=0), "bad shape"),
    (dict(n=-1), "bad shape"),
    (dict(m=1 << 40), "too many rows"),
    (dict(lda=16), "16-byte aligned"),
    (dict(ldb=40), "16-byte aligned"),
    (dict(ldo=7), "output row stride"),
    (dict(a=None), "null argument"),
    (dict(out=None), "null argument"),
    (dict(b_scales=0x1004), "16-byte aligned"),
    (dict(out=0x1002), "misaligned"),
]


@pytest.mark.parametrize("change,message", BAD_PRODUCT)
def test_product_refusals(change, message):
    a = dict(fmt=2, m=4, n=8, k=64, a=0x1000, lda=32, a_scales=0x2000, b=0x3000, ldb=32, b_scales=0x4000, out=0x5000,
             out_dtype=0, ldo=8)
    a.update(change)
    with pytest.raises(G.GatError, match=message) as e:
        G.fp4_product(a["fmt"], a["m"], a["n"], a["k"], a["a"], a["lda"], a["a_scales"], None, a["b"], a["ldb"],
                      a["b_scales"], None, a["out"], a["out_dtype"], a["ldo"])
    assert e.value.code == G.EINVAL
