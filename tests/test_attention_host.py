"""Refused calls of masked attention (no GPU needed)."""
import pytest

import gatb200 as G

NAN, INF = float("nan"), float("inf")
COMMON = [
    (dict(heads=0), "multiple of kv_heads", G.EINVAL),
    (dict(kv_heads=3), "multiple of kv_heads", G.EINVAL),
    (dict(dim=0), "multiple of 8", G.EUNSUPPORTED),
    (dict(dim=12), "multiple of 8", G.EUNSUPPORTED),
    (dict(dim=136), "multiple of 8", G.EUNSUPPORTED),
    (dict(n_k=1 << 40), "too many rows", G.EINVAL),
    (dict(nseg=-1), "segment count", G.EINVAL),
    (dict(scale=0.0), "scale", G.EINVAL),
    (dict(scale=NAN), "scale", G.EINVAL),
    (dict(scale=INF), "scale", G.EINVAL),
    (dict(cap=-1.0), "cap", G.EINVAL),
    (dict(cap=INF), "cap", G.EINVAL),
    (dict(cap=2e30), "cap", G.EINVAL),
    (dict(cap=1e-35), "cap too small", G.EINVAL),
    (dict(scale=2e30), "scale", G.EINVAL),
    (dict(ldq=100), "row stride", G.EINVAL),
    (dict(ldo=124), "row stride", G.EINVAL),
    (dict(ldk=63), "row stride", G.EINVAL),
    (dict(ldv=68), "16-byte aligned", G.EINVAL),
    (dict(q=0x1008), "16-byte aligned", G.EINVAL),
    (dict(q=None), "null argument", G.EINVAL),
    (dict(v=None), "null argument", G.EINVAL),
    (dict(slopes=0x1002), "misaligned", G.EINVAL),
    (dict(lse=0x1002), "misaligned", G.EINVAL),
]
BASE = dict(heads=4, kv_heads=2, dim=32, nseg=2, n_q=10, n_k=10, q_row=0x1000, k_row=0x1000, mask=0, prefix=None, q=0x2000,
            ldq=128, k=0x3000, ldk=64, v=0x4000, ldv=64, scale=0.1, cap=0.0, slopes=None, out=0x5000, ldo=128, lse=None)


@pytest.mark.parametrize("change,message,code", COMMON + [
    (dict(mask=3), "bad mask", G.EINVAL),
    (dict(mask=-1), "bad mask", G.EINVAL),
    (dict(mask=2), "prefix lengths", G.EINVAL),
    (dict(nseg=0), "rows without segments", G.EINVAL),
    (dict(n_q=1 << 40), "too many rows", G.EINVAL),
    (dict(q_row=None), "null argument", G.EINVAL),
    (dict(k_row=0x1004), "misaligned", G.EINVAL),
])
def test_refusals(change, message, code):
    a = {**BASE, **change}
    with pytest.raises(G.GatError, match=message) as e:
        G.masked_attention(**a)
    assert e.value.code == code


@pytest.mark.parametrize("change,message,code", COMMON + [
    (dict(begin=None), "null argument", G.EINVAL),
    (dict(length=0x1004), "misaligned", G.EINVAL),
    (dict(workspace=None), "workspace too small", G.EINVAL),
    (dict(workspace_bytes=1000), "workspace too small", G.EINVAL),
    (dict(workspace=0x6008), "misaligned", G.EINVAL),
])
def test_step_refusals(change, message, code):
    a = {k: v for k, v in BASE.items() if k not in ("n_q", "q_row", "k_row", "mask", "prefix")}
    a.update(begin=0x1000, length=0x1000, workspace=0x6000, workspace_bytes=1 << 30)
    a.update(change)
    with pytest.raises(G.GatError, match=message) as e:
        G.masked_attention_step(**a)
    assert e.value.code == code


def test_nothing_to_do():
    G.masked_attention(**{**BASE, "n_q": 0, "nseg": 0, "q": None, "out": None})
    assert G.masked_attention_step_workspace(4, 32, 3) > 0
    assert G.masked_attention_step_workspace(0, 32, 3) == 0
