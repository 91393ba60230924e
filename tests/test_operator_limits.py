"""Sizes at the end of 32 bits that the attention operators refuse (no GPU needed)."""
import pytest

import gatb200 as G

BASE = dict(heads=4, kv_heads=2, dim=32, nseg=2, n_k=10, q=0x2000, ldq=128, k=0x3000, ldk=64, v=0x4000, ldv=64,
            scale=0.1, cap=0.0, slopes=None, out=0x5000, ldo=128, lse=None)


@pytest.mark.parametrize("nseg", [2 ** 31 - 1, 2 ** 31 - 32, 2 ** 31 - 512])
def test_segment_counts_past_32_bits(nseg):
    # the search over the segments counts 32 lanes past their end in 32 bits
    with pytest.raises(G.GatError, match="too many segments") as e:
        G.masked_attention(**{**BASE, "nseg": nseg}, n_q=10, q_row=0x1000, k_row=0x1000, mask=0, prefix=None)
    assert e.value.code == G.EINVAL
    with pytest.raises(G.GatError, match="too many") as e:
        G.masked_attention_step(**{**BASE, "nseg": nseg}, begin=0x1000, length=0x1000, workspace=0x6000,
                                workspace_bytes=1 << 63)
    assert e.value.code == G.EINVAL
