"""Masked attention where it is easily wrong: several non-finite values in a block, steep biases, caps that
saturate, rows outside the segments. Against the FP64 definition (attention_reference.py)."""
import pytest

torch = pytest.importorskip("torch")
import attention_reference as R  # noqa: E402
from test_gpu_attention import Batch  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    import gatb200
    return gatb200


def plant(b):
    """Non-finite values of many keys of the same blocks, on both sides of each block's key 64, in columns of their own
    and in shared ones (Inf and -Inf of one column make NaN, whichever key comes first)."""
    inf, nan = float("inf"), float("nan")
    for key, col, x in [(3, 0, inf), (5, 0, inf), (40, 1, -inf), (63, 2, inf), (64, 3, inf), (65, 4, nan), (66, 5, inf),
                        (67, 5, -inf), (100, 33, inf), (101, 34, -inf), (127, 35, inf), (130, 36, inf), (195, 37, nan),
                        (196, 38, inf), (210, 7, inf)]:
        b.v[key, col] = x


@pytest.mark.parametrize("mask", [0, 1, 2])
@pytest.mark.parametrize("dim", [40, 64, 72, 128])
def test_many_non_finite_values_of_a_block(G, dev, dim, mask):
    lens = [30, 100, 90]
    b = Batch(dev, lens, lens, 4, 2, dim, seed=dim)
    plant(b)
    prefix = [20, 99, 45] if mask == 2 else None
    b.run(G, mask, prefix)
    b.check(b.reference(mask=mask, prefix=prefix))
