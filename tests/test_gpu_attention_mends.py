"""Masked attention where it is easily wrong: several non-finite values in a block, steep biases, caps that
saturate, rows outside the segments. Against the FP64 definition (attention_reference.py)."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_reference as R  # noqa: E402
from test_gpu_attention import Batch, Step, slopes_of  # noqa: E402

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


@pytest.mark.parametrize("cap,bias", [(20.0, False), (50.0, False), (20.0, True), (50.0, True), (60.0, True), (0.0, True)])
@pytest.mark.parametrize("mask", [0, 1, 2])
@pytest.mark.parametrize("dim", [40, 128])
def test_many_non_finite_values_under_caps_and_biases(G, dev, dim, mask, cap, bias):
    lens = [30, 100, 90]
    b = Batch(dev, lens, lens, 4, 2, dim, seed=dim, qscale=4.0)
    plant(b)
    prefix = [20, 99, 45] if mask == 2 else None
    sl = slopes_of(4, dev) if bias else None
    b.run(G, mask, prefix, cap, sl)
    b.check(b.reference(mask=mask, prefix=prefix, cap=cap, slopes=sl))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3.3e38])
@pytest.mark.parametrize("cap,bias", [(20.0, False), (50.0, True)])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_masked_never_arrives_under_a_cap(G, dev, value, cap, bias, dim):
    """Segments and earlier rows beside non-finite keys and values, to the tolerance: the polynomial of the tanh is
    chosen by a block's products, masked ones among them, so the last bits may differ."""
    lens = [30, 100, 60, 200, 129]
    b = Batch(dev, lens, lens, 2, 2, dim, seed=5)
    sl = slopes_of(2, dev) if bias else None
    want = b.reference(mask=1, cap=cap, slopes=sl)
    b.k[40, :dim] = value
    b.v[45, 3] = value
    b.v[300, 10:30] = value
    b.q[200, 5] = value
    b.run(G, 1, None, cap, sl)
    rows = torch.tensor([i for s in (0, 2, 4) for i in range(b.q_row[s], b.q_row[s + 1])] + list(range(30, 40)) +
                        [i for i in range(190, 300) if i != 200], device=dev)
    R.check(b.out[rows, :2 * dim], b.lse[rows], {key: t[rows] for key, t in want.items()})


@pytest.mark.parametrize("cap", [30.0, 50.0, 53.0, 55.0, 55.4, 56.0])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_saturated_scores_under_a_bias(G, dev, cap, sign, dim):
    """All scores lie at -cap (or cap), so the bias alone decides: keys far below the nearest one's weight still count."""
    lens = [1500, 40]
    for slopes in ([0.5, 2.0 ** -8, -0.5, -2.0 ** -8], [3.0, 2.0 ** -6, 0.0, 2.0 ** -10]):
        b = Batch(dev, lens, lens, 4, 2, dim, seed=3)
        b.q[:b.nq, :4 * dim], b.k[:b.nk, :2 * dim] = 8.0, sign * 8.0
        sl = torch.tensor(slopes, device=dev)
        for mask in (0, 1):
            b.run(G, mask, None, cap, sl)
            b.check(b.reference(mask=mask, cap=cap, slopes=sl))


@pytest.mark.parametrize("cap", [30.0, 55.4, 56.0])
@pytest.mark.parametrize("sign,size", [(-1.0, 2.0 ** -20), (-1.0, 1.0), (1.0, 1.0), (1.0, 2.0 ** 40)])
@pytest.mark.parametrize("dim", [64, 128])
def test_saturated_scores_and_the_size_of_values(G, dev, cap, sign, size, dim):
    b = Batch(dev, [300, 1], [300, 1], 2, 1, dim, seed=3)
    b.q[:b.nq, :2 * dim], b.k[:b.nk, :dim] = 8.0, sign * 8.0
    b.v *= size
    b.run(G, 1, None, cap)
    b.check(b.reference(mask=1, cap=cap))


def lse_of(z):
    """log-sum-exp per row of FP64 scores [rows][keys] (-inf: not seen) and each key's share of its row."""
    lse = torch.logsumexp(z, 1)
    return lse, torch.exp(z - lse[:, None]).nan_to_num(0.0)


@pytest.mark.parametrize("cap", [0.0, 30.0, 60.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slope", [1.0, 64.0, 1000.0, 1e6, -64.0, -1e6])
@pytest.mark.parametrize("mask", [0, 1])
def test_steep_biases_keep_the_score(G, dev, cap, dim, slope, mask):
    """The bias of the key that decides a row may not carry the rounding of a larger one: at distance 0 a score stays what
    it is, whatever the slope."""
    first, n = 97, 403  # the second segment begins inside a tile, so that blocks end at every row of a warp
    b = Batch(dev, [first, n], [first, n], 1, 1, dim, seed=4, qscale=2.0)
    sl = torch.tensor([slope], device=dev)
    b.run(G, mask, None, cap, sl)
    q, k = b.q[first:first + n, :dim].double(), b.k[first:first + n, :dim].double()
    dot, mag = q @ k.t() * b.scale, q.abs() @ k.abs().t() * b.scale
    z = cap * torch.tanh(dot / cap) if cap else dot
    far = (torch.arange(n, device=dev)[:, None] - torch.arange(n, device=dev)[None, :])
    seen = far >= 0 if mask else far > -n
    far = far.abs().double()
    # FP32: dim products and sums, the coefficients' and the tanh's error, four roundings of the score (with the
    # reference that is taken off, a quarter of the cap), two of the key's own bias; shared out by the keys' weights
    err = mag * (dim + 4) * 2.0 ** -24 + (z.abs() + cap / 4) * 2.0 ** -21 + abs(slope) * far * 2.0 ** -22
    z = torch.where(seen, z - slope * far, torch.full_like(z, -float("inf")))
    lse, w = lse_of(z)
    # then the sum's logarithm and the reference added to it
    tol = 2 * (w * err).sum(1) + 2.0 ** -20 + (lse.abs() + cap) * 2.0 ** -22 + n * 2.0 ** -24
    over = (b.lse[first:first + n, 0].double() - lse).abs() / tol
    assert float(over.max()) <= 1, float(over.max())


@pytest.mark.parametrize("lens", [[1000], [40, 3, 0, 700], [20000], [9, 5000, 300]])
@pytest.mark.parametrize("dim", [64, 128])
def test_step_of_equal_values_is_that_value(G, dev, lens, dim):
    """A row is an average over its own rounded weights: here all weights but one round down by nearly half a step, and a
    constant column still comes out as it is."""
    b = Step(dev, lens, 4, 2, dim, seed=1)
    b.q[:, :4 * dim], b.k[:b.nk, :2 * dim] = 0, 0
    b.q[:b.nq, 0:4 * dim:dim], b.k[:b.nk, 0:2 * dim:dim] = 1.0, -1.0
    for s, n in enumerate(lens):
        if n:
            b.k[b.begin[s] + n // 2, :2 * dim] = 0.0  # the largest weight, 1
    b.scale = -math.log(0.5 * (1 + 0.0035))
    value = (1 + torch.arange(2 * dim, device=dev) / (2 * dim)).to(torch.bfloat16)
    b.v[:b.nk, :2 * dim] = value
    b.run_step(G)
    want = value.view(2, 1, dim).expand(2, 2, dim).reshape(-1)
    for s, n in enumerate(lens):
        assert torch.equal(b.out[s, :4 * dim], want if n else torch.zeros_like(want)), s
    b.check(b.want())


@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, True)])
@pytest.mark.parametrize("mask", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_row", [[0, 60, 150, 200], [0, 0, 0, 0], [10, 60, 130, 131], [0, 128, 128, 256], [0, 300, 700, 700]])
def test_rows_outside_the_segments_are_left_alone(G, dev, q_row, dim, mask, cap, bias):
    """A padded batch: fewer rows in the segments than in the table, the rest as they were."""
    b = Batch(dev, [300, 300, 100], [70, 300, 40], 2, 1, dim, seed=11)
    b.q_row = q_row
    sl = slopes_of(2, dev) if bias else None
    b.run(G, mask, None, cap, sl)
    first, last = q_row[0], q_row[-1]
    want = b.reference(mask=mask, cap=cap, slopes=sl)
    R.check(b.out[first:last, :2 * dim], b.lse[first:last], {key: t[first:last] for key, t in want.items()})
    for t in (b.out, b.lse):
        assert (t[:first] == -7).all() and (t[last:] == -7).all()


@pytest.mark.parametrize("part", [0.01, 0.1, 0.199, 0.201, 0.29, 0.599, 0.601, 0.9, 3.0])
@pytest.mark.parametrize("cap", [5.0, 30.0, 55.0, 60.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_capped_scores_to_a_few_roundings(G, dev, cap, dim, part):
    """Rows of one key, whose log-sum-exp is the capped score itself, with the largest score of a block on either side of
    the polynomials' limits (0.2 and 0.6 of the cap)."""
    n = 512
    b = Batch(dev, [1] * n, [1] * n, 1, 1, dim, seed=1)
    b.q[:n, :dim], b.k[:n, :dim] = 0, 0
    b.q[:n, 0] = 1.0
    top = torch.tensor(part * cap).to(torch.bfloat16).float()
    b.k[:n, 0] = (top.to(dev) * torch.linspace(-1, 1, n, device=dev)).to(torch.bfloat16)
    b.k[:n:32, 0] = top.to(dev).to(torch.bfloat16)
    b.scale = 1.0
    dot = b.k[:n, 0].double()
    z = cap * torch.tanh(dot / cap)
    # relative to z, in units of 2^-24: the polynomial 2 (1.2e-7), its coefficients and steps 5, the last product with
    # log2 e 2, the end 1; the tanh by ex2 and rcp (2^-22 and 2^-23 of their own) 6 more. Relative to |z| + cap / 4, as
    # the weight is relative to a quarter of the cap: its exponent, its logarithm (1 step), their sum. And ex2 itself.
    tol = (z.abs() * (10 if part < 0.6 else 16) + (z.abs() + cap / 4) * 4) * 2.0 ** -24 + 2.0 ** -21
    b.run(G, 0, None, cap, None)
    over = (b.lse[:n, 0].double() - z).abs() / tol
    assert float(over.max()) <= 1, float(over.max())
    s = Step(dev, [1] * n, 1, 1, dim, seed=1)
    s.q, s.k, s.scale = b.q, b.k, 1.0
    s.run_step(G, cap)
    over = (s.lse[:n, 0].double() - z).abs() / tol
    assert float(over.max()) <= 1, float(over.max())
