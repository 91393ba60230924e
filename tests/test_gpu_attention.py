"""Masked attention on the GPU against its FP64 definition (attention_reference.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import attention_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    import gatb200
    return gatb200


def rows(lens):
    return [int(x) for x in np.concatenate([[0], np.cumsum(lens)])]


def u64(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


class Batch:
    """Inputs of one call; every table is a slice of a wider one, with NaN around it."""

    def __init__(self, dev, q_lens, k_lens, heads, kv, dim, seed=0, pad=0, qscale=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.heads, self.kv, self.dim = dev, heads, kv, dim
        self.q_row, self.k_row = rows(q_lens), rows(k_lens)
        self.nq, self.nk = self.q_row[-1], self.k_row[-1]

        def make(n, w, s=1.0):
            t = torch.full((n + 3, w + pad), float("nan"), dtype=torch.bfloat16, device=dev)
            t[:n, :w] = (torch.randn(n, w, generator=g, device=dev) * s).to(torch.bfloat16)
            return t
        self.q, self.k, self.v = make(self.nq, heads * dim, qscale), make(self.nk, kv * dim), make(self.nk, kv * dim)
        self.out = torch.full((self.nq + 3, heads * dim + pad), -7.0, dtype=torch.bfloat16, device=dev)
        self.lse = torch.full((self.nq + 3, heads), -7.0, device=dev)
        self.scale = dim ** -0.5
        self.pad = pad

    def ld(self, h):
        return h * self.dim + self.pad

    def reference(self, **kw):
        return R.attention(self.q[:self.nq, :self.heads * self.dim], self.k[:self.nk, :self.kv * self.dim],
                           self.v[:self.nk, :self.kv * self.dim], self.q_row, self.k_row, self.heads, self.kv, self.dim,
                           self.scale, **kw)

    def run(self, G, mask=0, prefix=None, cap=0.0, slopes=None, stream=None, lse=True):
        h, kv, d = self.heads, self.kv, self.dim
        G.masked_attention(h, kv, d, len(self.q_row) - 1, self.nq, self.nk, u64(self.q_row, self.dev),
                           u64(self.k_row, self.dev), mask, None if prefix is None else u64(prefix, self.dev),
                           self.q, self.ld(h), self.k, self.ld(kv), self.v, self.ld(kv), self.scale, cap, slopes,
                           self.out, self.ld(h), self.lse if lse else None, stream=stream)
        torch.cuda.synchronize()
        G.check_device()

    def check(self, want, lse=True):
        w = self.heads * self.dim
        R.check(self.out[:self.nq, :w], self.lse[:self.nq] if lse else None, want)
        assert (self.out[self.nq:] == -7).all() and (self.out[:, w:] == -7).all()
        assert (self.lse[self.nq:] == -7).all() and (lse or (self.lse == -7).all())


def slopes_of(heads, dev):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, device=dev) / heads).float()


LENS = [[1], [2], [127], [128], [129], [300], [1, 1, 1], [5, 0, 20, 128, 1, 77], [0, 0, 3, 0], [513, 2],
        [40] * 30, [255, 256, 257, 1]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("mask", [0, 1, 2])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True), (30.0, True)])
def test_masks_caps_and_biases(G, dev, lens, mask, cap, bias):
    b = Batch(dev, lens, lens, 4, 2, 64, seed=len(lens), qscale=3.0)
    prefix = [n // 3 for n in lens] if mask == 2 else None
    sl = slopes_of(4, dev) if bias else None
    b.run(G, mask, prefix, cap, sl)
    b.check(b.reference(cap=cap, slopes=sl, mask=mask, prefix=prefix))


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (6, 2), (4, 1)])
def test_dims_heads_and_strides(G, dev, dim, heads, kv):
    b = Batch(dev, [70, 200, 33], [70, 200, 33], heads, kv, dim, seed=dim, pad=8 * (dim % 3))
    b.run(G, 1, None, 0.0, None)
    b.check(b.reference(mask=1))


@pytest.mark.parametrize("mask", [0, 1, 2])
@pytest.mark.parametrize("q_lens,k_lens", [([3, 50, 1], [400, 20, 700]), ([200, 10], [100, 0]), ([0, 5, 0], [128, 130, 5]),
                                           ([300], [1]), ([1], [3000]), ([130, 130], [0, 0])])
def test_rows_and_keys_of_different_counts(G, dev, mask, q_lens, k_lens):
    # a causal row before the first key sees nothing: zeros and -inf
    b = Batch(dev, q_lens, k_lens, 2, 1, 128, seed=3)
    prefix = [min(5, n) for n in k_lens] if mask == 2 else None
    sl = slopes_of(2, dev)
    b.run(G, mask, prefix, 0.0, sl)
    b.check(b.reference(mask=mask, prefix=prefix, slopes=sl))


def test_empty_batches(G, dev):
    b = Batch(dev, [0, 0], [4, 5], 2, 2, 32)
    b.run(G)
    assert (b.out == -7).all()
    b = Batch(dev, [4, 3], [0, 0], 2, 2, 32)
    b.run(G, 1)
    assert (b.out[:7] == 0).all() and torch.isinf(b.lse[:7]).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), -3.3e38])
@pytest.mark.parametrize("mask", [0, 1, 2])
def test_what_is_masked_never_arrives(G, dev, value, mask):
    lens = [30, 100, 60, 200, 129]
    b = Batch(dev, lens, lens, 2, 2, 64, seed=5)
    clean = Batch(dev, lens, lens, 2, 2, 64, seed=5)
    clean.run(G, mask, [0] * 5 if mask == 2 else None)
    b.k[40, :64] = value     # in segment 1
    b.v[45, 3] = value
    b.v[300, 70:90] = value  # in segment 3, late: its earlier rows do not see it under a causal mask
    b.q[200, 5] = value      # one row of segment 3
    b.run(G, mask, [0] * 5 if mask == 2 else None)
    other = [i for s in (0, 2, 4) for i in range(b.q_row[s], b.q_row[s + 1])]
    assert torch.equal(b.out[other], clean.out[other]) and torch.equal(b.lse[other], clean.lse[other])
    if mask:
        early = [i for i in range(b.q_row[1], 40)] + [i for i in range(b.q_row[3], 300) if i != 200]
        assert torch.equal(b.out[early], clean.out[early]) and torch.equal(b.lse[early], clean.lse[early])


def test_values_that_are_not_finite_reach_their_readers(G, dev):
    lens = [30, 100, 600]
    for mask in (0, 1):
        b = Batch(dev, lens, lens, 2, 1, 72, seed=8)
        for row, col, x in [(10, 0, float("inf")), (50, 71, -float("inf")), (51, 71, float("inf")), (300, 17, float("nan")),
                            (640, 64, float("inf"))]:
            b.v[row, col] = x
        b.run(G, mask)
        b.check(b.reference(mask=mask))


def test_large_scores(G, dev):
    # maxima that keep growing (every block moves the reference) and rows that drown the rest
    b = Batch(dev, [700, 130], [700, 130], 2, 2, 64, seed=2, qscale=40.0)
    b.k[:830, :128] *= torch.linspace(0.1, 3, 830, device=dev)[:, None].to(torch.bfloat16)
    for cap in (0.0, 50.0):
        for mask in (0, 1):
            b.run(G, mask, None, cap, None)
            b.check(b.reference(mask=mask, cap=cap))


@pytest.mark.parametrize("cap", [0.0, 20.0, 60.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("mask", [0, 1, 2])
def test_slopes_of_either_sign(G, dev, cap, dim, mask):
    sl = torch.tensor([1.5, -0.75, 0.0, -2.0], device=dev)
    for q_lens, k_lens in (([400, 30, 1], [400, 30, 1]), ([40, 300], [700, 20])):
        b = Batch(dev, q_lens, k_lens, 4, 2, dim, seed=9)
        prefix = [n // 2 for n in k_lens] if mask == 2 else None
        b.run(G, mask, prefix, cap, sl)
        b.check(b.reference(mask=mask, prefix=prefix, cap=cap, slopes=sl))
    s = Step(dev, [700, 1, 33], 4, 2, dim, seed=2)
    s.run_step(G, cap, sl)
    s.check(s.want(cap=cap, slopes=sl))


@pytest.mark.parametrize("cap", [1e-4, 0.3, 5.0, 56.0, 1000.0, 1e6, 1e20])
@pytest.mark.parametrize("dim", [64, 128])
def test_caps_far_from_the_scores(G, dev, cap, dim):
    # caps that all scores exceed, caps that no score comes near, and both sides of the polynomials' ranges
    lens = [300, 150]
    for bias in (False, True):
        sl = slopes_of(2, dev) if bias else None
        b = Batch(dev, lens, lens, 2, 1, dim, seed=4, qscale=6.0)
        b.run(G, 1, None, cap, sl)
        b.check(b.reference(mask=1, cap=cap, slopes=sl))
        s = Step(dev, lens, 2, 1, dim, seed=4)
        s.run_step(G, cap, sl)
        s.check(s.want(cap=cap, slopes=sl))


def test_fused_table_and_streams(G, dev):
    """Q, K and V as column ranges of one projection's output, on a stream of its own."""
    heads, kv, dim, n = 4, 2, 32, 333
    w = (heads + 2 * kv) * dim
    h = torch.randn(n, w, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    out = torch.empty(n, heads * dim, dtype=torch.bfloat16, device=dev)
    row = [0, 100, 101, 333]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    e = 2  # bytes of an element
    G.masked_attention(heads, kv, dim, 3, n, n, u64(row, dev), u64(row, dev), 1, None, h, w,
                       h.data_ptr() + heads * dim * e, w, h.data_ptr() + (heads + kv) * dim * e, w, dim ** -0.5, 0.0, None,
                       out, heads * dim, None, stream=st)
    torch.cuda.synchronize()
    q, k, v = h.split([heads * dim, kv * dim, kv * dim], 1)
    R.check(out, None, R.attention(q, k, v, row, row, heads, kv, dim, dim ** -0.5, mask=1))


def test_captured_call_follows_its_inputs(G, dev):
    lens = [60, 90, 150]
    b = Batch(dev, lens, lens, 2, 2, 64, seed=4)
    qr, kr = u64(b.q_row, dev), u64(b.k_row, dev)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        G.masked_attention(2, 2, 64, 3, b.nq, b.nk, qr, kr, 1, None, b.q, 128, b.k, 128, b.v, 128, b.scale, 0.0, None,
                           b.out, 128, b.lse, stream=st)
    for lens in ([60, 90, 150], [1, 298, 1], [0, 300, 0]):
        b.q_row = b.k_row = rows(lens)
        qr.copy_(u64(b.q_row, dev))
        kr.copy_(u64(b.q_row, dev))
        b.q[:300, :128] = torch.randn(300, 128, device=dev).to(torch.bfloat16)
        graph.replay()
        torch.cuda.synchronize()
        b.check(b.reference(mask=1))


# ------------------------------------------------------------- one new row
class Step(Batch):
    def __init__(self, dev, lens, heads, kv, dim, seed=0, pad=0, gap=0):
        super().__init__(dev, [1] * len(lens), [n + gap for n in lens], heads, kv, dim, seed, pad, qscale=2.0)
        self.lens = list(lens)
        self.begin = [self.k_row[i] + gap for i in range(len(lens))]
        self.work = None

    def run_step(self, G, cap=0.0, slopes=None, lse=True, stream=None):
        h, kv, d, n = self.heads, self.kv, self.dim, len(self.lens)
        if self.work is None:
            self.work = torch.full((G.masked_attention_step_workspace(h, d, n),), 0xFF, dtype=torch.uint8, device=self.dev)
        G.masked_attention_step(h, kv, d, n, self.nk, u64(self.begin, self.dev), u64(self.lens, self.dev), self.q,
                                self.ld(h), self.k, self.ld(kv), self.v, self.ld(kv), self.scale, cap, slopes, self.out,
                                self.ld(h), self.lse if lse else None, self.work, self.work.numel(), stream=stream)
        torch.cuda.synchronize()

    def want(self, **kw):
        w, q = self.kv * self.dim, self.q[:self.nq, :self.heads * self.dim]
        parts = [R.attention(q[i:i + 1], self.k[b:b + n, :w], self.v[b:b + n, :w], [0, 1], [0, n], self.heads, self.kv,
                             self.dim, self.scale, **kw) for i, (b, n) in enumerate(zip(self.begin, self.lens))]
        return {key: torch.cat([p[key] for p in parts]) for key in parts[0]}


STEPS = [[1], [0], [31], [32], [33], [127, 0, 1], [128], [129], [5000], [1, 2, 3, 4, 5, 0, 700], [300] * 40, [20000, 1, 17],
         [1] * 300, [0, 0, 9], [64, 128, 256, 512, 1024]]


@pytest.mark.parametrize("lens", STEPS)
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 1, 128), (32, 2, 40)])
def test_step_matches(G, dev, lens, heads, kv, dim):
    b = Step(dev, lens, heads, kv, dim, seed=len(lens))
    b.run_step(G)
    b.check(b.want())


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 48, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (15.0, False), (0.0, True), (25.0, True)])
def test_step_dims_caps_and_biases(G, dev, dim, cap, bias):
    b = Step(dev, [50, 700, 3], 6, 3, dim, seed=dim, pad=16, gap=5)
    sl = slopes_of(6, dev) if bias else None
    b.run_step(G, cap, sl, lse=not bias)
    b.check(b.want(cap=cap, slopes=sl), lse=not bias)


def test_step_many_cut_segments_odd_heads(G, dev):
    b = Step(dev, [300, 0, 517] * 34, 6, 3, 64, seed=3)
    b.run_step(G)
    b.check(b.want())


@pytest.mark.parametrize("n", [128, 129, 511, 512, 513, 1500])
def test_step_segment_counts(G, dev, n):
    b = Step(dev, [(7 * i) % 5 * ((i % 11) + 1) for i in range(n - 1)] + [900], 4, 2, 32, seed=n)
    b.run_step(G)
    b.check(b.want())


@pytest.mark.parametrize("heads,kv,dim,n", [(16, 4, 128, 300), (16, 16, 64, 90), (8, 2, 40, 777), (32, 1, 128, 200)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (25.0, True)])
def test_step_many_short_segments(G, dev, heads, kv, dim, n, cap, bias):
    lens = [(13 * i) % 97 for i in range(n)]
    lens[n // 2] = 3000  # one that many runs share
    b = Step(dev, lens, heads, kv, dim, seed=n, gap=1)
    sl = slopes_of(heads, dev) if bias else None
    b.run_step(G, cap, sl)
    b.check(b.want(cap=cap, slopes=sl))


def test_step_equals_the_last_row(G, dev):
    lens = [200, 1, 77]
    b = Batch(dev, lens, lens, 4, 2, 64, seed=1)
    b.run(G, 1, None, 10.0, slopes_of(4, dev))
    s = Step(dev, lens, 4, 2, 64)
    last = [r - 1 for r in b.q_row[1:]]
    s.q[:3, :256], s.k, s.v = b.q[last, :256], b.k, b.v
    s.run_step(G, 10.0, slopes_of(4, dev))
    s.check(s.want(cap=10.0, slopes=slopes_of(4, dev)))
    assert (s.lse[:3] - b.lse[last]).abs().max() < 1e-4


def test_step_overlapping_and_cut_segments(G, dev):
    b = Step(dev, [400], 4, 2, 64, seed=6)
    b.q = torch.randn(8, 256, device=dev).to(torch.bfloat16)
    b.out, b.lse = b.out[:1].repeat(8, 1), b.lse[:1].repeat(8, 1)
    b.nq, b.lens, b.begin = 5, [400, 100, 300, 10, 0], [0, 0, 100, 390, 17]
    want = b.want()
    b.lens[2], b.lens[3], b.lens[4] = 1 << 40, 11, 5  # reach past the table: cut off (300, 10), and
    b.begin[4] = 401                                  # a segment behind it: no keys
    b.run_step(G)
    b.check(want)


def test_step_many_segments_over_the_same_keys(G, dev):
    b = Step(dev, [700], 4, 1, 64, seed=8)
    b.q = torch.randn(43, 256, device=dev).to(torch.bfloat16)
    b.out, b.lse = b.out[:1].repeat(43, 1), b.lse[:1].repeat(43, 1)
    b.nq, b.lens, b.begin = 40, [700 - 3 * i for i in range(40)], [i for i in range(40)]
    b.run_step(G, 20.0)
    b.check(b.want(cap=20.0))


def test_step_non_finite_neighbours(G, dev):
    lens = [40, 60, 129]
    a, b = Step(dev, lens, 4, 2, 64, seed=7, gap=3), Step(dev, lens, 4, 2, 64, seed=7, gap=3)
    for t in (b.k, b.v):  # the gaps between the segments
        for s in range(3):
            t[b.k_row[s]:b.k_row[s] + 3] = float("nan")
    a.run_step(G)
    b.run_step(G)
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)
    b.v[b.begin[2] + 128, 1] = float("inf")
    b.k[b.begin[1] + 7] = float("nan")
    b.run_step(G)
    assert torch.equal(a.out[0], b.out[0]) and torch.isnan(b.out[1]).all()
    assert torch.isinf(b.out[2, 1]) and torch.isfinite(b.out[2, 2:64]).all()


def test_step_replays_with_new_lengths_and_own_workspaces(G, dev):
    lens = [3000, 10, 500]
    runs = []
    for seed in (1, 2):
        b = Step(dev, lens, 8, 2, 128, seed=seed)
        b.work = torch.empty(G.masked_attention_step_workspace(8, 128, 3), dtype=torch.uint8, device=dev)
        b.dbegin, b.dlen = u64(b.begin, dev), u64(b.lens, dev)
        st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            G.masked_attention_step(8, 2, 128, 3, b.nk, b.dbegin, b.dlen, b.q, 1024, b.k, 256, b.v, 256, b.scale, 0.0,
                                    None, b.out, 1024, b.lse, b.work, b.work.numel(), stream=st)
        runs.append((b, graph, torch.cuda.Stream()))
    for new in (lens, [1, 10, 0], [2500, 7, 499]):
        for b, graph, st in runs:
            b.lens = list(new)
            b.dlen.copy_(u64(new, dev))
        torch.cuda.synchronize()
        for b, graph, st in runs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for b, *_ in runs:
            b.check(b.want())


def test_step_offsets_past_32_bits(G, dev):
    # a table of more than 2^31 elements, the segment at its end
    ld, n = 2048, 1_050_000
    k = torch.zeros(n, ld, dtype=torch.bfloat16, device=dev)
    v = torch.zeros(n, ld, dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    tail = 300
    k[-tail:] = torch.randn(tail, ld, generator=g, device=dev).to(torch.bfloat16)
    v[-tail:] = torch.randn(tail, ld, generator=g, device=dev).to(torch.bfloat16)
    q = torch.randn(1, ld, generator=g, device=dev).to(torch.bfloat16)
    out = torch.empty(1, ld, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(1, 16, device=dev)
    work = torch.empty(G.masked_attention_step_workspace(16, 128, 1), dtype=torch.uint8, device=dev)
    G.masked_attention_step(16, 16, 128, 1, n, u64([n - tail], dev), u64([tail], dev), q, ld, k, ld, v, ld, 128 ** -0.5,
                            0.0, None, out, ld, lse, work, work.numel())
    R.check(out, lse, R.attention(q, k[-tail:], v[-tail:], [0, 1], [0, tail], 16, 16, 128, 128 ** -0.5))
    # the tile kernel at the same place: two segments, the first one without rows
    qr, kr = u64([0, 0, 1], dev), u64([0, n - tail, n], dev)
    G.masked_attention(16, 16, 128, 2, 1, n, qr, kr, 1, None, q, ld, k, ld, v, ld, 128 ** -0.5, 0.0, None, out, ld, lse)
    torch.cuda.synchronize()
    R.check(out, lse, R.attention(q, k[-tail:], v[-tail:], [0, 1], [0, tail], 16, 16, 128, 128 ** -0.5))


def test_quantised_projection_feeds_attention(G, dev):
    """The operators as one layer: features to 4 bits, projected to Q | K | V, attention inside each graph."""
    n, k, heads, kv, dim = 500, 256, 8, 8, 32
    w = (heads + 2 * kv) * dim
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(n, k, generator=g, device=dev).to(torch.bfloat16)
    wt = torch.randn(w, k, generator=g, device=dev) / 16
    t = {}
    for name, a, rows_, dt in (("x", x, n, G.BF16), ("w", wt, w, G.F32)):
        codes = torch.empty(rows_, G.fp4_ld(k), dtype=torch.uint8, device=dev)
        scales = torch.empty(G.fp4_scale_bytes(G.NVFP4, rows_, k), dtype=torch.uint8, device=dev)
        r = torch.empty(rows_, device=dev)
        vals = torch.empty(rows_, k, device=dev)
        G.fp4_quantize(G.NVFP4, rows_, k, a, dt, k, codes, G.fp4_ld(k), scales, r, vals, G.F32, k)
        t[name] = (codes, scales, r, vals)
    h = torch.empty(n, w, dtype=torch.bfloat16, device=dev)
    (xc, xs, xr, xv), (wc, ws, wr, wv) = t["x"], t["w"]
    G.fp4_product(G.NVFP4, n, w, k, xc, G.fp4_ld(k), xs, xr, wc, G.fp4_ld(k), ws, wr, h, G.BF16, w)
    want = xv.double() @ wv.double().t()
    mag = xv.double().abs() @ wv.double().abs().t()
    assert ((h.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * k * 2.0 ** -24).all()
    row = rows([20, 100, 7, 373])
    out = torch.empty(n, heads * dim, dtype=torch.bfloat16, device=dev)
    G.masked_attention(heads, kv, dim, 4, n, n, u64(row, dev), u64(row, dev), 0, None, h, w,
                       h.data_ptr() + 2 * heads * dim, w, h.data_ptr() + 2 * (heads + kv) * dim, w, dim ** -0.5, 30.0, None,
                       out, heads * dim)
    torch.cuda.synchronize()
    q, kk, v = h.split([heads * dim, kv * dim, kv * dim], 1)
    R.check(out, None, R.attention(q, kk, v, row, row, heads, kv, dim, dim ** -0.5, cap=30.0))
