"""Timed cases of the 4-bit projection and of masked attention, with their plain forms.

Operators (gat-tfs_b200/gatb200.py):

  fp4_quantize           rows -> 4-bit floating point (E2M1) with one scale per block
                         MXFP4: blocks of 32, scale 2^k (E8M0)
                         NVFP4: blocks of 16, scale E4M3, and a power of two per row
  fp4_product            out[i][j] = sum_k a[i][k] b[j][k] of two such tables
  masked_attention       softmax attention inside the segments (graphs, documents) of a packed
                         batch, full / causal / prefix mask, tanh cap, bias by distance
  masked_attention_step  the same for one new row per segment over its keys

run() computes a case's operator with elementary torch operations in FP32 (FP64 next to the
rounding borders), or through the library where `own` is true. exact() is the definition in
FP64, written apart.
"""
import math
import sys

import numpy as np
import torch

own = False

MX, NV = "mxfp4", "nvfp4"
BLOCK = {MX: 32, NV: 16}


def _lib():
    if "gat-tfs_b200" not in sys.path:
        sys.path.insert(0, "gat-tfs_b200")
    import gatb200
    return gatb200


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one new node's (token's) features before a 4-bit projection
        {"name": "quantize_one_row", "op": "quantize", "format": NV, "n": 1, "width": 4096, "dtype": "bf16", "pad": 0},
        # the input features of the mid-size graph (169,343 nodes x 128)
        {"name": "quantize_mid_graph", "op": "quantize", "format": MX, "n": 169343, "width": 128, "dtype": "f32", "pad": 0},
        # the input features of the large graph: 100 columns, so every row's last block is short
        {"name": "quantize_large_graph", "op": "quantize", "format": NV, "n": 2449029, "width": 100, "dtype": "f32", "pad": 0},
        # a new node's (token's) projection: the weights' bytes are the cost
        {"name": "product_one_row", "op": "product", "format": NV, "m": 1, "n": 8192, "k": 8192, "out": "bf16"},
        # a few rows against an odd-sized weight
        {"name": "product_few_rows", "op": "product", "format": MX, "m": 37, "n": 5003, "k": 2744, "out": "f32"},
        # the hidden layer of the mid-size graph: 256 -> 8 x 32 for every node
        {"name": "product_hidden_layer", "op": "product", "format": MX, "m": 169343, "n": 256, "k": 256, "out": "bf16"},
        # a wide projection of a long batch
        {"name": "product_wide", "op": "product", "format": NV, "m": 16384, "n": 8192, "k": 8192, "out": "bf16"},
        # many small graphs in one batch, every node sees its own graph; the model's 8 heads x 32
        {"name": "attention_small_graphs", "op": "attention", "heads": 8, "kv_heads": 8, "dim": 32, "segments": 150,
         "rows": 8192, "mask": "full", "cap": 0.0, "bias": False, "lens_seed": 3},
        # documents with a causal mask and capped scores, shared key heads
        {"name": "attention_documents_capped", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "segments": 3,
         "rows": 8192, "mask": "causal", "cap": 50.0, "bias": False, "lens_seed": 5},
        # ragged documents behind prefixes that everyone sees, scores biased by distance
        {"name": "attention_prefix_distance", "op": "attention", "heads": 12, "kv_heads": 12, "dim": 64, "segments": 7,
         "rows": 6001, "mask": "prefix", "cap": 0.0, "bias": True, "lens_seed": 7},
        # one new row over one long history
        {"name": "step_one_long", "op": "step", "heads": 32, "kv_heads": 8, "dim": 128, "segments": 1, "longest": 131072,
         "cap": 0.0, "bias": False, "lens_seed": 9},
        # a serving batch: one new row for each of 48 histories of very different lengths
        {"name": "step_ragged_batch", "op": "step", "heads": 16, "kv_heads": 4, "dim": 64, "segments": 48, "longest": 16384,
         "cap": 30.0, "bias": True, "lens_seed": 11},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "attention", "step"])
    fmt = rng.choice([MX, NV])
    if op == "quantize":
        width = _spread(rng, 1, 16384)
        n = _spread(rng, 1, min(2449029, max(1, 240_000_000 // width)))
        return {"op": op, "format": fmt, "n": n, "width": width, "dtype": rng.choice(["f32", "bf16"]),
                "pad": rng.choice([0, 0, 1, 8])}
    if op == "product":
        n, k = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
        m = _spread(rng, 1, 16384) if rng.random() < 0.6 else _spread(rng, 1, 64)
        return {"op": op, "format": fmt, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "f32"])}
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    dim = rng.choice([16, 32, 40, 64, 96, 128])
    cap, bias = rng.choice([0.0, 30.0, 50.0]), rng.random() < 0.5
    if op == "attention":
        rows = _spread(rng, 1, 8192)
        return {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "segments": min(rows, _spread(rng, 1, 256)),
                "rows": rows, "mask": rng.choice(["full", "causal", "prefix"]), "cap": cap, "bias": bias,
                "lens_seed": rng.randrange(1 << 30)}
    longest = _spread(rng, 1, 131072)
    return {"op": op, "heads": heads, "kv_heads": kv, "dim": dim,
            "segments": _spread(rng, 1, max(1, min(128, 262144 // longest))), "longest": longest, "cap": cap, "bias": bias,
            "lens_seed": rng.randrange(1 << 30)}


def _segment_rows(case):
    """Row pointers [segments + 1] of a packed batch: random cuts, empty segments among them."""
    r = np.random.RandomState(case["lens_seed"])
    cuts = np.sort(r.randint(0, case["rows"] + 1, case["segments"] - 1))
    return np.concatenate([[0], cuts, [case["rows"]]]).astype(np.int64)


def _step_lens(case):
    """Key counts per segment, spread over their logarithm; the first one is the longest."""
    r = np.random.RandomState(case["lens_seed"])
    lens = np.exp(r.uniform(0, math.log(case["longest"] + 0.5), case["segments"])).astype(np.int64)
    lens[0] = case["longest"]
    return np.clip(lens, 1, case["longest"])


def _prefix(case, row):
    """Prefix length per segment: a quarter of it."""
    return (np.diff(row) // 4).astype(np.int64)


def work(case):
    op = case["op"]
    if op == "quantize":
        n, w, b = case["n"], case["width"], BLOCK[case["format"]]
        per_row = w * (4 if case["dtype"] == "f32" else 2) + (w + 1) // 2 + -(-w // b) + 2 * w
        return {"bytes": n * (per_row + (4 if case["format"] == NV else 0)), "flops": 0}
    if op == "product":
        m, n, k, b = case["m"], case["n"], case["k"], BLOCK[case["format"]]
        row = (k + 1) // 2 + -(-k // b) + (4 if case["format"] == NV else 0)
        return {"bytes": (m + n) * row + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * m * n * k}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "attention":
        row = _segment_rows(case)
        lens = np.diff(row).astype(np.float64)
        pairs = lens * lens
        if case["mask"] != "full":
            pre = _prefix(case, row).astype(np.float64) if case["mask"] == "prefix" else 0 * lens
            pairs = lens * (lens + 1) / 2 + np.maximum(pre, 1) * (np.maximum(pre, 1) - 1) / 2
        n = case["rows"]
        return {"bytes": n * (2 * h * d * 2 + 2 * kv * d * 2 + 4 * h), "flops": float(4 * h * d * pairs.sum())}
    total = float(_step_lens(case).sum())
    return {"bytes": total * kv * d * 4 + case["segments"] * (4 * h * d + 4 * h), "flops": 4 * h * d * total}


# ----------------------------------------------- 4-bit tables, in plain operations
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _power(e):
    """2^e in FP32 for whole e in [-127, 127]."""
    bits = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 0x400000))
    return bits.to(torch.int32).view(torch.float32)


def _quantize(x, fmt):
    """(code 0..7 with its sign as 8, scale byte [n][blocks], scale value, row scale) of a table."""
    n, w = x.shape
    b = BLOCK[fmt]
    nb = -(-w // b)
    x = torch.nn.functional.pad(x.float(), (0, nb * b - w)).view(n, nb, b)
    amax = x.abs().amax(-1)
    if fmt == MX:
        # 2^(floor(log2 amax) - 2), so that the largest element lies in [4, 8) and saturates at 6
        e = torch.where(amax > 0, (torch.frexp(amax)[1] - 3).clamp(-127, 127), torch.full((), -127, device=x.device))
        byte, scale, row = (e + 127).to(torch.uint8), _power(e), None
        full = scale.double()
    else:
        # row: the smallest power of two (at least 2^-100) with amax_row / 6 <= 448 * row
        top = amax.amax(-1)
        m, e = torch.frexp(top)
        row = _power(torch.where(top > 0, (e - 11 - (m <= 0.65625).int()).clamp(min=-100), torch.zeros_like(e)))
        fp8 = (amax.double() / (6.0 * row.double()[:, None])).float().to(torch.float8_e4m3fn)
        byte, scale = fp8.view(torch.uint8), fp8.float()
        full = scale.double() * row.double()[:, None]
    y = x.abs().double() / full[..., None]
    y = torch.where(full[..., None] > 0, y, torch.zeros_like(y))
    # ties go to the even code: past the borders of odd index a tie already counts as above
    borders = torch.tensor([v if i % 2 == 0 else math.nextafter(v, 0.0) for i, v in enumerate(_BORDERS)],
                           dtype=torch.float64, device=x.device)
    code = torch.bucketize(y, borders).to(torch.uint8)
    code = torch.where(x < 0, code + 8, code)
    return code, byte, scale, row


def _value_table(device):
    return torch.tensor(_VALUES + tuple(-v for v in _VALUES), dtype=torch.float32, device=device)


def _pack(code, w):
    """Codes [n][blocks][block] -> bytes, two per byte (the even column in the low half), rows of 16-byte pieces."""
    n = code.shape[0]
    code = code.reshape(n, -1)
    ld = (w + 31) // 32 * 16
    code = torch.nn.functional.pad(code, (0, 2 * ld - code.shape[1]))
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _tile_scales(byte):
    """Scale bytes [n][blocks] in tiles of 128 rows x 4 blocks: byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4."""
    n, nb = byte.shape
    r, c = -(-n // 128), -(-nb // 4)
    byte = torch.nn.functional.pad(byte, (0, 4 * c - nb, 0, 128 * r - n))
    return byte.view(r, 4, 32, c, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _untile_scales(flat, n, nb):
    r, c = -(-n // 128), -(-nb // 4)
    return flat.view(r, c, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, c * 4)[:n, :nb]


def _table(x, fmt):
    """A user's 4-bit table of x: codes, tiled scales, row scales."""
    code, byte, _, row = _quantize(x, fmt)
    return {"codes": _pack(code, x.shape[1]), "scales": _tile_scales(byte), "row": row}


def _dequantize(t, fmt, n, w, dtype=torch.float32):
    """The values that a table stands for, without its row scales."""
    b = BLOCK[fmt]
    nb = -(-w // b)
    codes = torch.stack([t["codes"] & 15, t["codes"] >> 4], -1).view(n, -1)[:, :w]
    byte = _untile_scales(t["scales"], n, nb)
    scale = _power(byte.int() - 127) if fmt == MX else byte.contiguous().view(torch.float8_e4m3fn).float()
    v = _value_table(codes.device)[codes.int()].to(dtype)
    return v * scale.to(dtype).repeat_interleave(b, 1)[:, :w]


# -------------------------------------------------------------------- inputs
def _features(g, n, w, dev):
    """Features as layers see them: rows of different size, a few large columns."""
    x = torch.randn(n, w, generator=g, device=dev)
    x *= torch.exp(torch.randn(n, 1, generator=g, device=dev))
    x *= 1 + 15 * (torch.rand(1, w, generator=g, device=dev) > 0.99).float()
    return x


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "quantize":
        n, w, fmt = case["n"], case["width"], case["format"]
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        ldx = w + case["pad"]
        x = torch.zeros(n, ldx, dtype=dtype, device=dev)
        x[:, :w] = _features(g, n, w, dev).to(dtype)
        nb = -(-w // BLOCK[fmt])
        s |= {"x": x, "ldx": ldx, "ldc": (w + 31) // 32 * 16}
        s["codes"] = torch.empty(n, s["ldc"], dtype=torch.uint8, device=dev)
        s["scales"] = torch.empty(-(-n // 128) * -(-nb // 4) * 512, dtype=torch.uint8, device=dev)
        s["row"] = torch.empty(n, device=dev) if fmt == NV else None
        s["values"] = torch.empty(n, w, dtype=torch.bfloat16, device=dev)
        return s
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"] = _table(_features(g, m, k, dev), case["format"])
        s["b"] = _table(torch.randn(n, k, generator=g, device=dev) / math.sqrt(k), case["format"])
        s["out"] = torch.empty(m, n, dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float32, device=dev)
        return s
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "attention":
        row = _segment_rows(case)
        nq = nk = case["rows"]
        s["row"] = torch.from_numpy(row).to(dev)
        s["prefix"] = torch.from_numpy(_prefix(case, row)).to(dev) if case["mask"] == "prefix" else None
    else:
        lens = _step_lens(case)
        nq, nk = case["segments"], int(lens.sum())
        s["begin"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.int64)).to(dev)
        s["length"] = torch.from_numpy(lens).to(dev)
        s["longest"] = int(lens.max())
        s["n_k"] = nk
    rand = lambda n, c: torch.randn(n, c, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    s["q"] = (torch.randn(nq, h * d, generator=g, device=dev) * 2).to(torch.bfloat16)
    s["k"], s["v"] = rand(nk, kv * d), rand(nk, kv * d)
    # slopes 2^(-8 i / heads), i = 1..heads
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=dev) / h).float() if case["bias"] else None
    s["scale"] = 1.0 / math.sqrt(d)
    s["out"] = torch.empty(nq, h * d, dtype=torch.bfloat16, device=dev)
    s["lse"] = torch.empty(nq, h, device=dev)
    if op == "step":
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    return s


# ----------------------------------------------------------------------- run
def _run_own(s):
    G = _lib()
    c = s["case"]
    stream = torch.cuda.current_stream()
    if c["op"] == "quantize":
        G.fp4_quantize(G.MXFP4 if c["format"] == MX else G.NVFP4, c["n"], c["width"], s["x"],
                       G.F32 if c["dtype"] == "f32" else G.BF16, s["ldx"], s["codes"], s["ldc"], s["scales"], s["row"],
                       values=s["values"], v_dtype=G.BF16, ldv=c["width"], stream=stream)
        return {"values": s["values"]} | ({"row": s["row"]} if s["row"] is not None else {})
    if c["op"] == "product":
        a, b = s["a"], s["b"]
        G.fp4_product(G.MXFP4 if c["format"] == MX else G.NVFP4, c["m"], c["n"], c["k"],
                      a["codes"], a["codes"].shape[1], a["scales"], a["row"],
                      b["codes"], b["codes"].shape[1], b["scales"], b["row"],
                      s["out"], G.BF16 if c["out"] == "bf16" else G.F32, c["n"], stream=stream)
        return s["out"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "attention":
        mask = {"full": G.MASK_FULL, "causal": G.MASK_CAUSAL, "prefix": G.MASK_PREFIX}[c["mask"]]
        G.masked_attention(h, kv, d, c["segments"], c["rows"], c["rows"], s["row"], s["row"], mask, s["prefix"],
                           s["q"], h * d, s["k"], kv * d, s["v"], kv * d, s["scale"], c["cap"], s["slopes"],
                           s["out"], h * d, s["lse"], stream=stream)
    else:
        G.masked_attention_step(h, kv, d, c["segments"], s["n_k"], s["begin"], s["length"],
                                s["q"], h * d, s["k"], kv * d, s["v"], kv * d, s["scale"], c["cap"], s["slopes"],
                                s["out"], h * d, s["lse"], s["workspace"], s["workspace"].numel(), stream=stream)
    return {"out": s["out"], "lse": s["lse"]}


def _softmax_rows(score, seen):
    """(weights, log of the sum) over the last axis; rows that see nothing get zeros and -inf."""
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    return p.div_(torch.where(total > 0, total, torch.ones_like(total))), lse


def _score(dot, c, scale, slopes, distance):
    """dot [heads][...]: scale, cap, bias by distance."""
    s = dot.mul_(scale)
    if c["cap"] > 0:
        s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
    if slopes is not None:
        s = s.sub_(slopes.view(-1, 1, 1) * distance)
    return s


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "quantize":
        w = c["width"]
        code, _, scale, row = _quantize(s["x"][:, :w], c["format"])
        v = _value_table(code.device)[code.int()] * scale[..., None]
        v = v.view(c["n"], -1)[:, :w]
        if row is not None:
            return {"values": (v * row[:, None]).to(torch.bfloat16), "row": row}
        return {"values": v.to(torch.bfloat16)}
    if c["op"] == "product":
        out = _dequantize(s["a"], c["format"], c["m"], c["k"]) @ _dequantize(s["b"], c["format"], c["n"], c["k"]).t()
        if s["a"]["row"] is not None:
            out *= s["a"]["row"][:, None]
            out *= s["b"]["row"][None, :]
        return out.to(s["out"].dtype)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "attention":
        n, row = c["rows"], s["row"]
        pos = torch.arange(n, device=row.device)
        seg = torch.searchsorted(row, pos, right=True) - 1
        end = row[seg + 1]
        if c["mask"] != "full":
            end = torch.minimum(end, pos + 1)
        if c["mask"] == "prefix":
            end = torch.maximum(end, row[seg] + s["prefix"][seg])
        seen = (pos[None, :] >= row[seg][:, None]) & (pos[None, :] < end[:, None])
        q = s["q"].float().view(n, h, d).transpose(0, 1)
        k = s["k"].float().view(n, kv, d).transpose(0, 1).repeat_interleave(h // kv, 0)
        v = s["v"].float().view(n, kv, d).transpose(0, 1).repeat_interleave(h // kv, 0)
        far = (pos[:, None] - pos[None, :]).abs().float()[None] if c["bias"] else None
        p, lse = _softmax_rows(_score(torch.bmm(q, k.transpose(1, 2)), c, s["scale"], s["slopes"], far), seen)
        out = torch.bmm(p, v).transpose(0, 1).reshape(n, h * d)
        return {"out": out.to(torch.bfloat16), "lse": lse.t().contiguous()}
    b, length = c["segments"], s["length"]
    at = torch.arange(s["longest"], device=length.device)
    seen = at[None, :] < length[:, None]
    idx = (s["begin"][:, None] + at[None, :]).clamp(max=s["n_k"] - 1)
    group = h // kv
    k = s["k"][idx].float().view(b, -1, kv, d).permute(0, 2, 3, 1).reshape(b * kv, d, -1)
    v = s["v"][idx].float().view(b, -1, kv, d).transpose(1, 2).reshape(b * kv, -1, d)
    q = s["q"].float().view(b * kv, group, d)
    far = (length[:, None] - 1 - at[None, :]).abs().float()[None] if c["bias"] else None
    dot = torch.bmm(q, k).view(b, h, -1).transpose(0, 1)
    p, lse = _softmax_rows(_score(dot, c, s["scale"], s["slopes"], far), seen[None])
    out = torch.bmm(p.transpose(0, 1).reshape(b * kv, group, -1), v).view(b, h * d)
    return {"out": out.to(torch.bfloat16), "lse": lse.t().contiguous()}


# --------------------------------------------------------------------- exact
def _floor_log2(v):
    """floor(log2 v) for v > 0: log2 is rounded, so one step either way is put right by comparing."""
    e = torch.floor(torch.log2(v))
    e = torch.where(torch.exp2(e + 1) <= v, e + 1, e)
    return torch.where(torch.exp2(e) > v, e - 1, e)


def _exact_quantize(x, fmt):
    """Values and row scales by the definition: the nearest of the 15 values to x / (block scale * row scale), ties to
    the one whose code is even, in FP64."""
    n, w = x.shape
    b = BLOCK[fmt]
    nb = -(-w // b)
    x = torch.nn.functional.pad(x.double(), (0, nb * b - w)).view(n, nb, b)
    top = x.abs().amax(-1, keepdim=True)
    row = torch.ones(n, 1, 1, dtype=torch.float64, device=x.device)
    if fmt == MX:
        step = torch.exp2((_floor_log2(top.clamp(min=2.0 ** -149)) - 2).clamp(-127, 127))
    else:
        peak = top.amax(1, keepdim=True)
        e = torch.ceil(torch.log2(peak.clamp(min=2.0 ** -149) / 2688.0))
        e = torch.where(peak <= 2688.0 * torch.exp2(e - 1), e - 1, e)  # log2 is rounded: one step either way
        e = torch.where(peak > 2688.0 * torch.exp2(e), e + 1, e).clamp(min=-100)
        row = torch.where(peak > 0, torch.exp2(e), row)
        want = top / (6.0 * row)
        # nearest E4M3: steps of 2^(exponent - 3), 2^-9 below 2^-6; round() takes ties to even
        unit = torch.exp2(_floor_log2(want.clamp(min=2.0 ** -6)) - 3)
        step = torch.round(want / unit) * unit
    full = step * row
    y = torch.where(full > 0, x.abs() / torch.where(full > 0, full, torch.ones_like(full)), torch.zeros_like(x))
    y = y.clamp(max=6.0)
    unit = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = torch.round(y / unit) * unit  # the code's last bit is the last bit of y / unit
    return (torch.sign(x) * y * full).view(n, -1)[:, :w], row.view(n)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "quantize":
        parts = [_exact_quantize(x, c["format"]) for x in s["x"][:, :c["width"]].split(1 << 19)]
        v = torch.cat([p[0].to(torch.float32) for p in parts]).double()  # the values have few bits
        return {"values": v} | ({"row": torch.cat([p[1] for p in parts])} if c["format"] == NV else {})
    if c["op"] == "product":
        a = _dequantize(s["a"], c["format"], c["m"], c["k"], torch.float64)
        b = _dequantize(s["b"], c["format"], c["n"], c["k"], torch.float64)
        if s["a"]["row"] is not None:
            a, b = a * s["a"]["row"].double()[:, None], b * s["b"]["row"].double()[:, None]
        return torch.matmul(a, b.t())
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    nq = s["q"].shape[0]
    out = torch.zeros(nq, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((nq, h), -math.inf, dtype=torch.float64, device="cuda")
    if c["op"] == "attention":
        bounds = [(int(x), int(y), int(x), int(y)) for x, y in zip(s["row"][:-1], s["row"][1:])]
    else:
        bounds = [(i, i + 1, int(x), int(x) + int(y)) for i, (x, y) in enumerate(zip(s["begin"], s["length"]))]
    for i, (q0, q1, k0, k1) in enumerate(bounds):
        if q1 == q0 or k1 == k0:
            continue
        pre = int(s["prefix"][i]) if s.get("prefix") is not None else 0
        for r0 in range(q0, q1, 2048):
            r1 = min(q1, r0 + 2048)
            iq = torch.arange(r0 - q0 + (k1 - k0) - (q1 - q0), r1 - q0 + (k1 - k0) - (q1 - q0), device="cuda")
            jk = torch.arange(k1 - k0, device="cuda")
            seen = torch.ones(r1 - r0, k1 - k0, dtype=torch.bool, device="cuda")
            if c["op"] == "attention" and c["mask"] != "full":
                seen = (jk[None, :] <= iq[:, None]) | (jk[None, :] < pre)
            for head in range(h):
                kh = head // (h // kv)
                z = s["q"][r0:r1, head * d:(head + 1) * d].double() @ s["k"][k0:k1, kh * d:(kh + 1) * d].double().t()
                z = z * s["scale"]
                if c["cap"] > 0:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][head].double() * (iq[:, None] - jk[None, :]).abs().double()
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                lse[r0:r1, head] = torch.logsumexp(z, -1)
                out[r0:r1, head] = torch.softmax(z, -1) @ s["v"][k0:k1, kh * d:(kh + 1) * d].double()
    return {"out": out.view(nq, h * d), "lse": lse}
