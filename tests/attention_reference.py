"""Masked attention in torch FP64, from the definition, with the error that BF16
weights, FP32 scores and a BF16 output allow."""
import math

import torch

FULL, CAUSAL, PREFIX = 0, 1, 2


def attention(q, k, v, q_row, k_row, heads, kv_heads, dim, scale, cap=0.0, slopes=None, mask=FULL, prefix=None):
    """q [n_q][heads*dim], k / v [n_k][kv_heads*dim], row pointers as lists ->
    dict(out, lse, tol, lse_tol): FP64, tolerances per element."""
    dev = q.device
    n_q = q.shape[0]
    out = torch.zeros(n_q, heads, dim, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((n_q, heads), -math.inf, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros_like(lse)
    for s in range(len(q_row) - 1):
        q0, q1, k0, k1 = q_row[s], q_row[s + 1], k_row[s], k_row[s + 1]
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        pos = torch.arange(lq, device=dev) + (lk - lq)
        key = torch.arange(lk, device=dev)
        seen = torch.ones(lq, lk, dtype=torch.bool, device=dev)
        if mask != FULL:
            seen = key[None, :] <= pos[:, None]
        if mask == PREFIX:
            seen = seen | (key[None, :] < prefix[s])
        any_ = seen.any(1)
        for h in range(heads):
            g = h // (heads // kv_heads)
            a = q[q0:q1, h * dim:(h + 1) * dim].double()
            b = k[k0:k1, g * dim:(g + 1) * dim].double()
            c = v[k0:k1, g * dim:(g + 1) * dim].double()
            dot = a @ b.t() * scale
            z = cap * torch.tanh(dot / cap) if cap > 0 else dot
            # FP32: dim products and sums of the dot, then a handful of roundings of values up to z's size; a
            # tanh within 1.3e-6 < 2^-19 of itself (tanh' <= 1: the dot's error grows no further)
            err = (a.abs() @ b.abs().t()) * scale * (dim + 4) * 2.0 ** -24
            if slopes is not None:
                far = (pos[:, None] - key[None, :]).abs().double()
                z = z - slopes[h].double() * far
                err = err + slopes[h].double().abs() * far * 2.0 ** -21
            err = err + z.abs() * 2.0 ** (-19 if cap > 0 else -21) + 2.0 ** -20
            z = torch.where(seen, z, torch.full_like(z, -math.inf))
            err = torch.where(seen, err, torch.zeros_like(err))
            top = z.amax(1, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            p = torch.exp(z - top)
            p = torch.where(seen, p, torch.zeros_like(p))
            total = p.sum(1, keepdim=True)
            w = p / torch.where(total > 0, total, torch.ones_like(total))
            cc = torch.where(torch.isfinite(c), c, torch.zeros_like(c))
            o = w @ cc
            # values that are not finite reach the rows that see them, and only those
            for j in (~torch.isfinite(c).all(1)).nonzero().flatten().tolist():
                x = torch.where(torch.isfinite(c[j]), torch.zeros_like(c[j]), c[j])
                o = torch.where(seen[:, j:j + 1], o + w[:, j:j + 1] * x, o)
            # weights: half a BF16 step (2^-8) and the scores' errors, once in the sum and once in its norm
            rel = 2.0 ** -8 + 2 * err.amax(1, keepdim=True)
            first = rel * (w @ cc.abs())
            oh = torch.where(torch.isfinite(o), o, torch.zeros_like(o))
            out[q0:q1, h] = torch.where(any_[:, None], o, torch.zeros_like(o))
            tol[q0:q1, h] = first + 2.0 ** -8 * (oh.abs() + first) + 2.0 ** -60
            lse[q0:q1, h] = torch.where(any_, (top + total.log()).squeeze(1), torch.full_like(any_, -math.inf, dtype=torch.float64))
            ls = torch.where(torch.isfinite(lse[q0:q1, h]), lse[q0:q1, h], torch.zeros_like(lse[q0:q1, h]))
            lse_tol[q0:q1, h] = err.amax(1) + 2.0 ** -20 * (1 + ls.abs()) + lk * 2.0 ** -24
    return dict(out=out.view(n_q, heads * dim), lse=lse, tol=tol.view(n_q, heads * dim), lse_tol=lse_tol)


def check(got_out, got_lse, want):
    o, w = got_out.double(), want["out"]
    fin = torch.isfinite(w)
    assert torch.equal(torch.isnan(o), torch.isnan(w))
    assert torch.equal(o[~fin & ~torch.isnan(w)], w[~fin & ~torch.isnan(w)])
    over = ((o - w).abs() / want["tol"].clamp(min=1e-300))[fin]
    assert over.numel() == 0 or float(over.max()) <= 1, float(over.max())
    if got_lse is not None:
        l, x = got_lse.double(), want["lse"]
        inf = torch.isinf(x)
        assert torch.equal(l[inf], x[inf])
        d = ((l - x).abs() / want["lse_tol"].clamp(min=1e-300))[~inf & ~torch.isnan(x)]
        assert d.numel() == 0 or float(d.max()) <= 1, float(d.max())
