"""Paged-cache operators restated on the CPU in 64 bits (test oracle only).

Written from the definitions: a sequence's cache is gathered position by
position, every row is computed on its own. Alongside the value, attention()
returns what error bounds are made of: sum p |v| per output element, the
largest |score| terms and the number of positions of every row.
"""

from __future__ import annotations

import math

import torch


def sequences(rows: int, lens, starts):
    """(sequence, first row, end row, cache length) of every sequence with rows."""
    for b, n in enumerate(lens):
        a, z = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        if z > a:
            yield b, a, z, n


def gather(pages: torch.Tensor, table_row, length: int) -> torch.Tensor:
    """(HKV, length, D) of one sequence, in 64 bits."""
    size = pages.shape[2]
    parts = [pages[table_row[p // size], :, :min(size, length - p)] for p in range(0, length, size)]
    return torch.cat(parts, 1).double() if parts else pages.new_zeros(pages.shape[1], 0, pages.shape[3]).double()


def append(qkv, cos, sin, k_pages, v_pages, table, lens, starts, q_norm=None, k_norm=None, eps=1e-6):
    """-> (q (T, HQ, D), {(page, slot): (k (HKV, D), v (HKV, D))}, terms): 64-bit
    values of what is written; rows that are skipped stay NaN in q. ``terms``
    (T, HQ + HKV, D) is |h cos| + |rot(h) sin|, the scale of rounding errors."""
    hkv, size, dim = k_pages.shape[1:]
    rows = qkv.shape[0]
    heads = qkv.shape[1] // dim - 2 * hkv
    x = qkv.double().reshape(rows, heads + 2 * hkv, dim)
    q = torch.full((rows, heads, dim), math.nan, dtype=torch.float64)
    terms = torch.zeros(rows, heads + hkv, dim, dtype=torch.float64)
    written = {}
    for b, a, z, n in sequences(rows, lens, starts):
        for t in range(a, z):
            pos = n - (z - a) + (t - a)
            if pos < 0:
                continue
            h = x[t, :heads + hkv]
            if q_norm is not None:
                gain = torch.cat([q_norm.double().expand(heads, dim), k_norm.double().expand(hkv, dim)])
                h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * gain
            rot = torch.cat([-h[:, dim // 2:], h[:, :dim // 2]], -1)
            c, s = cos[pos].double(), sin[pos].double()
            y = h * c + rot * s
            terms[t] = (h * c).abs() + (rot * s).abs()
            q[t] = y[:heads]
            written[(int(table[b][pos // size]), pos % size)] = (t, y[heads:], x[t, heads + hkv:])
    return q, written, terms


def attention(q, k_pages, v_pages, table, lens, starts, scale=None, causal=True):
    """-> dict(out (T, HQ, D), lse (T, HQ), weight (T, HQ, D) = sum p |v|,
    terms (T, HQ) = max over positions of scale * sum |q k|, seen (T,), vmax)."""
    hkv, _, dim = k_pages.shape[1:]
    rows = q.shape[0]
    heads = q.shape[1] // dim
    group = heads // hkv
    scale = dim ** -0.5 if scale is None else scale
    qd = q.double().reshape(rows, hkv, group, dim)
    out = torch.full((rows, hkv, group, dim), math.nan, dtype=torch.float64)
    weight = torch.zeros_like(out)
    lse = torch.full((rows, hkv, group), math.nan, dtype=torch.float64)
    terms = torch.zeros(rows, hkv, group, dtype=torch.float64)
    seen = torch.zeros(rows, dtype=torch.int64)
    vmax = 0.0
    for b, a, z, n in sequences(rows, lens, starts):
        n = max(n, 0)
        k, v = gather(k_pages, table[b], n), gather(v_pages, table[b], n)
        if n:
            vmax = max(vmax, float(v.abs().max()))
        for t in range(a, z):
            limit = max(0, min(n, lens[b] - (z - a) + (t - a) + 1)) if causal else n
            seen[t] = limit
            if limit == 0:
                out[t], lse[t] = 0.0, -math.inf
                continue
            kk, vv = k[:, :limit], v[:, :limit]
            score = torch.einsum("hgd,hsd->hgs", qd[t], kk) * scale
            terms[t] = (torch.einsum("hgd,hsd->hgs", qd[t].abs(), kk.abs()) * scale).amax(-1)
            p = torch.softmax(score, -1)
            out[t] = torch.einsum("hgs,hsd->hgd", p, vv)
            weight[t] = torch.einsum("hgs,hsd->hgd", p, vv.abs())
            lse[t] = torch.logsumexp(score, -1)
    return dict(out=out.reshape(rows, heads, dim), lse=lse.reshape(rows, heads), weight=weight.reshape(rows, heads, dim),
                terms=terms.reshape(rows, heads), seen=seen, vmax=vmax)


def attention_bounds(ref, dim: int, dtype: torch.dtype):
    """Largest errors of out and lse that the kernels' arithmetic allows.

    u = half a step of the element type. The output is rounded once (u |out|).
    Each probability is rounded to the element type before its product with v
    (u sum p |v|; fp16 probabilities under its normal range lose up to 2^-25
    each, of a largest one that is at least 1/2). A score is an fp32 sum of D
    products whose partial sums are at most `terms` in magnitude: each of the
    D + 8 roundings (products are exact, the tensor cores may cut instead of
    round: 2^-23 each; scaling, base-2 conversion and the exponential take the
    rest) moves it by 2^-23 terms, and moves a probability by that much in
    relation, numerator and denominator alike. The sums over positions are
    fp32: 2^-23 per position of sum p |v|."""
    u = torch.finfo(dtype).eps / 2
    seen = ref["seen"].double()[:, None]
    score = (dim + 8) * 2.0 ** -23 * (ref["terms"] + 1)
    spread = (seen + 8) * 2.0 ** -23
    out = u * ref["out"].abs() + (u + 2 * score + 2 * spread)[..., None] * ref["weight"]
    if dtype == torch.float16:
        out = out + (seen * 2.0 ** -24 * ref["vmax"])[..., None] + 2.0 ** -25  # a subnormal result's own step
    return out, score + spread + 2.0 ** -22 * ref["lse"].abs().nan_to_num(posinf=0.0)
