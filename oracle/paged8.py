"""8-bit paged cache restated on the CPU in 64 bits (test oracle only).

An entry is an e4m3 value times 2^e, one e for each block of positions and kv head.
e4m3 values are computed here from the format's definition (steps of 2^-9 up to
2^-6, then an eighth of the power of two below), not by a cast.
"""

from __future__ import annotations

import math

import torch

from . import paged as op

E_MOST = 60


def nearest(x: torch.Tensor) -> torch.Tensor:
    """64-bit values to the nearest e4m3 value, ties to even, at most 448; infinite and NaN to NaN."""
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6, max=448.0))) - 3)
    y = (torch.round(x / step) * step).clamp(-448.0, 448.0)
    return torch.where(torch.isfinite(x), y, math.nan)


def exponent(top: float) -> int:
    """Least e from -60 to 60 with top <= 448 2^e."""
    if top == 0.0:
        return -E_MOST
    m, x = math.frexp(top)  # top = m 2^x with 1/2 <= m < 1; 448 is 7/8 of 2^9
    return max(-E_MOST, min(E_MOST, x - 9 + (m > 0.875)))


def scales_of(scales: torch.Tensor) -> torch.Tensor:
    """e of every scale byte, as the kernels read it."""
    return (scales.view(torch.uint8).int() - 127).clamp(-E_MOST, E_MOST)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """(pages, HKV, page size, D) in 64 bits."""
    pages, hkv, size, dim = codes.shape
    x = codes.double().reshape(pages, hkv, scales.shape[2], -1, dim)
    return (x * torch.exp2(scales_of(scales).double())[..., None, None]).reshape(pages, hkv, size, dim)


def block_parts(rows: int, lens, starts, block: int, limit: int | None = None):
    """(sequence, first row, rows, first position, kept) of every block's new tokens; kept: the block's older positions."""
    for b, a, z, n in op.sequences(rows, lens, starts):
        first = n - (z - a)
        p = max(first, 0)
        while p < (n if limit is None else min(n, limit)):
            kept = p % block
            m = min(block - kept, n - p) if limit is None else min(block - kept, min(n, limit) - p)
            yield b, a + p - first, m, p, kept
            p += m


def attention(q, codes, scales, table, lens, starts, scale=None, causal=True):
    """oracle.paged.attention on the values ((k, v) codes and scales); with the largest normalized weight
    p 2^e of every (row, head) as "heaviest", and the largest |q| |k| of one product."""
    k, v = values(codes[0], scales[0]), values(codes[1], scales[1])
    ref = op.attention(q, k, v, table, lens, starts, scale, causal)
    rows, heads = ref["lse"].shape
    hkv, dim, size = k.shape[1], k.shape[3], k.shape[2]
    group, block = heads // hkv, size // scales[0].shape[2]
    scale = dim ** -0.5 if scale is None else scale
    ref["heaviest"] = torch.zeros(rows, heads, dtype=torch.float64)
    qd = q.double().reshape(rows, hkv, group, dim)
    ev = scales_of(scales[1])
    for b, a, z, n in op.sequences(rows, lens, starts):
        n = max(n, 0)
        if n == 0:
            continue
        kk = op.gather(k, table[b], n)
        e = torch.stack([ev[table[b][p // size], :, p % size // block] for p in range(0, n, block)], 1)
        e = e.repeat_interleave(block, 1)[:, :n].double()
        for t in range(a, z):
            m = int(ref["seen"][t])
            if m:
                s = torch.einsum("hgd,hsd->hgs", qd[t], kk[:, :m]) * scale
                w = torch.softmax(s, -1) * torch.exp2(e[:, None, :m])
                ref["heaviest"][t] = w.amax(-1).reshape(heads)
    return ref


def attention_bounds(ref, dim: int, dtype: torch.dtype):
    """Largest errors of out and lse that the kernels' arithmetic allows.

    As oracle.paged.attention_bounds, but the probabilities (times their block's 2^e)
    enter the second product in fp16, 2^15 times their ratio to the largest one: half
    a step of fp16 each (2^-11 of their size), and, of those that are subnormal there,
    half of its smallest step, 2^-25 2^-15 of the largest one, times a code of at most
    448 (the largest one may be a running one, up to a factor 2^8 smaller than the
    final one's bound: 2^-32 covers it). Scores: bf16 queries are scaled by a power of
    two so that a row's largest entry is at least 2^14 in fp16, and lose at most 2^-25
    there: 2^-39 of the largest entry per product, far under the (dim + 8) 2^-23 of the
    sum's own roundings, which count for |q| |k| summed; 2^-23 more covers them where
    one entry is all there is. The sum of exponentials comes from the same weights: with
    exponents of v up to 100 apart, what fp32 flushes of a weight (under 2^-126, at 2^7
    times its size) is at most 2^-33 of the sum's largest term; further apart the sum is of
    weights 2^64 times as large."""
    u, up = torch.finfo(dtype).eps / 2, 2.0 ** -11
    seen = ref["seen"].double()[:, None]
    score = (dim + 9) * 2.0 ** -23 * (ref["terms"] + 1)
    spread = (seen + 8) * 2.0 ** -23 + seen * 2.0 ** -33
    out = u * ref["out"].abs() + (up + 2 * score + 2 * spread)[..., None] * ref["weight"]
    out = out + (seen * 2.0 ** -32 * 448.0 * ref["heaviest"])[..., None]
    if dtype == torch.float16:
        out = out + 2.0 ** -25  # a subnormal result's own step
    return out, score + spread + 2.0 ** -22 * ref["lse"].abs().nan_to_num(posinf=0.0)
