"""Seeded batches over an 8-bit paged cache for the tests: paged_cases' batches with
their pages quantised block by block. Every slot that no position needs holds NaN, every
scale that no position needs 255."""

from __future__ import annotations

import torch

from oracle import paged8 as o8
from tests import paged_cases as pc

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF, F16 = pc.BF, pc.F16


def quantise(x, used, block, level=None):
    """x (pages, HKV, page, D), its slots in use (pages, page) -> codes, scales; ``level``: e to add to each block."""
    pages, hkv, size, dim = x.shape
    x = x.double().masked_fill(~used[:, None, :, None], 0.0).reshape(pages, hkv, size // block, block, dim)
    if level is not None:
        x = x * torch.exp2(level.double())[..., None, None]
    live = used.reshape(pages, 1, size // block, block).any(-1).expand(pages, hkv, size // block)
    e = torch.tensor([o8.exponent(float(t)) for t in x.abs().amax((3, 4)).reshape(-1)]).reshape(live.shape)
    codes = o8.nearest(x * torch.exp2(-e.double())[..., None, None]).reshape(pages, hkv, size, dim)
    codes = codes.masked_fill(~used[:, None, :, None], float("nan")).float().to(F8)
    return codes, (e + 127).masked_fill(~live, 255).to(torch.uint8).view(E8)


def strided(t, layout):
    """The same tensor, stored (pages, slot, head, D) for "nhd"."""
    if layout != "nhd":
        return t
    u = t.view(torch.uint8)
    return u.transpose(1, 2).contiguous().transpose(1, 2).view(t.dtype)


def batch(lens, new, hq, hkv, dim, page, block, dtype=BF, seed=0, spare_rows=0, layout="hnd", qscale=1.0, spare_cols=1,
          levels=8):
    """paged_cases.batch, with k, v as codes and ks, vs as scales; blocks of v are 2^-levels .. 2^levels as large."""
    c = pc.batch(lens, new, hq, hkv, dim, page, dtype, seed, 0, spare_rows, "hnd", qscale, spare_cols)
    g = torch.Generator().manual_seed(seed + 1)
    per = (c["k"].shape[0], hkv, page // block)
    c["k"], c["ks"] = quantise(c["k"], c["used"], block, torch.randint(-1, 2, per, generator=g))
    c["v"], c["vs"] = quantise(c["v"], c["used"], block, torch.randint(-levels, levels + 1, per, generator=g))
    c["k"], c["v"] = strided(c["k"], layout), strided(c["v"], layout)
    c["block"] = block
    return c


def to(c, device):
    """As paged_cases.to, for the 8-bit types: strides are kept."""
    def move(t):
        u = t.view(torch.uint8) if t.dtype in (F8, E8) else t
        out = torch.empty_strided(u.shape, u.stride(), dtype=u.dtype, device=device).copy_(u)
        return out.view(t.dtype) if u is not t else out

    return {k: move(v) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def bits(t):
    return t.view(torch.uint8)
