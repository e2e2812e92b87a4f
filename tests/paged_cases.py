"""Seeded batches over a paged cache for the tests: every slot and table entry
that no position needs holds something that must not be read (NaN, page ids
far outside the cache)."""

from __future__ import annotations

import torch

BF, F16 = torch.bfloat16, torch.float16


def batch(lens, new, hq, hkv, dim, page, dtype=BF, seed=0, prefix=0, spare_rows=0, layout="hnd", qscale=1.0, spare_cols=1):
    """new: None (one token per sequence) or a list of new tokens per sequence.
    -> dict of CPU tensors; k_pages / v_pages (pages, hkv, page, dim) in the
    given layout ("hnd", or "nhd": stored (pages, page, hkv, dim))."""
    g = torch.Generator().manual_seed(seed)
    shared = prefix // page
    need = [max(0, -(-max(n, 0) // page) - shared) for n in lens]
    pages = shared + sum(need) + 2
    ids = torch.randperm(pages, generator=g)
    cols = max([shared] + [-(-max(n, 0) // page) for n in lens]) + spare_cols
    table = torch.full((len(lens), cols), 2 ** 30, dtype=torch.int32)
    at = shared
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        table[b, :shared] = ids[:shared]
        table[b, shared:shared + need[b]] = ids[at:at + need[b]]
        at += need[b]
        for p in range(0, max(n, 0), page):
            used[table[b, p // page], :min(page, n - p)] = True
    used[ids[:shared]] = True

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    kv = []
    for _ in range(2):
        t = normal(pages, hkv, page, dim)
        t[~used[:, None, :, None].expand_as(t)] = float("nan")
        t = t.to(dtype)
        kv.append(t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "nhd" else t)
    starts = None
    rows = len(lens)
    if new is not None:
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        rows = int(starts[-1]) + spare_rows
    return dict(q=(normal(rows, hq * dim) * qscale).to(dtype), k=kv[0], v=kv[1], table=table, rows=rows,
                lens=torch.tensor(lens, dtype=torch.int32), starts=starts, dim=dim, hq=hq, hkv=hkv, page=page,
                dtype=dtype, prefix=prefix, used=used)


def lists(c):
    """(table rows, lens, starts) as Python lists, for the oracle."""
    return c["table"].tolist(), c["lens"].tolist(), None if c["starts"] is None else c["starts"].tolist()


def to(c, device):
    def move(t):
        if t.dim() != 4:
            return t.to(device)
        out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)  # keeps the layout
        return out.copy_(t)

    return {k: move(v) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
