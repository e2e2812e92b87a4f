"""Paged KV cache held in 8 bits: half the bytes of breeze_b200.fused.paged's.

  paged_append_fp8      new tokens' q / k / v rows -> per-head RMSNorm, RoPE at each
                        token's position, k and v quantised into their pages, q returned
  paged_attention_fp8   softmax(scale q k^T) v over each sequence's pages, for one
                        new token per sequence or any ragged number of them
  paged_read_fp8        the last positions of each sequence back as bf16, fp16 or fp32
                        rows (to move a cache into a 16-bit one, or out of the GPU)

Every cache entry is an e4m3 code times a power of two that a block of positions of a
kv head shares (k and v have their own). A block's scale is 2^e with the least e from
-60 to 60 for which the largest finite magnitude that was written to it, since its
first position was, is at most 448 2^e. A block fills up over many calls: when a later
token needs a larger scale, the codes that are there are divided by the power of two in
between, which is exact but for the smallest; when it would need a smaller one, the
scale stays. So tokens that are taken back (rejected drafts: shorter lengths in the next
call) leave a block the scale that they needed, with the bits that its codes lost by
it, until its first position is written again. Infinite and NaN entries are held as NaN.

Arguments as in breeze_b200.fused.paged, but
  k_pages, v_pages    (pages, HKV, page size, D) float8_e4m3fn, any strides that are
                      multiples of 16 with contiguous D; page size a power of two
                      from 16 to 1024, D 64 or 128
  k_scales, v_scales  (pages, HKV, blocks) float8_e8m0fnu, contiguous blocks: page
                      size / blocks positions (16, 32, 64 or 128) share a scale.
                      ``pages.float()`` times the block's ``scales.float()`` is the
                      value. Nothing needs to be initialised: what holds no position
                      may hold anything. (An append behind positions of a block that
                      no append wrote finds their codes and scale as they are.)
page_table, seq_lens and q_starts are the same, and so is what is read on the device, the
error bits of ``device_status``, the stream, the scratch and what graphs may do. The
rows' dtype is bf16 or fp16, whatever wrote the cache. A page belongs to one sequence
where it is written; sequences may share pages that are only read.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from . import paged
from .paged import _CACHE_DT, _F32, _I32, _UNIT, _count, _launch, _real, _row_stride, _workspace_bytes_of

_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_OUT_DT = {**_CACHE_DT, _F32: _lib.DT_F32}
_pack_append = _lib.packer(_lib.Paged8AppendDesc)
_pack_attn = _lib.packer(_lib.Paged8AttnDesc)
_pack_read = _lib.packer(_lib.Paged8ReadDesc)


def _cache_fields(dev: int, rows: int, code: int, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts):
    """The leading fields of the descriptors, after the checks the calls share."""
    if dev < 0:
        raise RuntimeError("breeze_b200 kernels need CUDA tensors (there is no CPU path)")
    for t in (k_pages, v_pages, k_scales, v_scales, page_table, seq_lens):
        if t.get_device() != dev:
            raise RuntimeError("tensors on different devices: the rows, the cache and the lengths must share one")
    if k_pages.dtype != _E4M3 or v_pages.dtype != _E4M3:
        raise ValueError(f"pages must be float8_e4m3fn (got {k_pages.dtype}, {v_pages.dtype})")
    if k_scales.dtype != _E8M0 or v_scales.dtype != _E8M0:
        raise ValueError(f"scales must be float8_e8m0fnu (got {k_scales.dtype}, {v_scales.dtype})")
    shape, per = k_pages.shape, k_scales.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be (pages, HKV, page size, D) of one shape")
    if len(per) != 3 or v_scales.shape != per or per[:2] != shape[:2]:
        raise ValueError("k_scales and v_scales must be (pages, HKV, blocks) of one shape, pages and HKV the cache's")
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    a0, a1, a2 = k_scales.stride()
    b0, b1, b2 = v_scales.stride()
    ts = page_table.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
    if (a2 != 1 or b2 != 1) and per[2] != 1:
        raise ValueError("the last dimension of the scales must be contiguous")
    if page_table.dtype != _I32 or len(ts) != 2 or (ts[1] != 1 and page_table.shape[1] != 1):
        raise ValueError("page_table must be int32 (B, columns) with contiguous rows")
    batch, columns = page_table.shape
    if seq_lens.dtype != _I32 or seq_lens.shape != (batch,) or (seq_lens.stride() != _UNIT and batch != 1):
        raise ValueError("seq_lens must be a contiguous int32 (B,)")
    if q_starts is None:
        if rows != batch:
            raise ValueError(f"{rows} rows for {batch} sequences: ragged rows need q_starts")
        starts = 0
    else:
        if q_starts.dtype != _I32 or q_starts.shape != (batch + 1,) or q_starts.stride() != _UNIT:
            raise ValueError("q_starts must be a contiguous int32 (B + 1,)")
        if q_starts.get_device() != dev:
            raise RuntimeError("tensors on different devices: q_starts is not where the rows are")
        starts = q_starts.data_ptr()
    pages, hkv, size, dim = shape
    if pages == 0 or hkv == 0 or size == 0 or dim == 0 or per[2] == 0 or columns == 0 or batch == 0:
        raise ValueError("empty cache or batch")
    if size % per[2]:
        raise ValueError(f"{per[2]} scales do not divide a page of {size} positions")
    return (batch, hkv, dim, size, pages, columns, size // per[2], code, k_pages.data_ptr(), k0, k1, k2, v_pages.data_ptr(), v0,
            v1, v2, k_scales.data_ptr(), a0, a1, v_scales.data_ptr(), b0, b1, page_table.data_ptr(),
            ts[0] if batch > 1 else columns, seq_lens.data_ptr(), starts)


def _rows_dtype(t: torch.Tensor) -> int:
    code = _CACHE_DT.get(t.dtype)
    if code is None:
        raise ValueError(f"rows are bf16 or fp16 (got {t.dtype})")
    return code


def paged_append_fp8(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     k_scales: torch.Tensor, v_scales: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     q_starts: torch.Tensor | None = None, q_norm_w: torch.Tensor | None = None,
                     k_norm_w: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """paged.paged_append into an 8-bit cache: qkv (T, (HQ + 2 HKV) D) rows
    [q heads | k heads | v heads] of the new tokens -> q (T, HQ D), normed and
    rotated, in qkv's dtype; k (normed, rotated) and v quantised from fp32 into their
    pages, scales and older codes of the blocks that get new tokens brought up to date.
    ``cos`` / ``sin``: (positions, D) tables (fp32 or qkv's dtype). ``out`` may be
    ``qkv[:, :HQ * D]`` itself, and else shares no memory with ``qkv``. Tokens of
    an unused batch slot (seq_lens[b] less than its new tokens) are skipped where
    their position would be negative. The same call again changes nothing."""
    done = (paged._bound or paged._native()).append8(qkv, cos, sin, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens,
                                                     q_starts, q_norm_w, k_norm_w, eps, out, _lib.default_flags())
    if done is not None:
        return done if done.__class__ is not int else _lib.check(done, "bq_paged8_append")
    ldqkv = _row_stride(qkv, "qkv")
    rows, width = qkv.shape
    dev, dtype = qkv.get_device(), qkv.dtype
    fields = _cache_fields(dev, rows, _rows_dtype(qkv), k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim - 2 * hkv
    if hq <= 0 or (hq + 2 * hkv) * dim != width:
        raise ValueError(f"qkv width {width} does not split into q, k and v heads of {dim}")
    ldcs, cs_dtype, cs_shape = _row_stride(cos, "cos"), cos.dtype, cos.shape
    if cs_shape[1] != dim or sin.shape != cs_shape or sin.dtype != cs_dtype or _row_stride(sin, "sin") != ldcs:
        raise ValueError("cos and sin must be (positions, D) tables of one shape, stride and dtype")
    if cs_dtype != dtype and cs_dtype != _F32:
        raise ValueError(f"cos and sin must be fp32 or the rows' dtype (got {cs_dtype})")
    if not (cos.get_device() == sin.get_device() == dev):
        raise RuntimeError("cos and sin are on another device than qkv")
    qn = kn = 0
    if q_norm_w is not None and k_norm_w is not None:
        for t in (q_norm_w, k_norm_w):
            if t.dtype != dtype or t.shape != (dim,) or t.stride() != _UNIT or t.get_device() != dev:
                raise ValueError("norm weights must be contiguous (D,) vectors of the rows' dtype and device")
        qn, kn = q_norm_w.data_ptr(), k_norm_w.data_ptr()
    elif q_norm_w is not None or k_norm_w is not None:
        raise ValueError("q_norm_w and k_norm_w go together")
    ldq = hq * dim
    if out is None:
        out = qkv.new_empty((rows, ldq))
    elif out.shape != (rows, ldq) or out.dtype != dtype or out.get_device() != dev:
        raise ValueError("out must be (T, HQ D) of qkv's dtype and device")
    else:
        ldq = _row_stride(out, "out")
    desc = _pack_append(*fields, rows, hq, _lib._DT[cs_dtype], cs_shape[0], _real(eps, "eps"), _lib.default_flags(), qkv.data_ptr(), ldqkv,
                        cos.data_ptr(), sin.data_ptr(), ldcs, qn, kn, out.data_ptr(), ldq)
    _launch(dev, "bq_paged8_append", _lib.load().bq_paged8_append, desc)
    return out


def paged_attention_fp8(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor,
                        v_scales: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                        q_starts: torch.Tensor | None = None, scale: float | None = None, causal: bool = True,
                        max_q: int | None = None, out: torch.Tensor | None = None,
                        lse: torch.Tensor | None = None) -> torch.Tensor:
    """paged.paged_attention over an 8-bit cache: q (T, HQ D) of the new tokens
    (already in the cache: paged_append_fp8 first) -> (T, HQ D). Row i of the n new
    rows of sequence b sees positions [0, seq_lens[b] - n + i + 1); with
    ``causal=False`` all seq_lens[b]. A row that sees none gets zeros, one whose scores
    are all -inf gets NaN; NaN keys and values at positions it does not see stay
    without effect. Query head h reads kv head h // (HQ / HKV). ``scale`` defaults to
    D^-0.5. ``max_q``: most new tokens of one sequence, a hint that picks the kernel
    (0 or None: T / B rounded up; say it where they differ). ``lse`` (T, HQ) fp32
    receives log(sum(exp(scores))), -inf for a row that sees nothing."""
    flags = _lib.default_flags() | (0 if causal else _lib.PAGED_FULL)
    done = (paged._bound or paged._native()).attention8(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts,
                                                        scale, max_q, out, lse, flags)
    if done is not None:
        return done if done.__class__ is not int else _lib.check(done, "bq_paged8_attention")
    ldq = _row_stride(q, "q")
    rows, width = q.shape
    dev, dtype = q.get_device(), q.dtype
    fields = _cache_fields(dev, rows, _rows_dtype(q), k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim
    if hq == 0 or hq * dim != width or hq % hkv:
        raise ValueError(f"q width {width} does not split into heads of {dim} over {hkv} kv heads")
    ldo = width
    if out is None:
        out = q.new_empty((rows, width))
    elif out.shape != (rows, width) or out.dtype != dtype or out.get_device() != dev:
        raise ValueError("out must be (T, HQ D) of q's dtype and device")
    else:
        ldo = _row_stride(out, "out")
    lse_ptr = ldl = 0
    if lse is not None:
        if lse.shape != (rows, hq) or lse.dtype != _F32 or lse.get_device() != dev:
            raise ValueError("lse must be fp32 (T, HQ) on q's device")
        lse_ptr, ldl = lse.data_ptr(), _row_stride(lse, "lse")
    max_q = 0 if max_q is None else _count(max_q, "max_q")
    scale = dim ** -0.5 if scale is None else _real(scale, "scale")
    desc = _pack_attn(*fields, rows, hq, max_q, scale, flags, 0, q.data_ptr(), ldq, out.data_ptr(), ldo, lse_ptr, ldl)
    lib = _lib.load()
    size = ctypes.c_size_t(0)
    _launch(dev, "bq_paged8_attention_workspace_bytes", _workspace_bytes_of(lib.bq_paged8_attention_workspace_bytes), desc,
            ctypes.byref(size))
    need = size.value
    ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    _launch(dev, "bq_paged8_attention", lib.bq_paged8_attention, desc, ws.data_ptr() if need else None, need)
    return out


def _read_out(t: torch.Tensor | None, name: str, like: torch.Tensor, rows: int, hkv: int, dim: int, dtype: torch.dtype):
    """A (rows, HKV, D) output and its strides of a row and a head."""
    if t is None:
        t = torch.empty((rows, hkv, dim), dtype=dtype, device=like.device)
    elif t.shape != (rows, hkv, dim) or t.dtype != dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must be (rows, HKV, D) of the dtype asked for, on the cache's device")
    if t.stride(2) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return t, t.stride(0) if rows > 1 else hkv * dim, t.stride(1) if hkv > 1 else dim


def paged_read_fp8(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                   page_table: torch.Tensor, seq_lens: torch.Tensor, q_starts: torch.Tensor | None = None,
                   rows: int | None = None, dtype: torch.dtype = torch.bfloat16, k_out: torch.Tensor | None = None,
                   v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """An 8-bit cache back as rows: k and v (rows, HKV, D). Rows q_starts[b] ..
    q_starts[b + 1] are the last positions of sequence b, as paged_append_fp8 takes
    them (without ``q_starts`` its last one); q_starts of the lengths summed up read
    whole caches. ``rows``: how many there are, q_starts[B] or more (by default
    k_out's, or one per sequence). ``dtype``: bf16 and fp32 hold every value exactly,
    fp16 rounds once, a finite value to a finite one. Rows that are no position's (from
    q_starts[B] on, before a sequence's first position) are left as they were."""
    code = _OUT_DT.get(dtype)
    if code is None:
        raise ValueError(f"rows are read back as bf16, fp16 or fp32 (got {dtype})")
    if rows is not None:
        rows = _count(rows, "rows")
    elif k_out is not None:
        rows = k_out.shape[0]
    elif q_starts is None:
        rows = page_table.shape[0]
    else:
        raise ValueError("ragged rows need `rows` or k_out: their number is on the device")
    done = (paged._bound or paged._native()).read8(k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts, rows,
                                                   code, k_out, v_out, _lib.default_flags())
    if done is not None:
        return done if done.__class__ is not int else _lib.check(done, "bq_paged8_read")
    dev = k_pages.get_device()
    fields = _cache_fields(dev, rows, code, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    k_out, kr, kh = _read_out(k_out, "k_out", k_pages, rows, hkv, dim, dtype)
    v_out, vr, vh = _read_out(v_out, "v_out", k_pages, rows, hkv, dim, dtype)
    desc = _pack_read(*fields, rows, _lib.default_flags(), k_out.data_ptr(), kr, kh, v_out.data_ptr(), vr, vh)
    _launch(dev, "bq_paged8_read", _lib.load().bq_paged8_read, desc)
    return k_out, v_out
