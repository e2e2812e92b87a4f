"""Paged KV cache: streams of unequal length in one decode batch.

The static-cache attention step (breeze_b200.fused.kernels.attention_step, as
models/fused/kernels.py:505) has one cache position for the whole batch. Here
every sequence has its own length, in pages it shares with nobody or, for a
common prompt, with everybody:

  paged_append      new tokens' q / k / v rows -> per-head RMSNorm, RoPE at each
                    token's position, k and v into their pages, q returned
  paged_attention   softmax(scale q k^T) v over each sequence's pages, for one
                    new token per sequence or any ragged number of them
  prefix_attention  the same value for sequences whose tables begin with the
                    same pages: those are read once for the whole batch

Shared arguments:
  k_pages, v_pages  (pages, HKV, page size, D), bf16 or fp16, any strides with
                    contiguous D (a (pages, page size, HKV, D) cache is passed
                    as ``.transpose(1, 2)``); page size a power of two from 16
                    to 1024, D 64 or 128
  page_table        (B, columns) int32: page of positions [c * page size,
                    (c + 1) * page size) of each sequence; entries no position
                    needs may hold anything
  seq_lens          (B,) int32: positions of each sequence, new tokens included
  q_starts          (B + 1,) int32 ascending: rows q_starts[b] .. q_starts[b + 1]
                    are the new tokens of sequence b. None: one per sequence.
                    Rows from q_starts[B] on are left as they were.

Lengths, starts and tables are read on the device when the kernels run, so a
captured graph replays with whatever they then hold. A length or table entry
that does not fit is not read through; it sets a bit of ``device_status``
(BQ_DEVERR_POSITION, BQ_DEVERR_PAGE).

Everything runs on the current stream of the tensors' device. Scratch comes
from torch's allocator for each call: calls on different streams, and graphs
captured from them, share none.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib

_I32 = torch.int32


def _check(cond: bool, message: str) -> None:
    if not cond:
        raise ValueError(message)


def _cache_fields(rows: int, dtype: torch.dtype, dev: torch.device, k_pages, v_pages, page_table, seq_lens, q_starts):
    """The leading fields of both descriptors, after the checks both calls share."""
    for t in (k_pages, v_pages, page_table, seq_lens, q_starts):
        if t is not None and t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    if dev.type != "cuda":
        raise RuntimeError("breeze_b200 kernels need CUDA tensors (there is no CPU path)")
    _check(dtype in (torch.bfloat16, torch.float16), f"paged caches are bf16 or fp16 (got {dtype})")
    _check(k_pages.dtype == dtype and v_pages.dtype == dtype, "rows and pages must have one dtype")
    shape = k_pages.shape
    _check(len(shape) == 4 and v_pages.shape == shape, "k_pages and v_pages must be (pages, HKV, page size, D)")
    ks, vs = k_pages.stride(), v_pages.stride()
    _check(ks[3] == 1 and vs[3] == 1, "the last dimension of the pages must be contiguous")
    _check(page_table.dtype == _I32 and page_table.dim() == 2 and page_table.stride(1) == 1,
           "page_table must be int32 (B, columns) with contiguous rows")
    batch, columns = page_table.shape
    _check(seq_lens.dtype == _I32 and seq_lens.shape == (batch,) and seq_lens.is_contiguous(),
           "seq_lens must be a contiguous int32 (B,)")
    if q_starts is None:
        _check(rows == batch, f"{rows} rows for {batch} sequences: ragged rows need q_starts")
        starts = None
    else:
        _check(q_starts.dtype == _I32 and q_starts.shape == (batch + 1,) and q_starts.is_contiguous(),
               "q_starts must be a contiguous int32 (B + 1,)")
        starts = q_starts.data_ptr()
    pages, hkv, size, dim = shape
    _check(pages > 0 and hkv > 0 and columns > 0 and batch > 0, "empty cache or batch")
    return (batch, hkv, dim, size, pages, columns, _lib._DT[dtype], 0, k_pages.data_ptr(), ks[0], ks[1], ks[2],
            v_pages.data_ptr(), vs[0], vs[1], vs[2], page_table.data_ptr(),
            page_table.stride(0) if batch > 1 else columns, seq_lens.data_ptr(), starts)


def _row_tensor(t: torch.Tensor, name: str) -> int:
    """Row stride of a 2-D tensor with contiguous rows."""
    _check(t.dim() == 2 and t.stride(1) == 1, f"{name} must be a 2-D tensor with unit stride in the last dimension")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor, q_starts: torch.Tensor | None = None,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv (T, (HQ + 2 HKV) D) rows [q heads | k heads | v heads] of the new
    tokens -> q (T, HQ D), normed and rotated; k (normed, rotated) and v written
    into their pages. ``cos`` / ``sin``: (positions, D) tables (fp32 or the
    cache's dtype), row p for cache position p, both halves given as rotate_half
    takes them. The math is fp32 with one rounding at the end. ``out`` may be
    ``qkv[:, :HQ * D]`` itself. Tokens of an unused batch slot (seq_lens[b] less
    than its new tokens) are skipped where their position would be negative."""
    dev, dtype = qkv.device, qkv.dtype
    ldqkv = _row_tensor(qkv, "qkv")
    rows, width = qkv.shape
    fields = _cache_fields(rows, dtype, dev, k_pages, v_pages, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim - 2 * hkv
    _check(hq > 0 and (hq + 2 * hkv) * dim == width, f"qkv width {width} does not split into heads of {dim}")
    _check(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == dim and cos.dtype == sin.dtype,
           "cos and sin must be (positions, D) tables of one shape and dtype")
    _check(cos.dtype == dtype or cos.dtype == torch.float32, "cos and sin must be fp32 or the cache's dtype")
    ldcs = _row_tensor(cos, "cos")
    _check(_row_tensor(sin, "sin") == ldcs, "cos and sin must have equal strides")
    _check((q_norm_w is None) == (k_norm_w is None), "q_norm_w and k_norm_w go together")
    for t in (cos, sin, q_norm_w, k_norm_w, out):
        if t is not None and t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    if q_norm_w is not None:
        for t in (q_norm_w, k_norm_w):
            _check(t.dtype == dtype and t.shape == (dim,) and t.is_contiguous(),
                   "norm weights must be contiguous (D,) vectors of the cache's dtype")
    if out is None:
        out = torch.empty(rows, hq * dim, device=dev, dtype=dtype)
    else:
        _check(out.shape == (rows, hq * dim) and out.dtype == dtype, "out must be (T, HQ D) of the cache's dtype")
    desc = _lib.PagedAppendDesc(
        *fields, rows, hq, _lib._DT[cos.dtype], cos.shape[0], eps, _lib.default_flags(), qkv.data_ptr(), ldqkv,
        cos.data_ptr(), sin.data_ptr(), ldcs, None if q_norm_w is None else q_norm_w.data_ptr(),
        None if k_norm_w is None else k_norm_w.data_ptr(), out.data_ptr(), _row_tensor(out, "out"))
    with torch.cuda.device(dev):
        _lib.check(_lib.load().bq_paged_append(ctypes.byref(desc), _lib._stream(dev)), "bq_paged_append")
    return out


def _attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, causal, max_q, out, lse):
    dev, dtype = q.device, q.dtype
    ldq = _row_tensor(q, "q")
    rows, width = q.shape
    fields = _cache_fields(rows, dtype, dev, k_pages, v_pages, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim
    _check(hq > 0 and hq * dim == width and hq % hkv == 0,
           f"q width {width} does not split into heads of {dim} over {hkv} kv heads")
    if out is None:
        out = torch.empty(rows, width, device=dev, dtype=dtype)
    else:
        _check(out.shape == (rows, width) and out.dtype == dtype and out.device == dev,
               "out must be (T, HQ D) of q's dtype and device")
    lse_ptr, ldl = None, 0
    if lse is not None:
        _check(lse.shape == (rows, hq) and lse.dtype == torch.float32 and lse.device == dev,
               "lse must be fp32 (T, HQ) on q's device")
        lse_ptr, ldl = lse.data_ptr(), _row_tensor(lse, "lse")
    desc = _lib.PagedAttnDesc(
        *fields, rows, hq, prefix_len, 0 if max_q is None else max_q, dim ** -0.5 if scale is None else scale,
        _lib.default_flags() | (0 if causal else _lib.PAGED_FULL), q.data_ptr(), ldq, out.data_ptr(),
        _row_tensor(out, "out"), lse_ptr, ldl)
    lib = _lib.load()
    with torch.cuda.device(dev):
        need = ctypes.c_size_t(0)
        _lib.check(lib.bq_paged_attention_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)),
                   "bq_paged_attention_workspace_bytes")
        ws = torch.empty(need.value, device=dev, dtype=torch.uint8) if need.value else None
        _lib.check(lib.bq_paged_attention(ctypes.byref(desc), None if ws is None else ws.data_ptr(), need.value,
                                          _lib._stream(dev)), "bq_paged_attention")
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, q_starts: torch.Tensor | None = None, scale: float | None = None,
                    causal: bool = True, max_q: int | None = None, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None) -> torch.Tensor:
    """q (T, HQ D) of the new tokens (already in the cache: paged_append first)
    -> (T, HQ D). Row i of the n new rows of sequence b sees positions
    [0, seq_lens[b] - n + i + 1); with ``causal=False`` all seq_lens[b]. A row
    that sees none gets zeros. Query head h reads kv head h // (HQ / HKV).
    ``scale`` defaults to D^-0.5. ``max_q``: most new tokens of one sequence, a
    hint that picks the kernel (default: T / B rounded up). ``lse`` (T, HQ) fp32
    receives log(sum(exp(scores))), -inf for a row that sees nothing."""
    return _attention(q, k_pages, v_pages, page_table, seq_lens, 0, q_starts, scale, causal, max_q, out, lse)


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                     seq_lens: torch.Tensor, prefix_len: int, q_starts: torch.Tensor | None = None,
                     scale: float | None = None, causal: bool = True, max_q: int | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention for a batch that shares its first ``prefix_len``
    positions (a multiple of the page size): the first prefix_len / page size
    entries of every table row name the same pages. They are read once for all
    rows together, through row 0 of the table, and joined with each sequence's
    own positions; the value is paged_attention's."""
    return _attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, causal, max_q, out, lse)
