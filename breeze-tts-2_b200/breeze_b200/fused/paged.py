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

_I32, _F32 = torch.int32, torch.float32
_pack_append = _lib.packer(_lib.PagedAppendDesc)
_pack_attn = _lib.packer(_lib.PagedAttnDesc)
_WORKSPACE: dict = {}  # bytes by shape; a decode loop asks once


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Row stride of a 2-D tensor with contiguous rows."""
    st = t.stride()
    if len(st) != 2 or st[1] != 1:
        raise ValueError(f"{name} must be a 2-D tensor with unit stride in the last dimension")
    return st[0] if t.shape[0] > 1 else t.shape[1]


def _cache_fields(x: torch.Tensor, rows: int, k_pages, v_pages, page_table, seq_lens, q_starts):
    """The leading fields of both descriptors, after the checks both calls share."""
    dev, dtype = x.get_device(), x.dtype
    if dev < 0:
        raise RuntimeError("breeze_b200 kernels need CUDA tensors (there is no CPU path)")
    if (k_pages.get_device() != dev or v_pages.get_device() != dev or page_table.get_device() != dev
            or seq_lens.get_device() != dev or (q_starts is not None and q_starts.get_device() != dev)):
        raise RuntimeError(f"tensors on different devices: rows on {x.device}, cache or lengths elsewhere")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"paged caches are bf16 or fp16 (got {dtype})")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError(f"rows and pages must have one dtype (got {dtype}, {k_pages.dtype}, {v_pages.dtype})")
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be (pages, HKV, page size, D) of one shape")
    ks, vs, ts = k_pages.stride(), v_pages.stride(), page_table.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
    if page_table.dtype != _I32 or len(ts) != 2 or ts[1] != 1:
        raise ValueError("page_table must be int32 (B, columns) with contiguous rows")
    batch, columns = page_table.shape
    if seq_lens.dtype != _I32 or seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 (B,)")
    starts = 0
    if q_starts is not None:
        if q_starts.dtype != _I32 or q_starts.shape != (batch + 1,) or not q_starts.is_contiguous():
            raise ValueError("q_starts must be a contiguous int32 (B + 1,)")
        starts = q_starts.data_ptr()
    elif rows != batch:
        raise ValueError(f"{rows} rows for {batch} sequences: ragged rows need q_starts")
    pages, hkv, size, dim = shape
    if pages == 0 or hkv == 0 or dim == 0 or columns == 0 or batch == 0:
        raise ValueError("empty cache or batch")
    return (batch, hkv, dim, size, pages, columns, _lib._DT[dtype], 0, k_pages.data_ptr(), ks[0], ks[1], ks[2],
            v_pages.data_ptr(), vs[0], vs[1], vs[2], page_table.data_ptr(), ts[0] if batch > 1 else columns,
            seq_lens.data_ptr(), starts)


def _on_device(dev: int, call, *args):
    """call(*args) with ``dev`` as the current device."""
    if dev == torch.cuda.current_device():
        return call(*args)
    with torch.cuda.device(dev):
        return call(*args)


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
    ldqkv = _row_stride(qkv, "qkv")
    rows, width = qkv.shape
    dev, dtype = qkv.get_device(), qkv.dtype
    fields = _cache_fields(qkv, rows, k_pages, v_pages, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim - 2 * hkv
    if hq <= 0 or (hq + 2 * hkv) * dim != width:
        raise ValueError(f"qkv width {width} does not split into q, k and v heads of {dim}")
    ldcs, cs_dtype = _row_stride(cos, "cos"), cos.dtype
    if cos.shape != sin.shape or cos.shape[1] != dim or cs_dtype != sin.dtype or _row_stride(sin, "sin") != ldcs:
        raise ValueError("cos and sin must be (positions, D) tables of one shape, stride and dtype")
    if cs_dtype != dtype and cs_dtype != _F32:
        raise ValueError(f"cos and sin must be fp32 or the cache's dtype (got {cs_dtype})")
    if cos.get_device() != dev or sin.get_device() != dev:
        raise RuntimeError("cos and sin are on another device than qkv")
    qn = kn = 0
    if q_norm_w is not None and k_norm_w is not None:
        for t in (q_norm_w, k_norm_w):
            if t.dtype != dtype or t.shape != (dim,) or not t.is_contiguous() or t.get_device() != dev:
                raise ValueError("norm weights must be contiguous (D,) vectors of the cache's dtype and device")
        qn, kn = q_norm_w.data_ptr(), k_norm_w.data_ptr()
    elif q_norm_w is not None or k_norm_w is not None:
        raise ValueError("q_norm_w and k_norm_w go together")
    if out is None:
        out = qkv.new_empty((rows, hq * dim))
    elif out.shape != (rows, hq * dim) or out.dtype != dtype or out.get_device() != dev:
        raise ValueError("out must be (T, HQ D) of the cache's dtype and device")
    desc = _pack_append(*fields, rows, hq, _lib._DT[cs_dtype], cos.shape[0], eps, _lib.default_flags(), qkv.data_ptr(),
                        ldqkv, cos.data_ptr(), sin.data_ptr(), ldcs, qn, kn, out.data_ptr(), _row_stride(out, "out"))
    _lib.check(_on_device(dev, _lib.load().bq_paged_append, desc, torch._C._cuda_getCurrentRawStream(dev)),
               "bq_paged_append")
    return out


def _workspace_bytes(desc: bytes) -> int:
    need = ctypes.c_size_t(0)
    _lib.check(_lib.load().bq_paged_attention_workspace_bytes(desc, ctypes.byref(need)),
               "bq_paged_attention_workspace_bytes")
    return need.value


def _attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, causal, max_q, out, lse):
    ldq = _row_stride(q, "q")
    rows, width = q.shape
    dev = q.get_device()
    fields = _cache_fields(q, rows, k_pages, v_pages, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim
    if hq == 0 or hq * dim != width or hq % hkv:
        raise ValueError(f"q width {width} does not split into heads of {dim} over {hkv} kv heads")
    if out is None:
        out = q.new_empty((rows, width))
    elif out.shape != (rows, width) or out.dtype != q.dtype or out.get_device() != dev:
        raise ValueError("out must be (T, HQ D) of q's dtype and device")
    lse_ptr = ldl = 0
    if lse is not None:
        if lse.shape != (rows, hq) or lse.dtype != _F32 or lse.get_device() != dev:
            raise ValueError("lse must be fp32 (T, HQ) on q's device")
        lse_ptr, ldl = lse.data_ptr(), _row_stride(lse, "lse")
    max_q = 0 if max_q is None else max_q
    desc = _pack_attn(*fields, rows, hq, prefix_len, max_q, dim ** -0.5 if scale is None else scale,
                      _lib.default_flags() | (0 if causal else _lib.PAGED_FULL), q.data_ptr(), ldq, out.data_ptr(),
                      _row_stride(out, "out"), lse_ptr, ldl)
    key = (dev, rows, hq, hkv, dim, fields[0], prefix_len > 0, max_q, q_starts is None)
    need = _WORKSPACE.get(key)
    if need is None:
        if len(_WORKSPACE) >= 4096:
            _WORKSPACE.clear()
        need = _WORKSPACE[key] = _on_device(dev, _workspace_bytes, desc)
    ws = torch.empty(need, device=q.device, dtype=torch.uint8)
    _lib.check(_on_device(dev, _lib.load().bq_paged_attention, desc, ws.data_ptr(), need,
                          torch._C._cuda_getCurrentRawStream(dev)), "bq_paged_attention")
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
