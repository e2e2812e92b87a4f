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
import math
import operator
import warnings

import torch

from .. import _lib

_I32, _F32 = torch.int32, torch.float32
_UNIT = (1,)  # stride of a contiguous vector
_CACHE_DT = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_pack_append = _lib.packer(_lib.PagedAppendDesc)
_pack_attn = _lib.packer(_lib.PagedAttnDesc)
_bound = None


class _Python:
    """Stands in for compiled calls that do not load: the functions below check and launch every call themselves."""

    @staticmethod
    def append(*args):
        return None

    attention = append8 = attention8 = read8 = append


def _native():
    """The compiled calls (csrc/bind_paged.cpp), bound to the loaded library:
    plain calls in a few microseconds of host time. They answer None where
    something is to be refused or is out of the ordinary (another device is
    current): then the functions below check, raise or launch."""
    global _bound
    if _bound is None:
        lib = _lib.load()
        try:
            from .. import _paged_bind

            built_for = _paged_bind.torch_version
            if built_for != torch.__version__:
                raise ImportError(f"built for torch {built_for}, not {torch.__version__}")
        except ImportError as e:
            warnings.warn(f"breeze_b200/_paged_bind.so does not load ({e}): calls of the paged operators take 6 us more. "
                          "Build it with `python breeze-tts-2_b200/build.py`", RuntimeWarning, stacklevel=2)
            _bound = _Python
            return _bound
        _paged_bind.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.bq_paged_append, lib.bq_paged_attention, lib.bq_paged_attention_workspace_bytes)))
        _paged_bind.bind8(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.bq_paged8_append, lib.bq_paged8_attention, lib.bq_paged8_attention_workspace_bytes, lib.bq_paged8_read)))
        _bound = _paged_bind
    return _bound


def _count(value, name: str) -> int:
    """A number of positions or rows, as the descriptors hold it."""
    n = operator.index(value)
    if not 0 <= n < 2 ** 31:
        raise ValueError(f"{name} must be from 0 to 2^31 - 1 (got {n})")
    return n


def _real(value, name: str) -> float:
    """A number that fp32 can hold."""
    if not math.isfinite(value) or abs(value) >= 3.4e38:
        raise ValueError(f"{name} must be finite in fp32 (got {value})")
    return value


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Row stride of a 2-D tensor with contiguous rows (a dimension of size one has no stride)."""
    st = t.stride()
    if len(st) != 2 or (st[1] != 1 and t.shape[1] != 1):
        raise ValueError(f"{name} must be a 2-D tensor with unit stride in the last dimension")
    return st[0] if t.shape[0] > 1 else t.shape[1]


def _cache_fields(dev: int, dtype: torch.dtype, rows: int, k_pages, v_pages, page_table, seq_lens, q_starts):
    """The leading fields of both descriptors, after the checks both calls share."""
    if dev < 0:
        raise RuntimeError("breeze_b200 kernels need CUDA tensors (there is no CPU path)")
    if not (k_pages.get_device() == v_pages.get_device() == page_table.get_device() == seq_lens.get_device() == dev):
        raise RuntimeError("tensors on different devices: the rows, the cache and the lengths must share one")
    if not (k_pages.dtype == v_pages.dtype == dtype):
        raise ValueError(f"rows and pages must have one dtype (got {dtype}, {k_pages.dtype}, {v_pages.dtype})")
    code = _CACHE_DT.get(dtype)
    if code is None:
        raise ValueError(f"paged caches are bf16 or fp16 (got {dtype})")
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be (pages, HKV, page size, D) of one shape")
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    ts = page_table.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
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
    if pages == 0 or hkv == 0 or dim == 0 or columns == 0 or batch == 0:
        raise ValueError("empty cache or batch")
    return (batch, hkv, dim, size, pages, columns, code, 0, k_pages.data_ptr(), k0, k1, k2, v_pages.data_ptr(), v0, v1, v2,
            page_table.data_ptr(), ts[0] if batch > 1 else columns, seq_lens.data_ptr(), starts)


def _launch(dev: int, what: str, call, *args) -> None:
    """call(*args, stream): a library entry on the current stream of ``dev``, made the current device for it."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch._C._cuda_getDevice():
        rc = call(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = call(*args, stream)
    if rc:
        _lib.check(rc, what)


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor, q_starts: torch.Tensor | None = None,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv (T, (HQ + 2 HKV) D) rows [q heads | k heads | v heads] of the new
    tokens -> q (T, HQ D), normed and rotated; k (normed, rotated) and v written
    into their pages. ``cos`` / ``sin``: (positions, D) tables (fp32 or the
    cache's dtype), row p for cache position p, both halves given as rotate_half
    takes them. The math is fp32 with one rounding at the end. ``out`` may be
    ``qkv[:, :HQ * D]`` itself, and else shares no memory with ``qkv``. Tokens of an unused batch slot (seq_lens[b] less
    than its new tokens) are skipped where their position would be negative."""
    done = (_bound or _native()).append(qkv, cos, sin, k_pages, v_pages, page_table, seq_lens, q_starts, q_norm_w, k_norm_w,
                                        eps, out, _lib.default_flags())
    if done is not None:
        return done if done.__class__ is not int else _lib.check(done, "bq_paged_append")
    ldqkv = _row_stride(qkv, "qkv")
    rows, width = qkv.shape
    dev, dtype = qkv.get_device(), qkv.dtype
    fields = _cache_fields(dev, dtype, rows, k_pages, v_pages, page_table, seq_lens, q_starts)
    hkv, dim = fields[1], fields[2]
    hq = width // dim - 2 * hkv
    if hq <= 0 or (hq + 2 * hkv) * dim != width:
        raise ValueError(f"qkv width {width} does not split into q, k and v heads of {dim}")
    ldcs, cs_dtype, cs_shape = _row_stride(cos, "cos"), cos.dtype, cos.shape
    if cs_shape[1] != dim or sin.shape != cs_shape or sin.dtype != cs_dtype or _row_stride(sin, "sin") != ldcs:
        raise ValueError("cos and sin must be (positions, D) tables of one shape, stride and dtype")
    if cs_dtype != dtype and cs_dtype != _F32:
        raise ValueError(f"cos and sin must be fp32 or the cache's dtype (got {cs_dtype})")
    if not (cos.get_device() == sin.get_device() == dev):
        raise RuntimeError("cos and sin are on another device than qkv")
    qn = kn = 0
    if q_norm_w is not None and k_norm_w is not None:
        for t in (q_norm_w, k_norm_w):
            if t.dtype != dtype or t.shape != (dim,) or t.stride() != _UNIT or t.get_device() != dev:
                raise ValueError("norm weights must be contiguous (D,) vectors of the cache's dtype and device")
        qn, kn = q_norm_w.data_ptr(), k_norm_w.data_ptr()
    elif q_norm_w is not None or k_norm_w is not None:
        raise ValueError("q_norm_w and k_norm_w go together")
    ldq = hq * dim
    if out is None:
        out = qkv.new_empty((rows, ldq))
    elif out.shape != (rows, ldq) or out.dtype != dtype or out.get_device() != dev:
        raise ValueError("out must be (T, HQ D) of the cache's dtype and device")
    else:
        ldq = _row_stride(out, "out")
    desc = _pack_append(*fields, rows, hq, _lib._DT[cs_dtype], cs_shape[0], _real(eps, "eps"), _lib.default_flags(), qkv.data_ptr(), ldqkv,
                        cos.data_ptr(), sin.data_ptr(), ldcs, qn, kn, out.data_ptr(), ldq)
    _launch(dev, "bq_paged_append", _lib.load().bq_paged_append, desc)
    return out


def _workspace_bytes_of(entry):
    """A *_workspace_bytes entry as _launch calls it, with a stream behind the arguments."""
    return lambda desc, need, stream: entry(desc, need)


def _attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, causal, max_q, out, lse, extra=0):
    flags = _lib.default_flags() | extra
    if not causal:
        flags |= _lib.PAGED_FULL
    done = (_bound or _native()).attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, max_q, out,
                                           lse, flags)
    if done is not None:
        return done if done.__class__ is not int else _lib.check(done, "bq_paged_attention")
    ldq = _row_stride(q, "q")
    rows, width = q.shape
    dev, dtype = q.get_device(), q.dtype
    fields = _cache_fields(dev, dtype, rows, k_pages, v_pages, page_table, seq_lens, q_starts)
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
    desc = _pack_attn(*fields, rows, hq, _count(prefix_len, "prefix_len"), max_q, scale, flags, q.data_ptr(),
                      ldq, out.data_ptr(), ldo, lse_ptr, ldl)
    size = ctypes.c_size_t(0)
    _launch(dev, "bq_paged_attention_workspace_bytes", _workspace_bytes_of(_lib.load().bq_paged_attention_workspace_bytes), desc,
            ctypes.byref(size))
    need = size.value
    ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    _launch(dev, "bq_paged_attention", _lib.load().bq_paged_attention, desc, ws.data_ptr() if need else None, need)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, q_starts: torch.Tensor | None = None, scale: float | None = None,
                    causal: bool = True, max_q: int | None = None, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None) -> torch.Tensor:
    """q (T, HQ D) of the new tokens (already in the cache: paged_append first)
    -> (T, HQ D). Row i of the n new rows of sequence b sees positions
    [0, seq_lens[b] - n + i + 1); with ``causal=False`` all seq_lens[b]. A row
    that sees none gets zeros, one whose scores are all -inf gets NaN; infinite or NaN keys and values at positions it does
    not see stay without effect. Query head h reads kv head h // (HQ / HKV).
    ``scale`` defaults to D^-0.5. ``max_q``: most new tokens of one sequence, a
    hint that picks the kernel (0 or None: T / B rounded up; say it where they differ:
    a prompt among many running streams is slow in the kernel for few rows). ``lse`` (T, HQ) fp32
    receives log(sum(exp(scores))), -inf for a row that sees nothing."""
    return _attention(q, k_pages, v_pages, page_table, seq_lens, 0, q_starts, scale, causal, max_q, out, lse)


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                     seq_lens: torch.Tensor, prefix_len: int, q_starts: torch.Tensor | None = None,
                     scale: float | None = None, causal: bool = True, max_q: int | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                     always: bool = False) -> torch.Tensor:
    """paged_attention for a batch that shares its first ``prefix_len``
    positions (a multiple of the page size): of every sequence with new rows the
    first prefix_len / page size table entries name the same pages, as far as the
    sequence goes (an unused slot's entries may hold anything). They are read once
    for all rows together, through the table row of the longest such sequence, and
    joined with each sequence's own positions, where that pays (a short prefix of
    few sequences is read by each; ``always=True`` shares it all the same); the
    value is paged_attention's."""
    return _attention(q, k_pages, v_pages, page_table, seq_lens, prefix_len, q_starts, scale, causal, max_q, out, lse,
                      _lib.PAGED_SHARE if always else 0)
