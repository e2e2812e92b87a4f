"""Refusals of the paged-cache operators, on the host: no GPU is touched."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from breeze_b200 import _lib as L
from breeze_b200.fused import paged
from oracle import paged as op
from tests import paged_cases as pc

HEADER = (Path(__file__).resolve().parents[1] / "include" / "breeze_b200.h").read_text()


def _fill(d):
    d.B, d.HKV, d.D, d.page_size, d.num_pages, d.max_pages, d.dtype = 2, 4, 128, 64, 10, 5, L.DT_BF16
    d.k_pages = d.v_pages = d.page_table = d.seq_lens = 4096
    d.k_page_stride = d.v_page_stride = 4 * 64 * 128
    d.k_head_stride = d.v_head_stride = 64 * 128
    d.k_slot_stride = d.v_slot_stride = 128
    d.ld_table, d.T, d.HQ = 5, 2, 8
    return d


def attn(**kw):
    d = _fill(L.PagedAttnDesc())
    d.q = d.out = 4096
    d.ldq = d.ldo = 8 * 128
    d.scale = 0.1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def append(**kw):
    d = _fill(L.PagedAppendDesc())
    d.qkv = d.cos = d.sin = d.q_out = 4096
    d.ldqkv, d.ldcs, d.ldq, d.rope_rows, d.cs_dtype = 16 * 128, 128, 8 * 128, 320, L.DT_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_descriptors_have_the_headers_layout():
    kv = 8 * 4 + 2 * 4 * 8 + 4 * 8
    assert L.PagedAppendDesc.T.offset == kv and L.PagedAttnDesc.T.offset == kv
    assert ctypes.sizeof(L.PagedAppendDesc) == kv + 6 * 4 + 9 * 8
    assert ctypes.sizeof(L.PagedAttnDesc) == kv + 6 * 4 + 6 * 8
    for desc in (L.PagedAppendDesc, L.PagedAttnDesc):  # packed values and a filled Structure are the same bytes
        values = [i + 1 if t is not ctypes.c_float else 0.5 for i, (_, t) in enumerate(desc._fields_)]
        assert L.packer(desc)(*values) == bytes(desc(*values))
    for name, value in (("BQ_PAGED_FULL", L.PAGED_FULL), ("BQ_PAGED_SHARE", L.PAGED_SHARE), ("BQ_DEVERR_PAGE", L.BQ_DEVERR_PAGE)):
        assert int(re.search(rf"#define {name} (\d+)u", HEADER).group(1)) == value


SHARED = [
    (dict(dtype=L.DT_F32), L.BQ_ERR_FORMAT, "bf16 or fp16"),
    (dict(D=96), L.BQ_ERR_SHAPE, "head dim"),
    (dict(page_size=8), L.BQ_ERR_SHAPE, "page size"),
    (dict(page_size=48), L.BQ_ERR_SHAPE, "page size"),
    (dict(page_size=2048), L.BQ_ERR_SHAPE, "page size"),
    (dict(B=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(num_pages=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(max_pages=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(T=-1), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(HQ=6), L.BQ_ERR_SHAPE, "multiple"),
    (dict(HQ=0), L.BQ_ERR_SHAPE, "multiple"),
    (dict(HKV=0), L.BQ_ERR_SHAPE, "multiple"),
    (dict(T=3), L.BQ_ERR_SHAPE, "q_starts"),
    (dict(T=2 ** 28, q_starts=4096), L.BQ_ERR_SHAPE, "too many"),
    (dict(max_pages=2 ** 25, ld_table=2 ** 25), L.BQ_ERR_SHAPE, "2\\^30"),
    (dict(ld_table=4), L.BQ_ERR_SHAPE, "table stride"),
    (dict(k_pages=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(seq_lens=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(k_slot_stride=64), L.BQ_ERR_SHAPE, "strides"),
    (dict(v_head_stride=0), L.BQ_ERR_SHAPE, "strides"),
    (dict(v_page_stride=4 * 64 * 128 + 4), L.BQ_ERR_ALIGN, "multiples of 8"),
    (dict(v_pages=4104), L.BQ_ERR_ALIGN, "16-byte"),
]


@pytest.mark.parametrize("change,code,text", SHARED)
def test_shared_refusals(lib, change, code, text):
    n = ctypes.c_size_t(0)
    assert lib.bq_paged_append(ctypes.byref(append(**change)), None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged_attention(ctypes.byref(attn(**change)), None, 0, None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged_attention_workspace_bytes(ctypes.byref(attn(**change)), ctypes.byref(n)) == code


@pytest.mark.parametrize("change,code,text", [
    (dict(q=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(ldq=1000), L.BQ_ERR_SHAPE, "row strides"),
    (dict(ldo=8 * 128 + 4), L.BQ_ERR_ALIGN, "16-byte"),
    (dict(lse=4096, ldl=7), L.BQ_ERR_SHAPE, "lse"),
    (dict(scale=0.0), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=-1.0), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=float("nan")), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=float("inf")), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(prefix_len=63), L.BQ_ERR_SHAPE, "multiple of the page size"),
    (dict(prefix_len=-64), L.BQ_ERR_SHAPE, "multiple of the page size"),
    (dict(prefix_len=6 * 64), L.BQ_ERR_SHAPE, "exceeds"),
])
def test_attention_refusals(lib, change, code, text):
    assert lib.bq_paged_attention(ctypes.byref(attn(**change)), None, 0, None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged_attention(None, None, 0, None) == L.BQ_ERR_INVALID_ARG
    assert lib.bq_paged_attention_workspace_bytes(ctypes.byref(attn()), None) == L.BQ_ERR_INVALID_ARG


@pytest.mark.parametrize("change,code,text", [
    (dict(qkv=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(cs_dtype=L.DT_F16), L.BQ_ERR_INVALID_ARG, "cos / sin"),
    (dict(q_norm=4096), L.BQ_ERR_INVALID_ARG, "together"),
    (dict(ldqkv=15 * 128), L.BQ_ERR_SHAPE, "ldqkv"),
    (dict(ldq=7 * 128), L.BQ_ERR_SHAPE, "ldq"),
    (dict(rope_rows=0), L.BQ_ERR_SHAPE, "cos / sin"),
    (dict(ldcs=64), L.BQ_ERR_SHAPE, "cos / sin"),
    (dict(qkv=4098), L.BQ_ERR_ALIGN, "16-byte"),
    (dict(ldq=8 * 128 + 2), L.BQ_ERR_ALIGN, "16-byte"),
    (dict(q_norm=4096, k_norm=4100), L.BQ_ERR_ALIGN, "16-byte"),
])
def test_append_refusals(lib, change, code, text):
    assert lib.bq_paged_append(ctypes.byref(append(**change)), None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged_append(None, None) == L.BQ_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    c = pc.batch([5, 9], None, 2, 1, 64, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_append(torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(9, 64), torch.zeros(9, 64), c["k"], c["v"],
                           c["table"], c["lens"])


def test_the_compiled_calls_leave_what_is_not_plain_to_python():
    native = paged._native()
    c = pc.batch([5, 9], None, 2, 1, 64, 16)
    assert native.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], 0, None, None, None, None, None, 0) is None  # no GPU
    assert native.append(torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(9, 64), torch.zeros(9, 64), c["k"], c["v"],
                         c["table"], c["lens"], None, None, None, 1e-6, None, 0) is None
    assert native.attention() is None and native.attention(*[None] * 12) is None
    assert native.append(c["q"]) is None and native.append(*["x"] * 13) is None
    with pytest.raises(TypeError, match="three addresses"):
        native.bind(1)
    with pytest.raises(ValueError, match="address 0"):
        native.bind(1, 0, 1)


def test_oracle_agrees_with_the_dense_step():
    """A paged batch whose rows are all at one position is the static cache's step."""
    from oracle import attention as oa

    b, hq, hkv, dim, page, pos = 3, 4, 2, 64, 16, 37
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(b, (hq + 2 * hkv) * dim, generator=g).to(torch.bfloat16)
    k0 = torch.randn(b, hkv, 48, dim, generator=g).to(torch.bfloat16)
    v0 = torch.randn(b, hkv, 48, dim, generator=g).to(torch.bfloat16)
    ang = torch.arange(48)[:, None] * 1e4 ** (-torch.arange(0, dim, 2) / dim)
    cos, sin = torch.cat([ang, ang], -1).cos().to(torch.bfloat16), torch.cat([ang, ang], -1).sin().to(torch.bfloat16)
    dense, kd, vd = oa.attention_step(qkv, cos[pos:pos + 1], sin[pos:pos + 1], pos, k0.clone(), v0.clone(), torch.zeros(b, 48))
    table = torch.arange(9).reshape(3, 3).tolist()
    kp, vp = (t.reshape(b, hkv, 3, page, dim).transpose(1, 2).reshape(9, hkv, page, dim).clone() for t in (k0, v0))
    lens = [pos + 1] * b
    q, written, _ = op.append(qkv, cos, sin, kp, vp, table, lens, None)
    for (pg, slot), (_, k, v) in written.items():
        kp[pg, :, slot], vp[pg, :, slot] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    ref = op.attention(q.reshape(b, -1), kp, vp, table, lens, None)
    assert (ref["out"].reshape(b, -1) - dense.double()).abs().max() < 2e-2
    assert torch.equal(vp[table[0][2], :, pos % page], vd[0, :, pos])


def test_registers_move_by_one_instruction_per_warpgroup():
    """setmaxnreg is defined only where all warps of a warpgroup execute the same
    one: a second place in the code means that some warps take another."""
    for src in (Path(__file__).resolve().parents[1] / "breeze-tts-2_b200" / "csrc").glob("*.cu"):
        text = src.read_text()
        for kind in ("inc", "dec"):
            assert len(re.findall(rf'"setmaxnreg\.{kind}\.', text)) <= 1, (src.name, kind)


def test_a_scale_that_is_infinite_in_base_2_is_refused(lib):
    n = ctypes.c_size_t(0)
    for scale in (2.4e38, 2.9e38, 3.4e38):  # finite, but not times log2(e) = 1.44
        assert lib.bq_paged_attention_workspace_bytes(ctypes.byref(attn(scale=scale)), ctypes.byref(n)) == L.BQ_ERR_INVALID_ARG
        assert "scale" in L.last_error()


def test_a_negative_hint_is_refused(lib):
    n = ctypes.c_size_t(0)
    assert lib.bq_paged_attention_workspace_bytes(ctypes.byref(attn(max_q=-1)), ctypes.byref(n)) == L.BQ_ERR_INVALID_ARG
    assert "max_q" in L.last_error()
