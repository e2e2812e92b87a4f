"""8-bit paged cache on the host: refusals, descriptors and the oracle. No GPU is touched."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from breeze_b200 import _lib as L
from breeze_b200.fused import paged_fp8 as P
from oracle import paged8 as o8
from tests import paged_fp8_cases as pc

HEADER = (Path(__file__).resolve().parents[1] / "include" / "breeze_b200.h").read_text()


def _fill(d):
    d.B, d.HKV, d.D, d.page_size, d.num_pages, d.max_pages, d.block, d.dtype = 2, 4, 128, 64, 10, 5, 32, L.DT_BF16
    d.k_pages = d.v_pages = d.k_scales = d.v_scales = d.page_table = d.seq_lens = 4096
    d.k_page_stride = d.v_page_stride = 4 * 64 * 128
    d.k_head_stride = d.v_head_stride = 64 * 128
    d.k_slot_stride = d.v_slot_stride = 128
    d.k_scale_page_stride = d.v_scale_page_stride = 8
    d.k_scale_head_stride = d.v_scale_head_stride = 2
    d.ld_table, d.T = 5, 2
    return d


def _set(d, kw):
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def attn(**kw):
    d = _fill(L.Paged8AttnDesc())
    d.HQ, d.q, d.out, d.ldq, d.ldo, d.scale = 8, 4096, 4096, 8 * 128, 8 * 128, 0.1
    return _set(d, kw)


def append(**kw):
    d = _fill(L.Paged8AppendDesc())
    d.HQ, d.qkv, d.cos, d.sin, d.q_out = 8, 4096, 4096, 4096, 4096
    d.ldqkv, d.ldcs, d.ldq, d.rope_rows, d.cs_dtype = 16 * 128, 128, 8 * 128, 320, L.DT_BF16
    return _set(d, kw)


def read(**kw):
    d = _fill(L.Paged8ReadDesc())
    d.k_out = d.v_out = 4096
    d.k_out_row_stride = d.v_out_row_stride = 4 * 128
    d.k_out_head_stride = d.v_out_head_stride = 128
    return _set(d, kw)


def test_descriptors_have_the_headers_layout():
    kv = 8 * 4 + 2 * 4 * 8 + 2 * 3 * 8 + 4 * 8
    for desc in (L.Paged8AppendDesc, L.Paged8AttnDesc, L.Paged8ReadDesc):
        assert desc.T.offset == kv
        values = [i + 1 if t is not ctypes.c_float else 0.5 for i, (_, t) in enumerate(desc._fields_)]
        assert L.packer(desc)(*values) == bytes(desc(*values))
    assert ctypes.sizeof(L.Paged8AppendDesc) == kv + 6 * 4 + 9 * 8
    assert ctypes.sizeof(L.Paged8AttnDesc) == kv + 6 * 4 + 6 * 8
    assert ctypes.sizeof(L.Paged8ReadDesc) == kv + 2 * 4 + 6 * 8
    body = re.search(r"typedef struct bq_paged8_kv \{(.*?)\} bq_paged8_kv;", HEADER, re.S).group(1)
    names = re.findall(r"(\w+)(?:\[\d\])?[,;]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
    mine = [re.sub(r"_(page|head|slot)_stride", "_stride", n) for n, _ in L.Paged8AttnDesc._fields_[:26]]
    assert list(dict.fromkeys(mine)) == names


SHARED = [
    (dict(dtype=5), L.BQ_ERR_FORMAT, "bf16 or fp16"),
    (dict(D=96), L.BQ_ERR_SHAPE, "head dim"),
    (dict(page_size=8), L.BQ_ERR_SHAPE, "page size"),
    (dict(page_size=48), L.BQ_ERR_SHAPE, "page size"),
    (dict(page_size=2048), L.BQ_ERR_SHAPE, "page size"),
    (dict(block=8), L.BQ_ERR_SHAPE, "positions per scale"),
    (dict(block=48), L.BQ_ERR_SHAPE, "positions per scale"),
    (dict(block=128), L.BQ_ERR_SHAPE, "positions per scale"),
    (dict(block=256, page_size=1024), L.BQ_ERR_SHAPE, "positions per scale"),
    (dict(block=0), L.BQ_ERR_SHAPE, "positions per scale"),
    (dict(B=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(num_pages=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(max_pages=0), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(T=-1), L.BQ_ERR_SHAPE, "bad batch"),
    (dict(HKV=0), L.BQ_ERR_SHAPE, "kv heads"),
    (dict(T=3), L.BQ_ERR_SHAPE, "q_starts"),
    (dict(T=2 ** 28, q_starts=4096), L.BQ_ERR_SHAPE, "too many"),
    (dict(max_pages=2 ** 25, ld_table=2 ** 25), L.BQ_ERR_SHAPE, "2\\^30"),
    (dict(ld_table=4), L.BQ_ERR_SHAPE, "table stride"),
    (dict(k_pages=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(v_scales=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(seq_lens=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(k_slot_stride=64), L.BQ_ERR_SHAPE, "strides"),
    (dict(v_head_stride=0), L.BQ_ERR_SHAPE, "strides"),
    (dict(k_scale_head_stride=1), L.BQ_ERR_SHAPE, "scale strides"),
    (dict(v_scale_page_stride=0), L.BQ_ERR_SHAPE, "scale strides"),
    (dict(v_page_stride=4 * 64 * 128 + 8), L.BQ_ERR_ALIGN, "multiples of 16"),
    (dict(v_pages=4104), L.BQ_ERR_ALIGN, "16-byte"),
]


@pytest.mark.parametrize("change,code,text", SHARED)
def test_shared_refusals(lib, change, code, text):
    n = ctypes.c_size_t(0)
    assert lib.bq_paged8_append(ctypes.byref(append(**change)), None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged8_attention(ctypes.byref(attn(**change)), None, 0, None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged8_attention_workspace_bytes(ctypes.byref(attn(**change)), ctypes.byref(n)) == code
    if "T" not in change or change["T"] < 2 ** 28:  # reading back has no query heads
        assert lib.bq_paged8_read(ctypes.byref(read(**change)), None) == code
        assert re.search(text, L.last_error())


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=L.DT_F32), L.BQ_ERR_FORMAT, "bf16 or fp16"),
    (dict(HQ=6), L.BQ_ERR_SHAPE, "multiple"),
    (dict(HQ=0), L.BQ_ERR_SHAPE, "multiple"),
    (dict(q=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(ldq=1000), L.BQ_ERR_SHAPE, "row strides"),
    (dict(ldo=8 * 128 + 4), L.BQ_ERR_ALIGN, "16-byte"),
    (dict(lse=4096, ldl=7), L.BQ_ERR_SHAPE, "lse"),
    (dict(scale=0.0), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=-1.0), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=float("nan")), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(scale=2.9e38), L.BQ_ERR_INVALID_ARG, "scale"),
    (dict(max_q=-1), L.BQ_ERR_INVALID_ARG, "max_q"),
])
def test_attention_refusals(lib, change, code, text):
    n = ctypes.c_size_t(0)
    assert lib.bq_paged8_attention(ctypes.byref(attn(**change)), None, 0, None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged8_attention_workspace_bytes(ctypes.byref(attn(**change)), ctypes.byref(n)) == code
    assert lib.bq_paged8_attention(None, None, 0, None) == L.BQ_ERR_INVALID_ARG
    assert lib.bq_paged8_attention_workspace_bytes(ctypes.byref(attn()), None) == L.BQ_ERR_INVALID_ARG


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=L.DT_F32), L.BQ_ERR_FORMAT, "bf16 or fp16"),
    (dict(HQ=6), L.BQ_ERR_SHAPE, "multiple"),
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
    assert lib.bq_paged8_append(ctypes.byref(append(**change)), None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged8_append(None, None) == L.BQ_ERR_INVALID_ARG


@pytest.mark.parametrize("change,code,text", [
    (dict(k_out=0), L.BQ_ERR_INVALID_ARG, "non-NULL"),
    (dict(v_out_row_stride=64), L.BQ_ERR_SHAPE, "strides of k_out"),
    (dict(k_out_head_stride=132), L.BQ_ERR_ALIGN, "16-byte"),
    (dict(v_out=4100), L.BQ_ERR_ALIGN, "16-byte"),
])
def test_read_refusals(lib, change, code, text):
    assert lib.bq_paged8_read(ctypes.byref(read(**change)), None) == code
    assert re.search(text, L.last_error())
    assert lib.bq_paged8_read(None, None) == L.BQ_ERR_INVALID_ARG


def test_calls_without_rows_are_answered_on_the_host(lib):
    none = dict(T=0, q_starts=4096)
    assert lib.bq_paged8_append(ctypes.byref(append(**none)), None) == L.BQ_OK
    assert lib.bq_paged8_attention(ctypes.byref(attn(**none)), None, 0, None) == L.BQ_OK
    assert lib.bq_paged8_read(ctypes.byref(read(**none)), None) == L.BQ_OK


def test_cpu_tensors_are_refused():
    c = pc.batch([5, 9], None, 2, 1, 64, 16, 16)
    where = (c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_attention_fp8(c["q"], *where)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_append_fp8(torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(9, 64), torch.zeros(9, 64), *where)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_read_fp8(*where)


def test_the_compiled_calls_leave_what_is_not_plain_to_python():
    from breeze_b200.fused import paged

    native = paged._native()
    c = pc.batch([5, 9], None, 2, 1, 64, 16, 16)
    where = (c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"])
    assert native.attention8(c["q"], *where, None, None, None, None, None, 0) is None  # no GPU
    assert native.append8(torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(9, 64), torch.zeros(9, 64), *where, None, None,
                          None, 1e-6, None, 0) is None
    assert native.read8(*where, None, 2, L.DT_BF16, None, None, 0) is None
    for call, n in ((native.attention8, 13), (native.append8, 15), (native.read8, 12)):
        assert call() is None and call(*[None] * n) is None and call(*["x"] * n) is None
    with pytest.raises(TypeError, match="four addresses"):
        native.bind8(1)
    with pytest.raises(ValueError, match="address 0"):
        native.bind8(1, 0, 1, 1)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: reaches the checks behind the first one, never a kernel."""

    def get_device(self):
        return 0


@pytest.mark.parametrize("change,match", [
    (lambda a: a.update(k=a["k"].view(torch.uint8)), "float8_e4m3fn"),
    (lambda a: a.update(vs=a["vs"].view(torch.uint8)), "float8_e8m0fnu"),
    (lambda a: a.update(v=a["v"][:, :, :8]), "one shape"),
    (lambda a: a.update(ks=a["ks"][:3]), "pages and HKV the cache's"),
    (lambda a: a.update(ks=a["ks"][:, :, 0]), "pages and HKV the cache's"),
    (lambda a: a.update(k=a["k"].transpose(2, 3), v=a["v"].transpose(2, 3)), "last dimension of the pages"),
    (lambda a: a.update(ks=a["ks"].transpose(1, 2).contiguous().transpose(1, 2), vs=a["vs"]), "last dimension of the scales"),
    (lambda a: a.update(table=a["table"].long()), "page_table"),
    (lambda a: a.update(lens=a["lens"].long()), "seq_lens"),
    (lambda a: a.update(lens=a["lens"][:1]), "seq_lens"),
    (lambda a: a.update(q=a["q"][:1]), "q_starts"),
    (lambda a: a.update(q=a["q"].float()), "bf16 or fp16"),
    (lambda a: a.update(q=a["q"][:, :65]), "split into heads"),
    (lambda a: a.update(starts=torch.zeros(2, dtype=torch.int32)), "q_starts must be"),
    (lambda a: a.update(k=a["k"][:0], v=a["v"][:0], ks=a["ks"][:0], vs=a["vs"][:0]), "empty"),
    (lambda a: a.update(ks=torch.cat([a["ks"].view(torch.uint8)] * 2, 2)[:, :, :3].contiguous().view(pc.E8),
                        vs=torch.cat([a["vs"].view(torch.uint8)] * 2, 2)[:, :, :3].contiguous().view(pc.E8)), "divide"),
])
def test_python_refusals(change, match):
    c = pc.batch([5, 9], None, 4, 2, 64, 32, 16)
    change(c)
    t = {k: v.as_subclass(_OnGpu) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    with pytest.raises(ValueError, match=match):
        P.paged_attention_fp8(t["q"], t["k"], t["v"], t["ks"], t["vs"], t["table"], t["lens"], q_starts=t["starts"])


def test_reading_ragged_rows_needs_their_number():
    c = pc.batch([5, 9], [2, 3], 4, 2, 64, 32, 16)
    where = (c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], c["starts"])
    with pytest.raises(ValueError, match="rows"):
        P.paged_read_fp8(*where)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        P.paged_read_fp8(*where, rows=5, dtype=torch.float64)
    with pytest.raises(ValueError, match="2\\^31"):
        P.paged_read_fp8(*where, rows=-1)


def test_the_oracles_codes_are_e4m3():
    every = torch.arange(256, dtype=torch.uint8).view(pc.F8).double()
    fine = every[torch.isfinite(every)]
    assert torch.equal(o8.nearest(fine), fine)
    x = torch.cat([torch.randn(20000, dtype=torch.float64) * s for s in (1e-3, 0.1, 10.0, 150.0)]).clamp(-448, 448)
    mids = torch.sort(fine).values
    mids = (mids[1:] + mids[:-1]) / 2
    x = torch.cat([x, mids])
    assert torch.equal(o8.nearest(x), x.float().to(pc.F8).double())  # fp32 holds the midpoints exactly
    assert o8.nearest(torch.tensor([1e9, float("inf")]).double()).tolist()[0] == 448.0
    for top, e in ((448.0, 0), (448.0001, 1), (1.75, -8), (1.7501, -7), (2.0 ** -200, -60), (0.0, -60), (1e30, 60)):
        assert o8.exponent(top) == e
