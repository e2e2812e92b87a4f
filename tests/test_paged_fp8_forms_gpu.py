"""Which kernel answers a call over an 8-bit cache, and the uses that the size of a call would leave to one of them:
strides, far offsets, graphs, unusual queries and bad pages in the kernel for many rows; every division of a block's
rows in the append."""

import ctypes

import pytest
import torch

from breeze_b200 import _lib
from tests import paged_fp8_cases as pc
from tests import test_paged_fp8_edges_gpu as edges
from tests import test_paged_fp8_gpu as base
from tests.test_paged_fp8_gpu import DEV, _api, _clean_status, table_room, where  # noqa: F401

pytestmark = pytest.mark.gpu
BF, F16, E8 = pc.BF, pc.F16, pc.E8


def form(q, k, v, ks, vs, table, lens, q_starts=None, max_q=None, **_):
    """"cluster" (one launch, no workspace), "few" or "many" (their partial results' sizes)."""
    P = _api()
    fields = P._cache_fields(0, q.shape[0], P._rows_dtype(q), k, v, ks, vs, table, lens, q_starts)
    dim = fields[2]
    ldq = q.stride(0) if q.shape[0] > 1 else q.shape[1]
    desc = P._pack_attn(*fields, q.shape[0], q.shape[1] // dim, max_q or 0, 0.1, 0, 0, q.data_ptr(), ldq, q.data_ptr(), ldq, 0, 0)
    size = ctypes.c_size_t(0)
    assert _lib.load().bq_paged8_attention_workspace_bytes(desc, ctypes.byref(size)) == 0
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return "cluster" if size.value == 0 else "many" if size.value > 2 * sms * 256 * dim * 4 else "few"


def case_form(c, **kw):
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    return form(d["q"], *where(d), q_starts=None if c["starts"] is None else c["starts"].to(DEV), **kw)


@pytest.mark.parametrize("room,new,want", [(0, None, "cluster"), (0, [6, 5], "cluster"), (4096, None, "few"), (4096, [6, 5], "few"),
                                           (0, [16, 16], "few"), (0, [16, 17], "many"), (4096, [40, 90], "many")])
def test_the_form_of_a_call(room, new, want):
    """Two query heads per kv head: 16 rows and less, 32 and less, more; a table's room tells the first two apart."""
    c = pc.batch([700, 260], new, 4, 2, 128, 32, 16, BF, seed=1)
    c["table"] = torch.nn.functional.pad(c["table"], (0, room), value=-1)
    assert case_form(c) == want


@pytest.fixture
def many(monkeypatch):
    """Attention calls with a hint that sends them to the kernel for many rows."""
    P = _api()
    plain = P.paged_attention_fp8

    def call(*args, **kw):
        kw["max_q"] = 1000
        assert form(*args, **kw) == "many"
        return plain(*args, **kw)

    monkeypatch.setattr(P, "paged_attention_fp8", call)


def test_many_rows_strides(many):
    base.test_strides([21, 64])
    base.test_strides([60, 131])


def test_many_rows_offsets_behind_four_gigabytes(many, table_room):
    base.test_offsets_behind_four_gigabytes([3, 70], table_room)


def test_many_rows_captured_graphs(many, table_room):
    base.test_captured_graphs([4, 80], table_room)


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_many_rows_an_unusual_query_stays_in_its_row(many, what, table_room):
    base.test_an_unusual_query_stays_in_its_row([40, 30], what, table_room)


def test_many_rows_a_row_whose_scores_are_all_minus_infinity(many, table_room):
    base.test_a_row_whose_scores_are_all_minus_infinity([40, 30], table_room)


def test_many_rows_lengths_behind_the_table_and_bad_pages_are_reported(many):
    base.test_lengths_behind_the_table_and_bad_pages_are_reported()


def test_many_rows_two_streams_at_once(many):
    base.test_two_streams_at_once([30, 200])


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("new", [[6, 5], [40, 90]])
def test_large_scores_and_values_that_are_nan(new, dtype, table_room):
    """A NaN value at a sequence's last position: its last row shows it, in that entry alone, and no other row."""
    c = table_room(pc.batch([700, 260], new, 4, 2, 128, 32, 16, dtype, seed=3, levels=2))
    c["q"][:] = 1.0
    edges.fill(c, lambda b, p: 1.75 if p == 5 else 0.5)
    for b, n in enumerate((700, 260)):
        pc.bits(c["v"])[c["table"][b, (n - 1) // 32], :, (n - 1) % 32, 9] = 0x7F
    out, _ = base.run(c, scale=1e9 / (1.75 * 128 * edges.LOG2E))
    o = out.double().reshape(c["rows"], 4, 128)
    for r, b, n in edges.visible(c):
        want = edges.gathered(c, c["v"], c["vs"], b, n)[:, 5].repeat_interleave(2, 0)
        if n == (700, 260)[b]:
            want[:, 9] = float("nan")
        assert torch.equal(o[r].nan_to_num(-999.0), want.nan_to_num(-999.0)), r


# Each group of lanes holds 2, 4 or 8 rows of a block: by the block's size and the head's.
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,block,dtype,cdt,normed", [
    ([300, 129, 64], [300, 100, 64], 5, 5, 128, 64, 64, BF, torch.float32, True),   # 4 rows; starts inside a block
    ([200, 70, 131], [3, 15, 17], 8, 2, 128, 128, 64, F16, F16, False),             # 4; fewer rows than groups
    ([300, 129, 128], [300, 100, 128], 6, 3, 64, 128, 128, BF, BF, True),           # 4
    ([200, 400, 31], [5, 33, 31], 4, 1, 64, 1024, 128, F16, torch.float32, True),   # 4
    ([260, 129], [260, 40], 3, 1, 128, 128, 128, BF, torch.float32, True),          # 8; fp32 tables
    ([200, 140], [190, 2], 4, 2, 128, 256, 128, F16, F16, True),                    # 8
    ([100, 50], [90, 50], 2, 1, 64, 16, 16, BF, BF, True),                          # 2; four heads to a CTA, two of them there
    ([77, 200], [77, 3], 6, 3, 128, 32, 32, F16, torch.float32, True),              # 2
])
def test_append_by_every_division_of_a_block(lens, new, hq, hkv, dim, page, block, dtype, cdt, normed, layout):
    base.test_append(lens, new, hq, hkv, dim, page, block, dtype, cdt, normed, layout)


@pytest.mark.parametrize("page,block,dim", [(64, 64, 128), (128, 128, 64)])
def test_append_and_attend_in_large_blocks(page, block, dim):
    """A prompt, a chunk and single tokens in the layout that a decode stack takes by default (64 positions to a scale)."""
    hq, hkv, lens = 4, 2, torch.zeros(2, dtype=torch.int32)
    P, g = _api(), torch.Generator().manual_seed(12)
    table = torch.randperm(16, generator=g).reshape(2, 8).to(torch.int32)
    k, v = (torch.full((16, hkv, page, dim), 0x7F, dtype=torch.uint8, device=DEV).view(pc.F8) for _ in range(2))
    ks, vs = (torch.full((16, hkv, page // block), 255, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2))
    cos, sin = base.tables(400, dim, BF, g)
    norms = [(1 + 0.3 * torch.randn(dim, generator=g)).to(BF) for _ in range(2)]
    for new in ([150, 40], [70, 100], None, [3, 1], None):
        rows = 2 if new is None else sum(new)
        lens = lens + torch.tensor(new or [1, 1], dtype=torch.int32)
        starts = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32)
        qkv = (torch.randn(rows, (hq + 2 * hkv) * dim, generator=g) * 2).to(BF)
        c = dict(k=k.cpu(), v=v.cpu(), ks=ks.cpu(), vs=vs.cpu(), table=table, lens=lens, starts=starts, rows=rows, hq=hq, hkv=hkv,
                 dim=dim, page=page, block=block, dtype=BF)
        d = dict(k=k, v=v, ks=ks, vs=vs, table=table.to(DEV), lens=lens.to(DEV))
        before = base.caches(d)
        q = base.append(c, d, qkv, cos, sin, norms, 1e-6)
        after = base.caches(d)
        base.check_append(c, before, after, q, qkv, cos, sin, norms, 1e-6)
        c.update(k=after[0], v=after[1], ks=after[2], vs=after[3], q=q)
        lse = torch.empty(rows, hq, device=DEV)
        out = P.paged_attention_fp8(q.to(DEV), *where(d), q_starts=None if starts is None else starts.to(DEV), lse=lse,
                                    max_q=None if new is None else max(new))
        base.compare(c, out.cpu(), lse.cpu())
