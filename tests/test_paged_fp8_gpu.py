"""8-bit paged cache against the 64-bit oracle (oracle/paged8.py): attention element by
element within bounds derived from the arithmetic (attention_bounds there), codes and
scales exactly wherever fp32 arithmetic does not stand before them."""

import math

import pytest
import torch

from oracle import paged as op
from oracle import paged8 as o8
from tests import paged_fp8_cases as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F8, E8 = pc.BF, pc.F16, pc.F8, pc.E8


def _api():
    from breeze_b200.fused import paged_fp8

    return paged_fp8


def _status(clear=True):
    from breeze_b200 import _lib

    return _lib.device_status(0, clear=clear)


@pytest.fixture(autouse=True)
def _clean_status():
    _status()
    yield
    assert _status() == 0


@pytest.fixture(params=["tight", "roomy"])
def table_room(request):
    """A table that ends with its longest sequence, and one with room for another
    65536 positions: the room decides how a sequence is divided among CTAs."""

    def apply(c):
        if request.param == "roomy":
            c["table"] = torch.nn.functional.pad(c["table"], (0, 65536 // c["page"]), value=-(2 ** 30))
        return c

    return apply


def where(d):
    return d["k"], d["v"], d["ks"], d["vs"], d["table"], d["lens"]


def oracle(c, causal=True, scale=None):
    table, lens, starts = c["table"].tolist(), c["lens"].tolist(), None if c["starts"] is None else c["starts"].tolist()
    return o8.attention(c["q"], (c["k"], c["v"]), (c["ks"], c["vs"]), table, lens, starts, scale, causal)


def run(c, causal=True, scale=None, max_q=None):
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    lse = torch.full((c["rows"], c["hq"]), 7.0, device=DEV)
    out = torch.full((c["rows"], c["hq"] * c["dim"]), 3.0, device=DEV, dtype=c["dtype"])
    _api().paged_attention_fp8(d["q"], *where(d), q_starts=starts, scale=scale, causal=causal, max_q=max_q, out=out, lse=lse)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def compare(c, out, lse, causal=True, scale=None):
    ref = oracle(c, causal, scale)
    tol, ltol = o8.attention_bounds(ref, c["dim"], c["dtype"])
    rows = c["rows"] if c["starts"] is None else int(c["starts"][-1])
    o = out.double().reshape(c["rows"], c["hq"], c["dim"])
    err = (o[:rows] - ref["out"][:rows]).abs()
    assert torch.isfinite(o[:rows]).all()
    assert (err <= tol[:rows]).all(), (float((err / tol[:rows].clamp(min=1e-30)).max()), float(err.max()))
    empty = torch.isinf(ref["lse"][:rows])
    assert torch.equal(torch.isinf(lse[:rows]) & (lse[:rows] < 0), empty)
    lerr = (lse[:rows].double() - ref["lse"][:rows]).abs()[~empty]
    assert (lerr <= ltol[:rows][~empty]).all(), float(lerr.max())
    assert (o[rows:] == 3.0).all() and (lse[rows:] == 7.0).all()  # rows behind the last sequence


DECODE = [
    # lens, hq, hkv, dim, page, block, dtype
    ([1], 1, 1, 128, 16, 16, BF),
    ([1, 2, 3, 15, 16, 17, 31, 32, 33], 4, 4, 64, 16, 16, BF),
    ([63, 64, 65, 127, 128, 129], 16, 16, 128, 64, 32, BF),
    ([256, 700], 16, 16, 128, 64, 64, BF),
    ([300, 1, 0, 77], 8, 1, 128, 32, 16, F16),        # an unused batch slot
    ([515], 32, 8, 128, 128, 128, BF),
    ([2000, 5, 900], 6, 2, 64, 64, 16, F16),
    ([4097], 24, 3, 128, 256, 128, BF),
    ([1500, 1499, 1], 40, 2, 64, 1024, 64, BF),       # 20 query heads per kv head
    ([333] * 70, 2, 2, 128, 16, 16, F16),
    ([90, 17], 33, 1, 128, 32, 32, BF),               # 33 query heads on one kv head
    ([90, 200, 41], 300, 2, 64, 32, 32, F16),         # 150 query heads per kv head
]


@pytest.mark.parametrize("lens,hq,hkv,dim,page,block,dtype", DECODE)
def test_one_token_per_sequence(lens, hq, hkv, dim, page, block, dtype, table_room):
    c = table_room(pc.batch(lens, None, hq, hkv, dim, page, block, dtype, seed=hq + dim + len(lens)))
    compare(c, *run(c))


RAGGED = [
    # lens, new, hq, hkv, dim, page, block, dtype
    ([5], [5], 4, 2, 128, 16, 16, BF),
    ([40, 70, 33], [3, 1, 5], 8, 4, 128, 16, 16, BF),
    ([130, 64, 200], [7, 64, 1], 16, 8, 128, 64, 32, F16),
    ([300], [300], 4, 4, 64, 64, 64, BF),
    ([129, 0, 257, 9], [129, 0, 120, 0], 6, 2, 128, 128, 64, BF),  # sequences without new rows
    ([700, 650], [1, 260], 8, 2, 64, 32, 16, F16),
    ([513], [257], 5, 1, 128, 512, 128, BF),
    ([2, 3], [4, 3], 2, 1, 64, 16, 16, BF),                         # more rows than positions: the first see nothing
    ([1100], [150], 24, 2, 128, 64, 32, F16),                       # 12 query heads per kv head
    ([260, 31], [9, 2], 16, 1, 64, 16, 16, BF),
]


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,block,dtype", RAGGED)
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_rows(lens, new, hq, hkv, dim, page, block, dtype, causal, table_room):
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, block, dtype, seed=hq + dim + sum(new), spare_rows=3))
    compare(c, *run(c, causal=causal), causal=causal)


@pytest.mark.parametrize("max_q", [1, 3, 16, 1000])
def test_the_hint_changes_no_value(max_q, table_room):
    """max_q picks the kernel; a wrong one is still answered right."""
    c = table_room(pc.batch([150, 300, 40], [40, 1, 17], 8, 4, 128, 32, 32, BF, seed=3))
    compare(c, *run(c, max_q=max_q))
    c = table_room(pc.batch([150, 300, 40], None, 8, 4, 64, 32, 16, F16, seed=4))
    compare(c, *run(c, max_q=max_q))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("new", [None, [40, 90]])
def test_large_scores(dtype, new, table_room):
    """Scores of some thousands: one position takes all, nothing overflows."""
    c = table_room(pc.batch([700, 260], new, 4, 2, 128, 64, 32, dtype, seed=8, qscale=60.0))
    compare(c, *run(c, scale=3.0), scale=3.0)


@pytest.mark.parametrize("new", [None, [40, 90]])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_and_scales_that_move_at_each_block(new, rising, table_room):
    """Every position's score is above (below) all before it, and every block's values are of another size."""
    c = table_room(pc.batch([900, 333], new, 2, 1, 64, 32, 16, BF, seed=9))
    c["q"][:] = 1.0
    k = torch.zeros(c["k"].shape)
    level = torch.zeros(c["vs"].shape)
    for b in range(2):
        for p in range(int(c["lens"][b])):
            k[c["table"][b, p // 32], :, p % 32] = p / 64 if rising else -p / 64
            level[c["table"][b, p // 32], :, p % 32 // 16] = (p // 16) * (1 if rising else -1) / 2
    v = c["q"].new_zeros(c["v"].shape, dtype=torch.float32).normal_(generator=torch.Generator().manual_seed(1))
    c["k"], c["ks"] = pc.quantise(k, c["used"], 16)
    c["v"], c["vs"] = pc.quantise(v, c["used"], 16, level.floor())
    compare(c, *run(c))


@pytest.mark.parametrize("new", [None, [40, 90]])
def test_scales_far_apart(new, table_room):
    """Blocks of 2^-60 and 2^60, queries from 2^-100 to 2^100 in one row: nothing is lost that counts."""
    c = table_room(pc.batch([200, 100], new, 4, 2, 64, 32, 16, BF, seed=19, levels=0))
    g = torch.Generator().manual_seed(4)
    vs = pc.bits(c["vs"])
    at = torch.rand(vs.shape, generator=g) < 0.5
    vs[at & (vs != 255)] = 67
    vs[~at & (vs != 255)] = 187
    q = c["q"].view(c["rows"], 4, 64)
    q[:, 0] *= 2.0 ** -100
    q[:, 1, 1:] *= 2.0 ** -60
    compare(c, *run(c))


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,block,dtype", [
    ([90, 700, 33], [3, 2, 3], 10, 2, 128, 32, 16, BF),      # a few drafted tokens
    ([2600, 41], [16, 16], 3, 3, 64, 16, 16, F16),
    ([400, 131], [150, 131], 4, 2, 128, 64, 64, BF),         # prompts
    ([700, 300], [260, 41], 5, 1, 64, 16, 16, F16),
    ([3900], [600], 2, 1, 128, 128, 32, F16),                # shared by many CTAs
])
def test_what_a_row_does_not_see_may_be_nan(lens, new, hq, hkv, dim, page, block, dtype, table_room):
    """Keys and values of later tokens reach no earlier row, whatever they hold; the rows that see them show it."""
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, block, dtype, seed=41))
    clean = dict(c, k=c["k"].clone(), v=c["v"].clone())
    table, starts = c["table"].tolist(), c["starts"].tolist()
    for b, (n, m) in enumerate(zip(lens, new)):
        for i, back in enumerate(sorted({1, 2, m // 2, m - 1} & set(range(1, m)))):  # `back` - 1 rows later than the last
            pos = n - back
            spot = (table[b][pos // page], i % hkv, pos % page)
            pc.bits(c["v"])[spot][(7 * i) % dim] = 0x7F
            pc.bits(c["v"])[spot][dim - 1 - i] = 0xFF
            pc.bits(clean["v"])[spot][(7 * i) % dim] = pc.bits(clean["v"])[spot][dim - 1 - i] = 0
        last = (table[b][(n - 1) // page], 0, (n - 1) % page)
        pc.bits(c["k"])[last][3] = 0x7F
        pc.bits(clean["k"])[last][3] = 0
    ref, fine = oracle(c), oracle(clean)
    tol, ltol = o8.attention_bounds(fine, dim, dtype)
    out, lse = run(c)
    o = out.double().reshape(c["rows"], hq, dim)
    sees_k = torch.zeros(c["rows"], hq, dtype=torch.bool)  # a NaN key: the sequences' last rows, kv head 0
    sees_k[[s - 1 for s in starts[1:]], :hq // hkv] = True
    odd = torch.isnan(ref["out"]) & ~sees_k[..., None]
    assert odd.any() and torch.isnan(o)[odd].all()
    assert torch.isnan(o[sees_k]).all() and torch.isnan(lse[sees_k]).all()
    good = torch.isfinite(ref["out"]) & ~sees_k[..., None]
    assert ((o - ref["out"]).abs() <= tol)[good].all()
    assert ((lse.double() - ref["lse"]).abs() <= ltol)[~sees_k].all()


@pytest.mark.parametrize("new", [None, [40, 30]])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_an_unusual_query_stays_in_its_row(new, what, table_room):
    c = table_room(pc.batch([300, 90], new, 4, 2, 128, 32, 32, BF, seed=43))
    c["q"][1, 130] = what  # head 1 of row 1: an infinite product of either sign, or 0 times infinity
    out, lse = run(c)
    ref = oracle(c)
    odd = torch.zeros_like(lse, dtype=torch.bool)
    odd[1, 1] = True
    o = out.reshape(c["rows"], 4, 128)
    assert torch.isnan(o[1, 1]).all()
    assert torch.isfinite(o[~odd]).all() and torch.isfinite(lse[~odd]).all()
    tol, _ = o8.attention_bounds(ref, 128, BF)
    assert ((o.double() - ref["out"]).abs() <= tol)[~odd].all()


@pytest.mark.parametrize("new", [None, [40, 30]])
def test_a_row_whose_scores_are_all_minus_infinity(new, table_room):
    """0 / 0 as softmax has it, and an lse of -inf; fp32 scores below its range are such scores."""
    c = table_room(pc.batch([70, 40], new, 2, 1, 64, 16, 16, BF, seed=44))
    c["q"][0, :64] = -3e38
    pc.bits(c["k"])[:] = torch.where(c["used"][:, None, :, None], torch.tensor(126, dtype=torch.uint8), pc.bits(c["k"]))
    out, lse = run(c, scale=100.0)
    assert torch.isnan(out[0, :64]).all() and float(lse[0, 0]) == -math.inf
    assert torch.isfinite(out[0, 64:]).all() and torch.isfinite(out[1:]).all() and torch.isfinite(lse[1:]).all()


@pytest.mark.parametrize("new", [None, [21, 64]])
def test_strides(new):
    """Pages stored (pages, slot, head, D) with interleaved k / v, scales in one tensor, wide q / out / lse rows."""
    c = pc.batch([200, 131], new, 8, 4, 128, 64, 16, BF, seed=2, layout="nhd")
    compare(c, *run(c))
    rows, pages = c["rows"], c["k"].shape[0]
    both = torch.full((pages, 2, 4, 64, 128), 0x7F, dtype=torch.uint8)
    both[:, 0], both[:, 1] = pc.bits(c["k"]), pc.bits(c["v"])
    scales = torch.full((pages, 4, 2, 6), 255, dtype=torch.uint8)
    scales[:, :, 0, 1:5], scales[:, :, 1, 1:5] = pc.bits(c["ks"]), pc.bits(c["vs"])
    d, s = both.to(DEV).view(F8), scales.to(DEV).view(E8)
    wide = torch.zeros(rows, 3 * 1024, dtype=BF, device=DEV)
    wide[:, 1024:2048] = c["q"].to(DEV)
    out = torch.full((rows, 1024 + 64), 3.0, dtype=BF, device=DEV)
    lse = torch.full((rows, 40), 7.0, device=DEV)
    table = torch.full((2, c["table"].shape[1] + 5), -9, dtype=torch.int32, device=DEV)
    table[:, 2:-3] = c["table"].to(DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    _api().paged_attention_fp8(wide[:, 1024:2048], d[:, 0], d[:, 1], s[:, :, 0, 1:5], s[:, :, 1, 1:5], table[:, 2:-3],
                               c["lens"].to(DEV), q_starts=starts, out=out[:, 64:], lse=lse[:, 16:24])
    torch.cuda.synchronize()
    assert (out[:, :64] == 3.0).all() and (lse[:, :16] == 7.0).all() and (lse[:, 24:] == 7.0).all()
    compare(c, out[:, 64:].cpu(), lse[:, 16:24].cpu())


@pytest.mark.parametrize("new", [None, [3, 70]])
def test_offsets_behind_four_gigabytes(new, table_room):
    """Pages more than 2^32 codes from the base."""
    c = table_room(pc.batch([200, 131], new, 4, 2, 128, 64, 32, BF, seed=2))
    pages, step = c["k"].shape[0], (1 << 32) // (c["k"].shape[0] - 1) // 16 * 16 + 64
    k, v = (torch.empty(pages * step, dtype=torch.uint8, device=DEV).as_strided((pages, 2, 64, 128), (step, 8192, 128, 1))
            for _ in range(2))
    k.copy_(pc.bits(c["k"]))
    v.copy_(pc.bits(c["v"]))
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    lse = torch.empty(c["rows"], 4, device=DEV)
    rest = (pc.bits(c["ks"]).to(DEV).view(E8), pc.bits(c["vs"]).to(DEV).view(E8), c["table"].to(DEV), c["lens"].to(DEV))
    out = _api().paged_attention_fp8(c["q"].to(DEV), k.view(F8), v.view(F8), *rest, q_starts=starts, lse=lse)
    kk, vv = _api().paged_read_fp8(k.view(F8), v.view(F8), *rest, q_starts=starts, rows=c["rows"])
    torch.cuda.synchronize()
    compare(c, out.cpu(), lse.cpu())
    check_read(c, kk, vv, BF)


@pytest.mark.parametrize("new", [None, [9, 150, 1]])
def test_reruns_are_bit_identical(new, table_room):
    c = table_room(pc.batch([900, 2000, 400], new, 16, 4, 128, 64, 64, BF, seed=6))
    first = run(c)
    for _ in range(3):
        again = run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---------------------------------------------------------------- reading back
def check_read(c, k, v, dtype):
    table, lens = c["table"].tolist(), c["lens"].tolist()
    starts = None if c["starts"] is None else c["starts"].tolist()
    for got, codes, scales in ((k, c["k"], c["ks"]), (v, c["v"], c["vs"])):
        want = o8.values(codes, scales)
        if dtype == F16:
            want = want.clamp(-65504, 65504)
        for b, a, z, n in op.sequences(c["rows"], lens, starts):
            for t in range(a, z):
                pos = n - z + t
                if pos >= 0:
                    x = want[table[b][pos // c["page"]], :, pos % c["page"]].to(dtype)
                    assert torch.equal(got[t].cpu().nan_to_num(5.0), x.nan_to_num(5.0)), (b, t)


READ = [
    ([1], None, 1, 128, 16, 16, BF, "hnd"),
    ([33, 0, 128, 7], None, 3, 64, 32, 16, F16, "nhd"),
    ([200, 131, 77], [200, 131, 77], 4, 128, 64, 32, BF, "hnd"),
    ([300, 0, 50], [41, 0, 50], 5, 64, 16, 16, torch.float32, "hnd"),
    ([2, 70], [5, 70], 2, 128, 1024, 128, F16, "nhd"),              # rows before the first position
    ([90] * 40, [1] * 40, 1, 64, 32, 32, BF, "hnd"),
    ([1000, 3], [999, 1], 6, 128, 128, 64, torch.float32, "nhd"),
]


@pytest.mark.parametrize("lens,new,hkv,dim,page,block,dtype,layout", READ)
def test_reading_back(lens, new, hkv, dim, page, block, dtype, layout):
    c = pc.batch(lens, new, hkv, hkv, dim, page, block, BF, seed=sum(lens), layout=layout, spare_rows=2 if new else 0, levels=30)
    d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    k, v = (torch.full((c["rows"], hkv, dim), 3.0, dtype=dtype, device=DEV) for _ in range(2))
    got = _api().paged_read_fp8(*where(d), q_starts=starts, dtype=dtype, k_out=k, v_out=v)
    assert got[0] is k and got[1] is v
    check_read(c, k, v, dtype)
    live = torch.zeros(c["rows"], dtype=torch.bool)
    for _, a, z, n in op.sequences(c["rows"], lens, None if new is None else c["starts"].tolist()):
        live[a + max(0, (z - a) - n):z] = True
    assert (k[~live] == 3.0).all() and (v[~live] == 3.0).all()
    wide = torch.full((2, c["rows"], hkv + 1, 2 * dim), 3.0, dtype=dtype, device=DEV)  # wide rows and heads
    _api().paged_read_fp8(*where(d), q_starts=starts, rows=c["rows"], dtype=dtype, k_out=wide[0, :, 1:, dim:], v_out=wide[1, :, :-1, :dim])
    assert torch.equal(wide[0, :, 1:, dim:].nan_to_num(), k.nan_to_num()) and torch.equal(wide[1, :, :-1, :dim].nan_to_num(), v.nan_to_num())
    assert (wide[0, :, 0] == 3.0).all() and (wide[0, :, :, :dim] == 3.0).all() and (wide[1, :, -1] == 3.0).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F16, torch.float32])
@pytest.mark.parametrize("ragged", [False, True])
def test_reading_back_with_more_blocks_than_run_at_once(ragged, dtype, dim):
    """700 sequences of one to three rows: some 1400 thread blocks."""
    lens = [1 + (7 * i) % 40 for i in range(700)]
    new = [min(n, 1 + i % 3) for i, n in enumerate(lens)] if ragged else None
    c = pc.batch(lens, new, 3, 3, dim, 16, 16, BF, seed=33, levels=30)
    d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
    k, v = _api().paged_read_fp8(*where(d), q_starts=c["starts"].to(DEV) if ragged else None, rows=c["rows"], dtype=dtype)
    torch.cuda.synchronize()
    check_read(c, k, v, dtype)


def test_every_code_and_scale_is_read_as_what_it_is():
    codes = torch.arange(256, dtype=torch.uint8).repeat(64).reshape(1, 1, 128, 128)  # 8 blocks of 16 positions
    scales = torch.tensor([[[67, 187, 127, 110, 135, 0, 254, 255]]], dtype=torch.uint8)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([128], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    d, s = codes.to(DEV).view(F8), scales.to(DEV).view(E8)
    want = o8.values(codes.view(F8), scales.view(E8))[0, 0]
    for dtype in (BF, F16, torch.float32):
        k, v = _api().paged_read_fp8(d, d, s, s, table, lens, q_starts=starts, rows=128, dtype=dtype)
        x = (want.clamp(-65504, 65504) if dtype == F16 else want).to(dtype)
        assert torch.equal(k[:, 0].cpu().nan_to_num(9.0), x.nan_to_num(9.0)) and torch.equal(v.nan_to_num(), k.nan_to_num())


# ---------------------------------------------------------------- append
def check_append(c, before, after, q, qkv, cos, sin, norms, eps):
    """The caches after an append against those before it: values within one step of the code they were rounded to
    (plus fp32 roundings in front for k), scales and older codes exactly, everything else untouched."""
    hkv, dim, page, block, hq = c["hkv"], c["dim"], c["page"], c["block"], c["hq"]
    table, lens, starts = c["table"].tolist(), c["lens"].tolist(), None if c["starts"] is None else c["starts"].tolist()
    rows = qkv.shape[0]
    fake = torch.zeros(c["k"].shape[0], hkv, page, dim)
    want, written, terms = op.append(qkv, cos, sin, fake, fake, table, lens, starts, *norms, eps)
    u = torch.finfo(qkv.dtype).eps / 2
    slack = (dim / 2 + 8) * 2.0 ** -24
    got = q.double().reshape(rows, hq, dim)
    live = ~torch.isnan(want[:, 0, 0])
    odd = ~torch.isfinite(qkv.double()).reshape(rows, -1, dim).all(-1)  # heads with infinite or NaN entries
    fine = live[:, None] & ~odd[:, :hq]
    tiny = 2.0 ** -25 if qkv.dtype == F16 else 0.0
    assert ((got - want).abs() <= u * want.abs() + slack * terms[:, :hq] + tiny)[fine].all()
    assert (got[~live] == 3.0).all()
    touched = torch.zeros(c["k"].shape[0], hkv, page, dtype=torch.bool)
    scaled = torch.zeros(c["ks"].shape, dtype=torch.bool)
    for which in (0, 1):
        b_codes, b_scales = before[which], before[2 + which]
        a_codes, a_scales = after[which], after[2 + which]
        for b, r0, n, p, kept in o8.block_parts(rows, lens, starts, block):
            pg, s0, blk = table[b][p // page], p % page, p % page // block
            x = torch.stack([written[(pg, s0 + i)][1 + which] for i in range(n)], 1)  # (HKV, n, D), 64 bits
            err = torch.stack([terms[r0 + i, hq:] * slack for i in range(n)], 1) if which == 0 else torch.zeros_like(x)
            touched[pg, :, s0 - kept:s0 + n] = True
            scaled[pg, :, blk] = True
            for j in range(hkv):
                e = int(o8.scales_of(a_scales)[pg, j, blk])
                f = torch.isfinite(x[j])
                mag = x[j].abs().masked_fill(~f, 0.0)
                lo, hi = (o8.exponent(max(0.0, float((mag + s * err[j].masked_fill(~f, 0.0)).max()))) for s in (-1, 1))
                was = int(o8.scales_of(b_scales)[pg, j, blk])
                if kept:
                    lo, hi = max(lo, was), max(hi, was)
                    old = b_codes[pg, j, s0 - kept:s0].double()
                    now = a_codes[pg, j, s0 - kept:s0].double()
                    assert torch.equal(now.nan_to_num(999.0), (o8.nearest(old * 2.0 ** (was - e))).nan_to_num(999.0))
                assert lo <= e <= hi, (which, b, p, j, lo, e, hi)
                new = a_codes[pg, j, s0:s0 + n].double()
                y = (x[j] * 2.0 ** -e).clamp(-448, 448)
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6).masked_fill(~f, 1.0))) - 3)
                # half a step (a whole one up in the next binade counts for the value just below it)
                assert ((new - y).abs() <= step / 2 + err[j] * 2.0 ** -e)[f].all()
                if which == 1:
                    assert torch.equal(new[f], o8.nearest(y)[f])
                    assert torch.isnan(new[~f]).all()
        assert torch.equal(pc.bits(a_codes)[~touched], pc.bits(b_codes)[~touched])
        assert torch.equal(pc.bits(a_scales)[~scaled], pc.bits(b_scales)[~scaled])


def tables(positions, dim, dtype, g):
    ang = torch.rand(positions, dim // 2, generator=g) * 6.3
    return torch.cat([ang, ang], 1).cos().to(dtype), torch.cat([ang, ang], 1).sin().to(dtype)


def append(c, d, qkv, cos, sin, norms, eps, out=None):
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    x = qkv.to(DEV)
    if out is None:
        out = torch.full((qkv.shape[0], c["hq"] * c["dim"]), 3.0, dtype=qkv.dtype, device=DEV)
    n = [None if t is None else t.to(DEV) for t in norms]
    _api().paged_append_fp8(x, cos.to(DEV), sin.to(DEV), *where(d), q_starts=starts, q_norm_w=n[0], k_norm_w=n[1], eps=eps, out=out)
    torch.cuda.synchronize()
    return out.cpu()


def caches(d):
    return [d[k].cpu() for k in ("k", "v", "ks", "vs")]


APPEND = [
    # lens, new, hq, hkv, dim, page, block, dtype, cos dtype, norms
    ([1], None, 1, 1, 128, 16, 16, BF, BF, True),
    ([1, 2, 15, 16, 17, 33, 64], None, 4, 2, 64, 16, 16, BF, torch.float32, True),
    ([64, 65, 128, 0, 100], None, 16, 16, 128, 64, 64, F16, F16, False),
    ([300, 77], None, 8, 1, 128, 128, 128, BF, BF, True),
    ([5], [5], 4, 2, 128, 16, 16, BF, BF, True),
    ([40, 70, 33], [3, 1, 5], 8, 4, 128, 16, 16, F16, torch.float32, True),
    ([130, 64, 200], [7, 64, 1], 6, 3, 64, 64, 32, F16, F16, True),
    ([300, 129], [300, 100], 5, 5, 64, 64, 64, BF, BF, False),
    ([129, 0, 257, 9], [129, 0, 120, 0], 6, 2, 128, 128, 128, BF, torch.float32, True),
    ([513, 20], [257, 20], 5, 1, 128, 512, 128, BF, BF, True),
    ([2, 3, 40], [4, 3, 50], 2, 1, 64, 32, 16, BF, BF, True),      # more rows than positions: the first are skipped
    ([50] * 30, [2] * 30, 2, 2, 64, 16, 16, F16, F16, False),
]


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,block,dtype,cdt,normed", APPEND)
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_append(lens, new, hq, hkv, dim, page, block, dtype, cdt, normed, layout):
    c = pc.batch(lens, new, hq, hkv, dim, page, block, dtype, seed=dim + sum(lens), layout=layout, spare_rows=2 if new else 0)
    g = torch.Generator().manual_seed(5 + hq)
    qkv = torch.randn(c["rows"], (hq + 2 * hkv) * dim, generator=g) * torch.exp2(torch.randint(-9, 9, (c["rows"], hq + 2 * hkv, 1), generator=g).float()).expand(-1, -1, dim).reshape(c["rows"], -1)
    qkv = qkv.to(dtype)
    cos, sin = tables(max(max(lens), 1), dim, cdt, g)
    norms = [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) if normed else None for _ in range(2)]
    d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
    before = caches(d)
    q = append(c, d, qkv, cos, sin, norms, 1e-5)
    after = caches(d)
    check_append(c, before, after, q, qkv, cos, sin, norms, 1e-5)
    again = append(c, d, qkv, cos, sin, norms, 1e-5)  # the same call changes nothing
    assert torch.equal(q, again) and all(torch.equal(pc.bits(x), pc.bits(y)) for x, y in zip(after, caches(d)))


def test_append_of_unusual_values():
    """Infinite, NaN, zero, huge and tiny entries; what is infinite does not set a scale."""
    c = pc.batch([20, 40], [9, 33], 2, 2, 64, 16, 16, BF, seed=1)
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(42, 6 * 64, generator=g)
    qkv[3, 4 * 64 + 5], qkv[4, 4 * 64 + 6], qkv[5, 5 * 64 + 7] = math.inf, -math.inf, math.nan
    qkv[9:20, 4 * 64:] = 0.0
    qkv[20:30, 4 * 64:5 * 64] *= 2.0 ** 100
    qkv[20:30, 5 * 64:] *= 2.0 ** -100
    qkv[7, 2 * 64 + 3] = math.inf  # a k head: rotated into its pair, too
    qkv = qkv.to(BF)
    cos, sin = tables(40, 64, BF, g)
    d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
    before = caches(d)
    q = append(c, d, qkv, cos, sin, [None, None], 1e-5)
    check_append(c, before, caches(d), q, qkv, cos, sin, [None, None], 1e-5)


def test_append_into_its_own_rows_and_wide_ones():
    c = pc.batch([90, 31], [33, 2], 4, 2, 64, 32, 32, F16, seed=7)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(35, 8 * 64, generator=g).to(F16)
    cos, sin = tables(90, 64, F16, g)
    d, d2 = (pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV) for _ in range(2))
    q = append(c, d, qkv, cos, sin, [None, None], 1e-5)
    buf = torch.zeros(35, 10 * 64, dtype=F16, device=DEV)
    buf[:, 64:9 * 64] = qkv.to(DEV)
    x = buf[:, 64:9 * 64]
    out = _api().paged_append_fp8(x, cos.to(DEV), sin.to(DEV), *where(d2), q_starts=c["starts"].to(DEV), out=x[:, :4 * 64])
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), q) and all(torch.equal(pc.bits(a), pc.bits(b)) for a, b in zip(caches(d), caches(d2)))
    assert (buf[:, :64] == 0).all() and (buf[:, 9 * 64:] == 0).all() and torch.equal(x[:, 4 * 64:].cpu(), qkv[:, 4 * 64:])


@pytest.mark.parametrize("block", [16, 64])
def test_a_block_filled_token_by_token(block):
    """100 single-token calls, each token larger or smaller than those before: every value stays within what its
    code and the rescalings may lose, and the scale is the one that the largest so far needs."""
    hkv, dim, page = 2, 64, 64
    g = torch.Generator().manual_seed(block)
    x = torch.randn(100, 3 * hkv, dim, generator=g)
    x[:, 2 * hkv:] *= torch.exp2(torch.randint(-6, 7, (100, hkv, 1), generator=g).float())
    x = x.to(BF)
    k, v = (torch.full((2, hkv, page, dim), 0x7F, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
    ks, vs = (torch.full((2, hkv, page // block), 255, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2))
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    one, zero = torch.ones(128, dim, device=DEV), torch.zeros(128, dim, device=DEV)
    for t in range(100):
        lens += 1
        _api().paged_append_fp8(x[t].reshape(1, -1).to(DEV), one, zero, k, v, ks, vs, table, lens)
    starts = torch.tensor([0, 100], dtype=torch.int32, device=DEV)
    kk, vv = _api().paged_read_fp8(k, v, ks, vs, table, lens, q_starts=starts, rows=100, dtype=torch.float32)
    torch.cuda.synchronize()
    for got, want, scales in ((kk, x[:, hkv:2 * hkv], ks), (vv, x[:, 2 * hkv:], vs)):
        got, want = got.cpu().double(), want.double()
        for p in range(0, 100, block):
            top = want[p:p + block].abs().amax((0, 2))
            e = torch.tensor([o8.exponent(float(t)) for t in top])
            assert torch.equal(o8.scales_of(scales.cpu())[[1, 0][p // page], :, p % page // block].long(), e)
            # half a step of four significant bits once; then, where the code became subnormal, half of 2^(e - 9) at
            # each rescaling, which at least doubles it: 2^(e - 9) in all
            tol = want[p:p + block].abs() * 2.0 ** -4 + torch.exp2(e.double() - 9)[:, None]
            assert ((got[p:p + block] - want[p:p + block]).abs() <= tol).all()


@pytest.mark.parametrize("roomy", [False, True])
def test_append_attend_and_read_together(roomy):
    """A prompt, drafted tokens of which some are taken back, then single tokens; attention after each append."""
    hq, hkv, dim, page, block, B = 8, 2, 128, 32, 16, 3
    P = _api()
    g = torch.Generator().manual_seed(11)
    cols = 8 + (65536 // page if roomy else 0)
    table = torch.full((B, cols), -5, dtype=torch.int32)
    table[:, :8] = torch.randperm(B * 8, generator=g).reshape(B, 8)
    k, v = (torch.full((B * 8, hkv, page, dim), 0x7F, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
    ks, vs = (torch.full((B * 8, hkv, page // block), 255, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2))
    cos, sin = tables(256, dim, torch.float32, g)
    norms = [(1 + 0.3 * torch.randn(dim, generator=g)).to(BF) for _ in range(2)]
    lens = torch.zeros(B, dtype=torch.int32)
    steps = [[100, 37, 1], [5, 0, 5], "cut", [3, 4, 2], None, None, [0, 60, 9], None]
    for step in steps:
        if step == "cut":
            lens -= torch.tensor([3, 0, 4], dtype=torch.int32)
            continue
        new = [1] * B if step is None else step
        lens = lens + torch.tensor(new, dtype=torch.int32)
        starts = None if step is None else torch.tensor([0] + new).cumsum(0).to(torch.int32)
        rows = sum(new)
        qkv = (torch.randn(rows, (hq + 2 * hkv) * dim, generator=g) * 2).to(BF)
        c = dict(k=k.cpu(), v=v.cpu(), ks=ks.cpu(), vs=vs.cpu(), table=table, lens=lens, starts=starts, rows=rows, hq=hq, hkv=hkv,
                 dim=dim, page=page, block=block, dtype=BF)
        d = dict(k=k, v=v, ks=ks, vs=vs, table=table.to(DEV), lens=lens.to(DEV))
        before = caches(d)
        q = append(c, d, qkv, cos, sin, norms, 1e-6)
        after = caches(d)
        check_append(c, before, after, q, qkv, cos, sin, norms, 1e-6)
        c.update(k=after[0], v=after[1], ks=after[2], vs=after[3], q=q)
        ds = None if starts is None else starts.to(DEV)
        lse = torch.empty(rows, hq, device=DEV)
        out = P.paged_attention_fp8(q.to(DEV), *where(d), q_starts=ds, max_q=max(new), lse=lse)
        compare(c, out.cpu(), lse.cpu())
        kk, vv = P.paged_read_fp8(*where(d), q_starts=ds, rows=rows)
        check_read(c, kk, vv, BF)


def test_calls_without_rows():
    P = _api()
    c = pc.batch([5, 9], [0, 0], 4, 2, 64, 16, 16, BF, seed=1)
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    starts, one = c["starts"].to(DEV), torch.ones(16, 64, device=DEV)
    before = caches(d)
    assert P.paged_append_fp8(torch.zeros(0, 8 * 64, dtype=BF, device=DEV), one, one, *where(d), q_starts=starts).shape == (0, 256)
    assert P.paged_attention_fp8(torch.zeros(0, 256, dtype=BF, device=DEV), *where(d), q_starts=starts).shape == (0, 256)
    k, v = P.paged_read_fp8(*where(d), q_starts=starts, rows=0)
    assert k.shape == v.shape == (0, 2, 64)
    torch.cuda.synchronize()
    assert all(torch.equal(pc.bits(x), pc.bits(y)) for x, y in zip(before, caches(d)))


def test_lengths_below_zero_are_unused_slots():
    P = _api()
    c = pc.batch([40, 33, 20], [3, 4, 2], 2, 1, 64, 16, 16, BF, seed=3)
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    d["lens"][1] = -2 ** 31
    starts, one = c["starts"].to(DEV), torch.ones(64, 64, device=DEV)
    before = caches(d)
    out = torch.full((9, 128), 3.0, dtype=BF, device=DEV)
    P.paged_append_fp8(torch.ones(9, 4 * 64, dtype=BF, device=DEV), one, one, *where(d), q_starts=starts, out=out)
    assert (out[3:7] == 3.0).all() and (out[:3] != 3.0).any() and (out[7:] != 3.0).any()
    mine = c["table"][1, :3].long()
    assert all(torch.equal(pc.bits(x)[mine], pc.bits(y)[mine]) for x, y in zip(before, caches(d)))
    lse = torch.zeros(9, 2, device=DEV)
    for max_q in (4, 1000):
        o = P.paged_attention_fp8(d["q"], *where(d), q_starts=starts, max_q=max_q, lse=lse)
        assert (o[3:7] == 0).all() and (lse[3:7] == -math.inf).all() and torch.isfinite(lse[:3]).all()
    k, v = (torch.full((9, 1, 64), 3.0, dtype=BF, device=DEV) for _ in range(2))
    P.paged_read_fp8(*where(d), q_starts=starts, k_out=k, v_out=v)
    assert (k[3:7] == 3.0).all() and (v[3:7] == 3.0).all() and (v[:3] != 3.0).any()


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_one_page_or_one_kv_head(layout):
    """Dimensions of size one, whose strides mean nothing."""
    for lens, hkv, page in (([40], 1, 64), ([40], 3, 64), ([90, 20, 130], 1, 32)):
        for new in (None, [7 + b for b in range(len(lens))], [20] * len(lens)):
            c = pc.batch(lens, new, 8 * hkv, hkv, 64, page, 16, BF, seed=8, layout=layout)
            if page == 64:
                p = int(c["table"][0, 0])
                for n in ("k", "v", "ks", "vs"):
                    c[n] = c[n][p:p + 1]
                c["table"][0, 0] = 0
            compare(c, *run(c))
            compare(c, *run(c, max_q=1000))


# ---------------------------------------------------------------- errors, streams, graphs
def test_lengths_behind_the_table_and_bad_pages_are_reported():
    from breeze_b200 import _lib

    P = _api()
    c = pc.batch([30, 40, 20], [3, 4, 2], 2, 1, 64, 16, 16, BF, seed=3, spare_cols=0)
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    starts = c["starts"].to(DEV)
    qkv, one = torch.ones(9, 4 * 64, dtype=BF, device=DEV), torch.ones(64, 64, device=DEV)
    before = caches(d)
    for change, bit in ((lambda t: t["table"][1].fill_(10 ** 6), _lib.BQ_DEVERR_PAGE), (lambda t: t["table"][1].fill_(-1), _lib.BQ_DEVERR_PAGE),
                        (lambda t: t["lens"][1].fill_(60), _lib.BQ_DEVERR_POSITION)):
        bad = {k: v.clone() if k in ("table", "lens") else v for k, v in d.items()}
        change(bad)
        for call in (lambda: P.paged_attention_fp8(bad["q"], *where(bad), q_starts=starts, max_q=4),
                     lambda: P.paged_read_fp8(*where(bad), q_starts=starts, rows=9)):
            call()
            torch.cuda.synchronize()
            assert _status() == bit
        for ragged in (True, False):
            out = torch.full((9 if ragged else 3, 2 * 64), 3.0, dtype=BF, device=DEV)
            P.paged_append_fp8(qkv if ragged else qkv[:3], one, one, *where(bad), q_starts=starts if ragged else None, out=out)
            torch.cuda.synchronize()
            assert _status() == bit
            skipped = slice(3, 7) if ragged else slice(1, 2)
            assert (out[skipped] == 3.0).all() and (out[:1] != 3.0).all() and (out[-1:] != 3.0).all()
        now = caches(d)
        mine = c["table"][1].long()
        assert all(torch.equal(pc.bits(x)[mine], pc.bits(y)[mine]) for x, y in zip(before, now))
    short = torch.ones(39, 64, device=DEV)  # no cos / sin row for the last token of the longest
    P.paged_append_fp8(qkv, short, short, *where(d), q_starts=starts)
    torch.cuda.synchronize()
    assert _status() == _lib.BQ_DEVERR_POSITION


@pytest.mark.parametrize("new", [None, [4, 80]])
def test_captured_graphs(new, table_room):
    """Two graphs captured once, replayed at the same time on two streams with
    lengths, tables and rows changed in place after the capture."""
    P = _api()
    dim, hq, hkv = 128, 8, 4
    cases = [table_room(pc.batch([300, 500], new, hq, hkv, dim, 64, 32, BF, seed=s)) for s in (1, 2)]
    one, zero = torch.ones(512, dim, device=DEV), torch.zeros(512, dim, device=DEV)
    devs, graphs, outs, streams = [], [], [], []
    for c in cases:
        d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
        d["starts"] = None if c["starts"] is None else c["starts"].to(DEV)
        d["qkv"] = torch.zeros(c["rows"], (hq + 2 * hkv) * dim, dtype=BF, device=DEV)
        q, out = (torch.zeros(c["rows"], hq * dim, dtype=BF, device=DEV) for _ in range(2))
        lse = torch.zeros(c["rows"], hq, device=DEV)
        kv = [torch.zeros(c["rows"], hkv, dim, dtype=BF, device=DEV) for _ in range(2)]

        def call():
            P.paged_append_fp8(d["qkv"], one, zero, *where(d), q_starts=d["starts"], out=q)
            P.paged_attention_fp8(q, *where(d), q_starts=d["starts"], out=out, lse=lse)
            P.paged_read_fp8(*where(d), q_starts=d["starts"], k_out=kv[0], v_out=kv[1])

        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):  # the first call is the captured one
            call()
        devs.append(d)
        graphs.append(graph)
        outs.append((q, out, lse, kv))
        streams.append(st)
    changed = [pc.batch([190, 410], new, hq, hkv, dim, 64, 32, BF, seed=s + 10) for s in (1, 2)]
    g = torch.Generator().manual_seed(0)
    for c, d in zip(changed, devs):
        pages, cols = c["k"].shape[0], c["table"].shape[1]
        for name in ("k", "v", "ks", "vs"):
            pc.bits(d[name])[:pages] = pc.bits(c[name]).to(DEV)
        d["table"][:, :cols] = c["table"].to(DEV)
        d["lens"].copy_(c["lens"])
        d["qkv"].copy_(torch.randn(d["qkv"].shape, generator=g))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for c, d, (q, out, lse, kv) in zip(changed, devs, outs):
        pages = c["k"].shape[0]
        c["k"], c["v"], c["ks"], c["vs"] = (pc.bits(d[n]).cpu().view(d[n].dtype)[:pages] for n in ("k", "v", "ks", "vs"))
        c["q"] = q.cpu()
        assert torch.equal(q.cpu(), d["qkv"][:, :hq * dim].cpu())  # cos 1, sin 0, no norm
        compare(c, out.cpu(), lse.cpu())
        check_read(c, *kv, BF)


@pytest.mark.parametrize("new", [None, [30, 200]])
def test_two_streams_at_once(new):
    P = _api()
    cases = [pc.batch([1500, 3000], new, 8, 2, 128, 64, 64, BF, seed=s) for s in (21, 22)]
    alone = [run(c) for c in cases]
    devs = [pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV) for c in cases]
    starts = None if new is None else cases[0]["starts"].to(DEV)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (d, st) in enumerate(zip(devs, streams)):
            with torch.cuda.stream(st):
                lse = torch.empty(cases[i]["rows"], 8, device=DEV)
                got[i].append((P.paged_attention_fp8(d["q"], *where(d), q_starts=starts, lse=lse), lse))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out.cpu(), alone[i][0]) and torch.equal(lse.cpu(), alone[i][1])


def test_more_sequences_than_threads():
    """700 sequences: every pass over the batch takes several rounds."""
    lens = [1 + (7 * i) % 40 for i in range(700)]
    c = pc.batch(lens, None, 2, 1, 64, 16, 16, BF, seed=30)
    compare(c, *run(c))
    new = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    c = pc.batch(lens, new, 2, 1, 64, 16, 16, F16, seed=31)
    compare(c, *run(c))
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(c["rows"], 4 * 64, generator=g).to(F16)
    cos, sin = tables(40, 64, F16, g)
    d = pc.to({k: c[k] for k in ("k", "v", "ks", "vs", "table", "lens")}, DEV)
    before = caches(d)
    q = append(c, d, qkv, cos, sin, [None, None], 1e-5)
    check_append(c, before, caches(d), q, qkv, cos, sin, [None, None], 1e-5)
