"""Paged-cache operators against the 64-bit oracle (oracle/paged.py), element
by element within bounds derived from the arithmetic (attention_bounds there;
append: one rounding of the element type plus a few fp32 roundings)."""

import math

import pytest
import torch

from oracle import paged as op
from tests import paged_cases as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = pc.BF, pc.F16


def _api():
    from breeze_b200.fused import paged

    return paged


def _status(clear=True):
    from breeze_b200 import _lib

    return _lib.device_status(0, clear=clear)


@pytest.fixture(autouse=True)
def _clean_status():
    _status()
    yield
    assert _status() == 0


def run(c, causal=True, scale=None, prefix=None, out=None, lse=None, max_q=None, always=True):
    d = pc.to({k: c[k] for k in ("q", "k", "v", "table", "lens")}, DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    prefix = c["prefix"] if prefix is None else prefix
    if lse is None:
        lse = torch.full((c["rows"], c["hq"]), 7.0, device=DEV)
    if out is None:
        out = torch.full((c["rows"], c["hq"] * c["dim"]), 3.0, device=DEV, dtype=c["dtype"])
    kw = dict(q_starts=starts, scale=scale, causal=causal, max_q=max_q, out=out, lse=lse)
    if prefix:
        _api().prefix_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], prefix, always=always, **kw)
    else:
        _api().paged_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def compare(c, out, lse, causal=True, scale=None):
    table, lens, starts = pc.lists(c)
    ref = op.attention(c["q"], c["k"], c["v"], table, lens, starts, scale, causal)
    tol, ltol = op.attention_bounds(ref, c["dim"], c["dtype"])
    rows = c["rows"] if starts is None else starts[-1]
    o = out.double().reshape(c["rows"], c["hq"], c["dim"])
    err = (o[:rows] - ref["out"][:rows]).abs()
    assert torch.isfinite(o[:rows]).all()
    assert (err <= tol[:rows]).all(), (float((err / tol[:rows].clamp(min=1e-30)).max()), float(err.max()))
    empty = torch.isinf(ref["lse"][:rows])
    assert torch.equal(torch.isinf(lse[:rows]) & (lse[:rows] < 0), empty)
    lerr = (lse[:rows].double() - ref["lse"][:rows]).abs()[~empty]
    assert (lerr <= ltol[:rows][~empty]).all(), float(lerr.max())
    assert (o[rows:] == 3.0).all() and (lse[rows:] == 7.0).all()  # rows behind the last sequence


@pytest.fixture(params=["tight", "roomy"])
def table_room(request):
    """A table that ends with its longest sequence, and one with room for another
    32768 positions: the room decides how a sequence is divided among CTAs."""

    def apply(c):
        if request.param == "roomy":
            c["table"] = torch.nn.functional.pad(c["table"], (0, 32768 // c["page"]), value=-(2 ** 30))
        return c

    return apply


DECODE = [
    # lens, hq, hkv, dim, page, dtype
    ([1], 1, 1, 128, 16, BF),
    ([1, 2, 3, 15, 16, 17, 31, 32, 33], 4, 4, 64, 16, BF),
    ([63, 64, 65, 127, 128, 129], 16, 16, 128, 64, BF),
    ([256, 700], 16, 16, 128, 64, BF),
    ([300, 1, 0, 77], 8, 1, 128, 32, F16),        # an unused batch slot
    ([515], 32, 8, 128, 128, BF),
    ([2000, 5, 900], 6, 2, 64, 64, F16),
    ([4097], 24, 3, 128, 256, BF),
    ([1500, 1499, 1], 40, 2, 64, 1024, BF),       # 20 query heads per kv head
    ([333] * 70, 2, 2, 128, 16, F16),
    ([90, 17], 33, 1, 128, 16, BF),               # 33 query heads on one kv head
]


@pytest.mark.parametrize("lens,hq,hkv,dim,page,dtype", DECODE)
def test_one_token_per_sequence(lens, hq, hkv, dim, page, dtype, table_room):
    c = table_room(pc.batch(lens, None, hq, hkv, dim, page, dtype, seed=hq + dim + len(lens)))
    compare(c, *run(c))


RAGGED = [
    # lens, new, hq, hkv, dim, page, dtype
    ([5], [5], 4, 2, 128, 16, BF),
    ([40, 70, 33], [3, 1, 5], 8, 4, 128, 16, BF),
    ([130, 64, 200], [7, 64, 1], 16, 8, 128, 64, F16),
    ([300], [300], 4, 4, 64, 64, BF),
    ([129, 0, 257, 9], [129, 0, 120, 0], 6, 2, 128, 128, BF),  # sequences without new rows
    ([700, 650], [1, 260], 8, 2, 64, 32, F16),
    ([513], [257], 5, 1, 128, 512, BF),
    ([2, 3], [4, 3], 2, 1, 64, 16, BF),                         # more rows than positions: the first see nothing
    ([1100], [150], 24, 2, 128, 64, BF),                        # 12 query heads per kv head
]


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,dtype", RAGGED)
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_rows(lens, new, hq, hkv, dim, page, dtype, causal, table_room):
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=hq + dim + sum(new), spare_rows=3))
    compare(c, *run(c, causal=causal), causal=causal)


@pytest.mark.parametrize("max_q", [1, 3, 16, 1000])
def test_the_hint_changes_no_value(max_q, table_room):
    """max_q picks the kernel; a wrong one is still answered right."""
    c = table_room(pc.batch([150, 300, 40], [40, 1, 17], 8, 4, 128, 32, BF, seed=3))
    compare(c, *run(c, max_q=max_q))
    c = table_room(pc.batch([150, 300, 40], None, 8, 4, 64, 32, F16, seed=4))
    compare(c, *run(c, max_q=max_q))


PREFIX = [
    # lens, new, prefix, hq, hkv, dim, page, dtype
    ([130, 129, 200], None, 128, 4, 4, 128, 64, BF),
    ([512 + 9] * 5, None, 512, 16, 16, 128, 64, BF),
    ([1030, 1300, 1024 + 1, 1500], None, 1024, 32, 8, 128, 64, BF),
    ([300, 290, 0, 257], None, 256, 8, 2, 64, 16, F16),          # an unused slot
    ([256, 100, 300], None, 256, 8, 2, 128, 32, BF),             # nothing of its own; shorter than the prefix
    ([400 + i for i in range(70)], None, 384, 8, 4, 64, 128, F16),
    ([300, 280, 266], [4, 1, 9], 256, 8, 4, 128, 16, BF),
    ([700, 600], [150, 33], 448, 4, 2, 64, 64, F16),
    ([260, 258], [30, 1], 256, 4, 2, 128, 64, BF),               # new rows begin inside the prefix
    ([160 * 16 + 3] * 40, None, 160 * 16, 5, 1, 128, 16, BF),
    ([65], None, 64, 1, 1, 64, 64, BF),
]


@pytest.mark.parametrize("lens,new,prefix,hq,hkv,dim,page,dtype", PREFIX)
def test_shared_prefix(lens, new, prefix, hq, hkv, dim, page, dtype, table_room):
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=len(lens) + prefix, prefix=prefix,
                            spare_rows=0 if new is None else 2))
    out, lse = run(c)
    compare(c, out, lse)
    compare(c, *run(c, always=False))  # where sharing does not pay
    compare(c, *run(c, prefix=0))  # the same table without naming the prefix


def test_a_prefix_worth_sharing():
    """51 repeated readings of 4096 positions saved: shared without being told to."""
    lens = [4096 + 1 + 5 * i for i in range(52)]
    c = pc.batch(lens, None, 4, 1, 128, 64, BF, seed=31, prefix=4096)
    out, lse = run(c, always=False)
    compare(c, out, lse)
    told = run(c)
    assert torch.equal(out, told[0]) and torch.equal(lse, told[1])
    assert not torch.equal(lse, run(c, prefix=0)[1])  # another order of the same sums


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("new", [None, [40, 90]])
def test_large_scores(dtype, new, table_room):
    """Scores of some thousands: one position takes all, nothing overflows."""
    c = table_room(pc.batch([700, 260], new, 4, 2, 128, 64, dtype, seed=8, qscale=60.0))
    compare(c, *run(c, scale=3.0), scale=3.0)


@pytest.mark.parametrize("new", [None, [40, 90]])
def test_rising_scores(new, table_room):
    """Every position's score is above all before it: the running maximum moves at each step."""
    c = table_room(pc.batch([900, 333], new, 2, 1, 64, 32, BF, seed=9))
    c["q"][:] = 1.0
    for b in range(2):
        for p in range(int(c["lens"][b])):
            c["k"][c["table"][b, p // 32], :, p % 32] = p / 64
    compare(c, *run(c))


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,dtype", [
    ([90, 700, 33], [3, 2, 3], 10, 2, 128, 32, BF),      # a few drafted tokens
    ([2600, 41], [16, 16], 3, 3, 64, 16, F16),
    ([400, 131], [150, 131], 4, 2, 128, 64, BF),         # prompts
    ([700, 300], [260, 41], 5, 1, 64, 16, F16),
    ([3900], [600], 2, 1, 128, 128, F16),                # shared by many CTAs
])
def test_what_a_row_does_not_see_may_be_infinite_or_nan(lens, new, hq, hkv, dim, page, dtype, table_room):
    """Keys and values of later tokens reach no earlier row, whatever they hold; the rows that see them show it."""
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=41))
    clean = dict(c, k=c["k"].clone(), v=c["v"].clone())
    table, ls, starts = pc.lists(c)
    kinds = [float("inf"), float("-inf"), float("nan")]
    for b, (n, m) in enumerate(zip(lens, new)):
        for i, back in enumerate(sorted({1, 2, m // 2, m - 1} & set(range(1, m)))):  # `back` - 1 rows later than the last
            pos = n - back
            where = (table[b][pos // page], i % hkv, pos % page)
            c["v"][where][(7 * i) % dim] = kinds[i % 3]
            c["v"][where][dim - 1 - i] = kinds[(i + 1) % 3]
            clean["v"][where][(7 * i) % dim] = clean["v"][where][dim - 1 - i] = 0.0
        last = (table[b][(n - 1) // page], 0, (n - 1) % page)
        c["k"][last][3] = kinds[b % 3]
        clean["k"][last][3] = 0.0
    ref, fine = (op.attention(x["q"], x["k"], x["v"], table, ls, starts) for x in (c, clean))
    tol, ltol = op.attention_bounds(fine, dim, dtype)
    out, lse = run(c)
    o = out.double().reshape(c["rows"], hq, dim)
    sees_k = torch.zeros(c["rows"], hq, dtype=torch.bool)  # an unusual key: the sequences' last rows, kv head 0
    sees_k[[s - 1 for s in starts[1:]], :hq // hkv] = True
    odd = ~torch.isfinite(ref["out"]) & ~sees_k[..., None]
    assert odd.any() and torch.equal(torch.isnan(o)[odd], torch.isnan(ref["out"])[odd])
    inf = odd & torch.isinf(ref["out"])
    assert torch.equal(o[inf], ref["out"][inf])
    good = torch.isfinite(ref["out"]) & ~sees_k[..., None]
    assert ((o - ref["out"]).abs() <= tol)[good].all()
    assert ((lse.double() - ref["lse"]).abs() <= ltol)[~sees_k].all()


@pytest.mark.parametrize("new", [None, [40, 30]])
def test_a_nan_query_stays_in_its_row(new, table_room):
    c = table_room(pc.batch([300, 90], new, 4, 2, 128, 32, BF, seed=43))
    c["q"][1, 130] = float("nan")  # head 1 of row 1
    out, lse = run(c)
    odd = torch.zeros_like(lse, dtype=torch.bool)
    odd[1, 1] = True
    assert torch.equal(torch.isnan(lse), odd)
    assert torch.equal(torch.isnan(out.reshape(c["rows"], 4, 128)), odd[..., None].expand(-1, -1, 128))


@pytest.mark.parametrize("new", [None, [21, 64]])
@pytest.mark.parametrize("prefix", [0, 64])
def test_strides(new, prefix):
    """Pages stored (pages, slot, head, D) and interleaved k / v, wide q / out / lse rows."""
    c = pc.batch([200, 131], new, 8, 4, 128, 64, BF, seed=2, prefix=prefix, layout="nhd")
    compare(c, *run(c))
    rows = c["rows"]
    both = torch.full((c["k"].shape[0], 2, 4, 64, 128), float("nan"), dtype=BF)
    both[:, 0], both[:, 1] = c["k"], c["v"]
    d = both.to(DEV)
    wide = torch.zeros(rows, 3 * 1024, dtype=BF, device=DEV)
    wide[:, 1024:2048] = c["q"].to(DEV)
    out = torch.full((rows, 1024 + 64), 3.0, dtype=BF, device=DEV)
    lse = torch.full((rows, 40), 7.0, device=DEV)
    table = torch.full((2, c["table"].shape[1] + 5), -9, dtype=torch.int32, device=DEV)
    table[:, 2:-3] = c["table"].to(DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    args = (wide[:, 1024:2048], d[:, 0], d[:, 1], table[:, 2:-3], c["lens"].to(DEV))
    kw = dict(q_starts=starts, out=out[:, 64:], lse=lse[:, 16:24])
    _api().prefix_attention(*args, prefix, always=True, **kw) if prefix else _api().paged_attention(*args, **kw)
    torch.cuda.synchronize()
    assert (out[:, :64] == 3.0).all() and (lse[:, :16] == 7.0).all() and (lse[:, 24:] == 7.0).all()
    compare(c, out[:, 64:].cpu(), lse[:, 16:24].cpu())


@pytest.mark.parametrize("new", [None, [3, 70]])
def test_offsets_behind_two_gigabytes(new, table_room):
    """Pages more than 2^31 elements from the base."""
    c = table_room(pc.batch([200, 131], new, 4, 2, 128, 64, BF, seed=2))
    pages, step = c["k"].shape[0], (1 << 31) // (c["k"].shape[0] - 1) // 8 * 8 + 64
    k, v = (torch.empty(pages * step, dtype=BF, device=DEV).as_strided((pages, 2, 64, 128), (step, 8192, 128, 1))
            for _ in range(2))
    k.copy_(c["k"])
    v.copy_(c["v"])
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    lse = torch.empty(c["rows"], 4, device=DEV)
    out = _api().paged_attention(c["q"].to(DEV), k, v, c["table"].to(DEV), c["lens"].to(DEV), q_starts=starts, lse=lse)
    torch.cuda.synchronize()
    compare(c, out.cpu(), lse.cpu())


@pytest.mark.parametrize("new,prefix", [(None, 0), ([9, 150, 1], 0), (None, 128), ([9, 150, 1], 128)])
def test_reruns_are_bit_identical(new, prefix, table_room):
    c = table_room(pc.batch([900, 2000, 400], new, 16, 4, 128, 64, BF, seed=6, prefix=prefix))
    first = run(c)
    for _ in range(3):
        again = run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("new,prefix", [(None, 0), ([4, 80], 0), (None, 64)])
def test_captured_graphs(new, prefix, table_room):
    """Two graphs captured once, replayed at the same time on two streams with
    lengths, tables and rows changed in place after the capture."""
    P = _api()
    cases = [table_room(pc.batch([300, 500], new, 8, 4, 128, 64, BF, seed=s, prefix=prefix)) for s in (1, 2)]
    devs, graphs, outs, streams = [], [], [], []
    for c in cases:
        d = pc.to({k: c[k] for k in ("q", "k", "v", "table", "lens")}, DEV)
        d["starts"] = None if c["starts"] is None else c["starts"].to(DEV)
        out = torch.zeros(c["rows"], 8 * 128, dtype=BF, device=DEV)
        lse = torch.zeros(c["rows"], 8, device=DEV)

        def call():
            a = (d["q"], d["k"], d["v"], d["table"], d["lens"])
            kw = dict(q_starts=d["starts"], out=out, lse=lse)
            P.prefix_attention(*a, prefix, always=True, **kw) if prefix else P.paged_attention(*a, **kw)

        call()
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call()
        devs.append(d)
        graphs.append(graph)
        outs.append((out, lse))
        streams.append(st)
    changed = [pc.batch([190, 410], new, 8, 4, 128, 64, BF, seed=s + 10, prefix=prefix) for s in (1, 2)]
    for c, d in zip(changed, devs):
        pages, cols = min(c["k"].shape[0], d["k"].shape[0]), c["table"].shape[1]
        d["k"][:pages] = c["k"][:pages].to(DEV)
        d["v"][:pages] = c["v"][:pages].to(DEV)
        d["table"][:, :cols] = c["table"].to(DEV)
        d["lens"].copy_(c["lens"])
        d["q"].copy_(c["q"])
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for c, (out, lse) in zip(changed, outs):
        compare(c, out.cpu(), lse.cpu())


@pytest.mark.parametrize("new", [None, [5, 70, 1]])
def test_a_bad_page_is_flagged_and_harms_no_other_sequence(new, table_room):
    from breeze_b200 import _lib

    for bad in (-1, 10 ** 9):
        c = table_room(pc.batch([300, 200, 150], new, 4, 2, 128, 64, BF, seed=5))
        whole = c["table"].clone()
        c["table"][1, 1] = bad
        out, lse = run(c)
        assert _status() == _lib.BQ_DEVERR_PAGE
        c["table"] = whole
        rows = [0, 2] if new is None else [r for r in range(76) if not 5 <= r < 75]
        ref = op.attention(c["q"], c["k"], c["v"], *pc.lists(c))
        tol, _ = op.attention_bounds(ref, 128, BF)
        err = (out.double().reshape(c["rows"], 4, 128) - ref["out"]).abs()
        assert (err[rows] <= tol[rows]).all()


@pytest.mark.parametrize("new", [None, [1, 20]])
def test_a_length_behind_the_table_is_flagged(new):
    from breeze_b200 import _lib

    c = pc.batch([64, 128], new, 4, 2, 64, 64, BF, seed=5, spare_cols=0)
    c["lens"][1] = 10 ** 6
    run(c, causal=False)
    assert _status() == _lib.BQ_DEVERR_POSITION


def test_a_mixed_batch_with_tiles_of_few_rows():
    """Running streams of one token beside long new pieces, in the kernel for many
    rows: most of a tile's warps have no row, and must stay in step with the
    others over many units; repeated, since a step out of turn is a matter of time."""
    new = [200, 1, 3, 1, 130, 2, 1, 1, 40, 1, 1, 5]
    lens = [1500, 900, 2100, 1024, 700, 1300, 1700, 640, 2000, 129, 128, 1999]
    c = pc.batch(lens, new, 16, 4, 128, 64, BF, seed=21)
    first = run(c)
    compare(c, *first)
    for _ in range(20):
        again = run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_many_short_sequences():
    """More tiles than CTAs, most of them whole in one; some empty; repeated."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (300,), generator=g).tolist()
    for new in (None, [min(n, 1 + i % 23) for i, n in enumerate(lens)]):
        c = pc.batch(lens, new, 12, 6, 64, 16, F16, seed=22)
        compare(c, *run(c))
        compare(c, *run(c, max_q=100))


def test_more_sequences_than_threads():
    """Every thread that looks for a share's place has two sequences or more, in both kernels."""
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 60, (900,), generator=g).tolist()
    c = pc.batch(lens, [min(n, i % 4) for i, n in enumerate(lens)], 3, 1, 64, 16, BF, seed=23)
    compare(c, *run(c, max_q=3))
    compare(c, *run(c, max_q=100))


@pytest.mark.parametrize("new", [None, [40, 7, 300]])
def test_two_streams_at_once(new):
    """Calls that overlap on two streams share nothing."""
    P = _api()
    batches = [pc.to(pc.batch([900, 1300, 500], new, 8, 4, 128, 64, BF, seed=s), DEV) for s in (61, 62)]

    def call(c):
        lse = torch.empty(c["rows"], 8, device=DEV)
        return P.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], q_starts=c["starts"], lse=lse), lse

    alone = [call(c) for c in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(20):
        for c, st, to in zip(batches, streams, got):
            with torch.cuda.stream(st):
                to.append(call(c))
    torch.cuda.synchronize()
    for (out, lse), runs in zip(alone, got):
        for o2, l2 in runs:
            assert torch.equal(out, o2) and torch.equal(lse, l2)


# ------------------------------------------------------------------ append
def rope(positions, dim, dtype):
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


APPEND = [
    # lens, new, hq, hkv, dim, page, dtype, norm, table dtype, layout
    ([1], None, 1, 1, 128, 16, BF, True, BF, "hnd"),
    ([300, 17, 0, 64, 65], None, 16, 16, 128, 64, BF, True, BF, "hnd"),
    ([700, 31], None, 32, 8, 128, 16, F16, False, torch.float32, "nhd"),
    ([40, 20, 33], [40, 0, 7], 12, 4, 64, 16, F16, True, F16, "hnd"),
    ([2, 90], [4, 90], 3, 1, 64, 32, BF, True, torch.float32, "nhd"),  # positions under zero are skipped
    ([150] * 130, [1] * 130, 5, 5, 128, 128, BF, False, BF, "hnd"),
]


@pytest.mark.parametrize("lens,new,hq,hkv,dim,page,dtype,norm,cst,layout", APPEND)
@pytest.mark.parametrize("inplace", [False, True])
def test_append(lens, new, hq, hkv, dim, page, dtype, norm, cst, layout, inplace):
    c = pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=hq + dim, layout=layout, spare_rows=0 if new is None else 2)
    g = torch.Generator().manual_seed(11)
    rows = c["rows"]
    qkv = torch.randn(rows, (hq + 2 * hkv) * dim, generator=g).to(dtype)
    gains = [(1 + 0.1 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)] if norm else [None, None]
    cos, sin = rope(max(lens), dim, cst)
    table, ln, starts = pc.lists(c)
    q, written, terms = op.append(qkv, cos, sin, c["k"], c["v"], table, ln, starts, *gains)
    d = pc.to(c, DEV)
    x = qkv.to(DEV)
    out = x[:, :hq * dim] if inplace else torch.full((rows, hq * dim), 3.0, dtype=dtype, device=DEV)
    before = out.cpu().clone()
    res = _api().paged_append(x, cos.to(DEV), sin.to(DEV), d["k"], d["v"], d["table"], d["lens"], q_starts=d["starts"],
                              q_norm_w=None if not norm else gains[0].to(DEV),
                              k_norm_w=None if not norm else gains[1].to(DEV), out=out)
    torch.cuda.synchronize()
    assert res is out
    u = torch.finfo(dtype).eps / 2
    # one rounding of the result; the fp32 norm (a sum of D squares halved by the root, three
    # products) and rotation (three roundings) move each of its two terms by under (D / 2 + 8) 2^-24
    tol = lambda y, t: u * y.abs() + (dim / 2 + 8) * 2.0 ** -24 * t + (2.0 ** -25 if dtype == F16 else 0.0)  # noqa: E731
    got = out.cpu().double().reshape(rows, hq, dim)
    skipped = torch.isnan(q[:, 0, 0])
    assert torch.equal(out.cpu()[skipped], before[skipped])
    keep = ~skipped
    assert ((got[keep] - q[keep]).abs() <= tol(q, terms[:, :hq])[keep]).all()
    k_want, v_want = c["k"].clone(), c["v"].clone()
    k_got, v_got = d["k"].cpu(), d["v"].cpu()
    for (pg, slot), (t, k, v) in written.items():
        assert ((k_got[pg, :, slot].double() - k).abs() <= tol(k, terms[t, hq:])).all()
        v_want[pg, :, slot] = v.to(dtype)
        k_want[pg, :, slot] = k_got[pg, :, slot]
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))  # noqa: E731
    assert same(v_got, v_want) and same(k_got, k_want)  # v to the bit, every other slot untouched


def test_append_flags_what_does_not_fit():
    from breeze_b200 import _lib

    cases = [("page", _lib.BQ_DEVERR_PAGE), ("table", _lib.BQ_DEVERR_POSITION), ("rope", _lib.BQ_DEVERR_POSITION)]
    for what, bit in cases:
        c = pc.batch([40, 20], None, 2, 1, 64, 16, BF, seed=1, spare_cols=0)
        qkv = torch.randn(2, 4 * 64, generator=torch.Generator().manual_seed(12)).to(BF)
        cos, sin = rope(30 if what == "rope" else 64, 64, BF)
        if what == "page":
            c["table"][0, 2] = -3
        if what == "table":
            c["lens"][0] = 49
        d = pc.to(c, DEV)
        out = torch.full((2, 128), 300.0, dtype=BF, device=DEV)  # no q is that large
        _api().paged_append(qkv.to(DEV), cos.to(DEV), sin.to(DEV), d["k"], d["v"], d["table"], d["lens"], out=out)
        torch.cuda.synchronize()
        assert _status() == bit
        assert (out[0] == 300.0).all() and not (out[1] == 300.0).any()
        k = d["k"].cpu()
        changed = (k.view(torch.int16) != c["k"].view(torch.int16)).any(-1).any(1).nonzero().tolist()
        assert changed == [[int(c["table"][1, 1]), 3]]


def test_append_then_attention_follows_a_growing_batch():
    """Prompts in one ragged call, then decode steps: append and attention as a
    server runs them, against the oracle over the cache the appends wrote."""
    P = _api()
    hq, hkv, dim, page = 8, 4, 128, 16
    c = pc.batch([37, 5, 50], [37, 5, 50], hq, hkv, dim, page, BF, seed=3, spare_cols=2)
    lens, cols = [37, 5, 50], c["table"].shape[1]
    pages = 3 * cols
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(3, cols)
    k = torch.full((pages, hkv, page, dim), float("nan"), dtype=BF, device=DEV)
    v = k.clone()
    cos, sin = rope(cols * page, dim, torch.float32)
    g = torch.Generator().manual_seed(4)
    dt, dl = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    for step in range(6):
        starts = torch.tensor([0, 37, 42, 92], dtype=torch.int32) if step == 0 else None
        rows = 92 if step == 0 else 3
        if step:
            lens = [n + 1 for n in lens]
            dl += 1
        qkv = torch.randn(rows, (hq + 2 * hkv) * dim, generator=g).to(BF)
        ds = None if starts is None else starts.to(DEV)
        q = P.paged_append(qkv.to(DEV), cos.to(DEV), sin.to(DEV), k, v, dt, dl, q_starts=ds)
        lse = torch.empty(rows, hq, device=DEV)
        out = P.paged_attention(q, k, v, dt, dl, q_starts=ds, lse=lse)
        torch.cuda.synchronize()
        case = dict(c, q=q.cpu(), k=k.cpu(), v=v.cpu(), table=table, lens=torch.tensor(lens), starts=starts, rows=rows)
        compare(case, out.cpu(), lse.cpu())


def test_python_refusals():
    P = _api()
    c = pc.to(pc.batch([40, 20], None, 4, 2, 64, 16, BF, seed=1), DEV)
    cos, sin = (t.to(DEV) for t in rope(64, 64, BF))
    qkv = torch.zeros(2, 8 * 64, dtype=BF, device=DEV)
    good = dict(q=c["q"], k_pages=c["k"], v_pages=c["v"], page_table=c["table"], seq_lens=c["lens"])
    for change, error, text in [
        (dict(q=c["q"].float()), ValueError, "one dtype"),
        (dict(q=c["q"].float(), k_pages=c["k"].float(), v_pages=c["v"].float()), ValueError, "bf16 or fp16"),
        (dict(q=c["q"].half()), ValueError, "one dtype"),
        (dict(q=c["q"][:, :100]), ValueError, "does not split"),
        (dict(q=c["q"][:, ::2]), ValueError, "unit stride"),
        (dict(q=c["q"][:1]), ValueError, "ragged rows need q_starts"),
        (dict(q=c["q"][:, :192]), ValueError, "does not split"),
        (dict(v_pages=c["v"][1:]), ValueError, "one shape"),
        (dict(k_pages=c["k"].transpose(2, 3)), ValueError, "one shape|contiguous"),
        (dict(page_table=c["table"].long()), ValueError, "int32"),
        (dict(page_table=c["table"].t()), ValueError, "contiguous rows|seq_lens"),
        (dict(seq_lens=c["lens"].long()), ValueError, "int32"),
        (dict(seq_lens=c["lens"][:1]), ValueError, "int32"),
        (dict(q_starts=torch.zeros(2, dtype=torch.int32, device=DEV)), ValueError, "q_starts"),
        (dict(seq_lens=c["lens"].cpu()), RuntimeError, "different devices"),
        (dict(out=torch.empty(2, 128, dtype=BF, device=DEV)), ValueError, "out must be"),
        (dict(lse=torch.empty(2, 4, dtype=BF, device=DEV)), ValueError, "lse must be"),
        (dict(scale=-1.0), ValueError, "scale"),
    ]:
        with pytest.raises(error, match=text):
            P.paged_attention(**{**good, **change})
    with pytest.raises(ValueError, match="multiple of the page size"):
        P.prefix_attention(**good, prefix_len=17)
    put = dict(qkv=qkv, cos=cos, sin=sin, k_pages=c["k"], v_pages=c["v"], page_table=c["table"], seq_lens=c["lens"])
    for change, error, text in [
        (dict(qkv=qkv[:, :4 * 64]), ValueError, "does not split"),
        (dict(qkv=qkv[:, :500]), ValueError, "does not split"),
        (dict(cos=cos.half()), ValueError, "cos and sin"),
        (dict(cos=cos.half(), sin=sin.half()), ValueError, "fp32 or the cache's dtype"),
        (dict(cos=cos[:, :32], sin=sin[:, :32]), ValueError, "cos and sin"),
        (dict(q_norm_w=cos[0]), ValueError, "go together"),
        (dict(q_norm_w=cos[0], k_norm_w=sin[0].float()), ValueError, "norm weights"),
        (dict(out=qkv), ValueError, "out must be"),
        (dict(sin=sin.cpu()), RuntimeError, "another device"),
    ]:
        with pytest.raises(error, match=text):
            P.paged_append(**{**put, **change})


class _Aside:
    """Stands in for the compiled calls: leaves every call to Python."""

    @staticmethod
    def append(*args):
        assert len(args) == 13

    @staticmethod
    def attention(*args):
        assert len(args) == 12


@pytest.mark.parametrize("new", [None, [3, 70]])
def test_compiled_calls_and_python_do_the_same(new, monkeypatch):
    P = _api()
    c = pc.batch([600, 131], new, 4, 2, 64, 32, BF, seed=51, prefix=64)
    cos, sin = (t.to(DEV) for t in rope(600, 64, BF))
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(c["rows"], 8 * 64, generator=g).to(BF).to(DEV)
    gain = torch.nn.Parameter((1 + 0.1 * torch.randn(64, generator=g)).to(BF).to(DEV))  # weights come as parameters

    def calls():
        d = pc.to(c, DEV)
        where = (d["k"], d["v"], d["table"], d["lens"])
        kw = dict(q_starts=d["starts"])
        q = P.paged_append(qkv, cos, sin, *where, q_norm_w=gain, k_norm_w=gain, eps=1e-5, **kw)
        inplace = torch.empty_like(q)
        assert P.paged_append(qkv, cos, sin, *where, out=inplace, **kw) is inplace
        lse = torch.empty(c["rows"], 4, device=DEV)
        outs = [q, inplace, lse, d["k"], d["v"], P.paged_attention(q, *where, scale=0.2, causal=False, max_q=2, **kw),
                P.paged_attention(q, *where, lse=lse, **kw), P.prefix_attention(q, *where, 64, always=True, **kw)]
        out = torch.empty_like(q)
        assert P.paged_attention(q, *where, out=out, **kw) is out
        assert not q.requires_grad
        torch.cuda.synchronize()
        return outs + [out]

    with monkeypatch.context() as m:
        m.setattr(P, "_cache_fields", None)  # plain calls never reach Python's checks
        fast = calls()
    monkeypatch.setattr(P, "_bound", _Aside)
    for a, b in zip(fast, calls(), strict=True):
        assert torch.equal(a.nan_to_num(), b.nan_to_num()) and a.dtype == b.dtype and a.stride() == b.stride()


def test_no_rows():
    """A ragged call without new rows is answered without a launch."""
    P = _api()
    c = pc.to(pc.batch([40, 20], None, 4, 2, 64, 16, BF, seed=1), DEV)
    starts = torch.zeros(3, dtype=torch.int32, device=DEV)
    cos, sin = (t.to(DEV) for t in rope(64, 64, BF))
    args = (c["k"], c["v"], c["table"], c["lens"])
    empty = torch.empty(0, 8 * 64, dtype=BF, device=DEV)
    assert P.paged_append(empty, cos, sin, *args, q_starts=starts).shape == (0, 4 * 64)
    assert P.paged_attention(empty[:, :256], *args, q_starts=starts).shape == (0, 256)
    assert P.prefix_attention(empty[:, :256], *args, 16, q_starts=starts).shape == (0, 256)
