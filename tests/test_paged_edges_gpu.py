"""Paged-cache operators where the definition is easily missed: values that only
some rows of a shared prefix see, unused slots before it, scores of minus
infinity, cut lengths, strides of dimensions of size one, long caches. Against
the 64-bit oracle, within the bounds derived there."""

import pytest
import torch

from oracle import paged as op
from tests import paged_cases as pc
from tests.test_paged_gpu import _clean_status, _status, compare, run, table_room  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = pc.BF, pc.F16
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("lens,new,prefix,hq,hkv,dim,page,dtype,at", [
    ([260, 258], [30, 1], 256, 4, 2, 128, 64, BF, [(250, INF), (235, NAN)]),         # new rows begin inside the prefix
    ([256, 100, 300], [40, 40, 40], 256, 8, 2, 128, 32, BF, [(99, -INF), (200, NAN)]),  # one ends in it
    ([700, 600], [150, 33], 640, 4, 2, 64, 64, F16, [(580, INF), (639, -INF), (555, NAN)]),
    ([1500, 1033], [500, 20], 1024, 2, 2, 128, 16, BF, [(1001, INF), (1022, NAN), (1010, -INF)]),
    ([70, 66, 40], None, 64, 2, 1, 128, 16, BF, [(50, INF), (39, NAN)]),             # few rows
    ([70, 66, 40], [5, 3, 1], 64, 1, 1, 64, 16, F16, [(63, NAN), (39, INF)]),
])
def test_a_prefix_value_reaches_only_the_rows_that_see_it(lens, new, prefix, hq, hkv, dim, page, dtype, at):
    c = pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=47, prefix=prefix)
    clean = dict(c, v=c["v"].clone())
    table, ls, starts = pc.lists(c)
    for i, (pos, what) in enumerate(at):
        where = (table[0][pos // page], i % hkv, pos % page)
        c["v"][where][5 * i + 1] = what
        clean["v"][where][5 * i + 1] = 0.0
    ref, fine = (op.attention(x["q"], x["k"], x["v"], table, ls, starts) for x in (c, clean))
    tol, ltol = op.attention_bounds(fine, dim, dtype)
    good = torch.isfinite(ref["out"])
    assert not good.all() and good.any(-1).all()
    for always in (True, False):
        out, lse = run(c, always=always)
        o = out.double().reshape(c["rows"], hq, dim)
        assert torch.isfinite(o)[good].all()
        assert ((o - ref["out"]).abs() <= tol)[good].all()
        assert torch.equal(torch.isnan(o)[~good], torch.isnan(ref["out"])[~good])
        inf = torch.isinf(ref["out"])
        assert torch.equal(o[inf], ref["out"][inf])
        assert ((lse.double() - ref["lse"]).abs() <= ltol).all()


@pytest.mark.parametrize("hole", [2 ** 30, -1])
@pytest.mark.parametrize("lens,new,prefix,hq,hkv,dim,page,dtype", [
    ([0, 300, 290, 257], None, 256, 8, 2, 64, 16, F16),           # slot 0 is unused
    ([0, 0, 1100, 1024, 1300], None, 1024, 32, 8, 128, 64, BF),
    ([100, 256, 300], None, 256, 8, 2, 128, 32, BF),              # slot 0 ends in the prefix
    ([0, 700, 600], [0, 150, 33], 448, 4, 2, 64, 64, F16),        # no new rows in slot 0
    ([200, 260, 258], [90, 30, 1], 256, 4, 2, 128, 64, BF),
    ([40, 90, 33], None, 128, 4, 2, 128, 16, BF),                 # nobody reaches the prefix's end
    ([0, 0], None, 64, 4, 2, 64, 16, BF),                         # nobody at all
])
def test_unused_slots_need_no_prefix_pages(lens, new, prefix, hq, hkv, dim, page, dtype, hole):
    c = pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=len(lens) + prefix, prefix=prefix)
    for b, n in enumerate(lens):
        c["table"][b, -(-n // page):] = hole
    if new is not None and new[0] == 0:  # nor does a sequence without new rows, whatever its length says
        c["table"][0, :] = hole
        c["lens"][0] = 10 ** 6 if hole < 0 else 2
        lens = c["lens"].tolist()
    out, lse = run(c, always=True)
    if new is not None and new[0] == 0 and hole < 0:
        from breeze_b200 import _lib

        assert _status() == _lib.BQ_DEVERR_POSITION
    compare(c, out, lse)
    compare(c, *run(dict(c, lens=c["lens"].clamp(max=c["table"].shape[1] * page)), always=False))


MINUS = [
    # lens, new, prefix, hq, hkv, dim, page, dtype
    ([300, 90], None, 0, 4, 2, 128, 32, BF),
    ([2000, 5], None, 0, 2, 1, 64, 16, F16),
    ([900, 333], [40, 30], 0, 4, 2, 128, 32, BF),
    ([4000], [300], 0, 2, 1, 64, 64, F16),
    ([300, 280], [4, 9], 256, 4, 2, 128, 16, BF),
    ([700, 600], [150, 33], 448, 4, 2, 64, 64, F16),
    ([700, 690], None, 640, 2, 2, 128, 64, BF),
]


@pytest.mark.parametrize("lens,new,prefix,hq,hkv,dim,page,dtype", MINUS)
@pytest.mark.parametrize("single", [True, False])
def test_scores_of_minus_infinity(lens, new, prefix, hq, hkv, dim, page, dtype, single, table_room):  # noqa: F811
    """All of a row's scores -inf: the softmax is 0 / 0, the row NaN, its lse -inf
    (the logarithm of 0). With one finite score among them (``single``: the rows
    that see position lens[0] / 2 of sequence 0) the row is that v."""
    c = table_room(pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=53, prefix=prefix))
    table, ls, starts = pc.lists(c)
    c["k"][..., 7] = -INF  # everywhere, but at one position
    alone = lens[0] // 2
    if single:
        c["k"][table[0][alone // page], :, alone % page] = 0.5
    c["q"].view(-1, hq, dim)[..., 7] = 1.0
    q = c["q"].view(-1, hq, dim)
    q[0, 0, 7] = 0.0  # 0 * -inf: NaN scores
    ref = op.attention(c["q"], c["k"], c["v"], table, ls, starts)
    out, lse = run(c)
    o = out.double().reshape(c["rows"], hq, dim)
    first = torch.zeros(c["rows"], hq, dtype=torch.bool)
    first[0, 0] = True
    assert torch.equal(torch.isnan(o), torch.isnan(ref["out"]))
    assert torch.equal(torch.isnan(lse), first)
    none = torch.isinf(ref["lse"])
    assert (none.any() or single) and torch.equal(lse[none], ref["lse"][none].float())
    rest = torch.isfinite(ref["lse"])
    if rest.any():  # one position takes all: v itself, within the output's rounding
        u = torch.finfo(dtype).eps / 2
        assert ((o - ref["out"]).abs() <= u * ref["out"].abs() + 2.0 ** -22)[rest].all()
        # |score| <= sum |q k| terms of which each of D + 8 roundings takes 2^-23
        bound = (dim + 8) * 2.0 ** -23 * (c["q"].double().abs().sum(-1).max() / 2 + 1)
        assert ((lse.double() - ref["lse"]).abs()[rest] <= bound).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,prefix,dim", [(None, 0, 64), ([1, 20], 0, 64), ([1, 100], 0, 128), ([70, 100], 0, 64),
                                            ([1, 20], 64, 64), ([1, 100], 64, 128), (None, 64, 128)])
def test_a_cut_length_reads_what_the_table_holds(causal, new, prefix, dim):
    from breeze_b200 import _lib

    c = pc.batch([200, 256], new, 4, 2, dim, 64, BF, seed=5, spare_cols=0, prefix=prefix)
    ref = op.attention(c["q"], c["k"], c["v"], *pc.lists(c), None, causal)
    full = op.attention(c["q"], c["k"], c["v"], *pc.lists(c), None, False)  # its rows all lie behind the table
    cut = 1 if new is None else new[0]
    want = {k: torch.cat([ref[k][:cut], full[k][cut:]]) for k in ("out", "lse", "weight", "terms", "seen")}
    tol, ltol = op.attention_bounds(dict(want, vmax=full["vmax"]), dim, BF)
    c["lens"][1] = 10 ** 6
    out, lse = run(c, causal=causal)
    assert _status() == _lib.BQ_DEVERR_POSITION
    assert ((out.double().reshape(want["out"].shape) - want["out"]).abs() <= tol).all()
    assert ((lse.double() - want["lse"]).abs() <= ltol).all()


@pytest.mark.parametrize("new", [None, [70, 3]])
@pytest.mark.parametrize("stride", [0, 1, 4, 2 ** 41])
def test_strides_of_dimensions_of_size_one(new, stride):
    """One kv head, one page, one sequence, one query head: what their strides say does not matter."""
    from breeze_b200.fused import paged

    c = pc.batch([200, 131], new, 4, 1, 128, 64, BF, seed=2)
    same = lambda t, dims: t.as_strided(t.shape, [stride if i in dims else s for i, s in enumerate(t.stride())])  # noqa: E731
    d = pc.to(c, DEV)
    lse = torch.empty(c["rows"], 4, device=DEV)
    out = paged.paged_attention(d["q"], same(d["k"], [1]), same(d["v"], [1]), d["table"], d["lens"], q_starts=d["starts"], lse=lse)
    torch.cuda.synchronize()
    compare(c, out.cpu(), lse.cpu())
    rows = 1 if new is None else 70
    c = pc.batch([50], None if new is None else [50], 1, 1, 64, 64, BF, seed=2, spare_cols=0)
    c["k"], c["v"], c["table"] = c["k"][int(c["table"][0, 0])][None], c["v"][int(c["table"][0, 0])][None], torch.zeros(1, 1, dtype=torch.int32)
    d = pc.to(c, DEV)
    rows = c["rows"]
    lse = torch.empty(rows, 1, device=DEV)
    out = paged.paged_attention(same(d["q"], [0] if rows == 1 else []), same(d["k"], [0, 1]), same(d["v"], [0, 1]), same(d["table"], [0, 1]),
                                same(d["lens"], [0]), q_starts=d["starts"], lse=same(lse, [1] if rows > 1 else [0, 1]))
    torch.cuda.synchronize()
    compare(c, out.cpu(), lse.cpu())


def test_a_length_far_below_zero_is_an_unused_slot():
    from breeze_b200.fused import paged

    for new in (None, [3, 2]):
        c = pc.batch([5, 20], new, 2, 1, 64, 16, BF, seed=1)
        c["lens"][0] = -2 ** 31
        d = pc.to(c, DEV)
        rows = c["rows"]
        qkv = torch.randn(rows, 4 * 64, generator=torch.Generator().manual_seed(12)).to(BF).to(DEV)
        table = torch.ones(64, 64, device=DEV)
        out = torch.full((rows, 128), 300.0, dtype=BF, device=DEV)
        paged.paged_append(qkv, table, table, d["k"], d["v"], d["table"], d["lens"], q_starts=d["starts"], out=out)
        torch.cuda.synchronize()
        dead = rows - (1 if new is None else 2)
        assert (out[:dead] == 300.0).all() and not (out[dead:] == 300.0).any(-1).any()


@pytest.mark.parametrize("prefix", [0, 64])
@pytest.mark.parametrize("hq,dim", [(2, 128), (8, 64)])
def test_rows_before_the_first_sequence_are_left(prefix, hq, dim, table_room):  # noqa: F811
    """q_starts[0] > 0: the rows before it belong to nobody, as those behind the last."""
    c = table_room(pc.batch([130, 90, 300], [20, 1, 40], hq, 2, dim, 32, BF, seed=6, prefix=prefix, spare_rows=9))
    lead = 5
    moved = dict(c, starts=c["starts"] + lead)
    out, lse = run(moved)
    assert (out[:lead] == 3.0).all() and (lse[:lead] == 7.0).all()
    table, lens, starts = pc.lists(moved)
    ref = op.attention(c["q"], c["k"], c["v"], table, lens, starts)
    tol, ltol = op.attention_bounds(ref, dim, BF)
    rows = slice(lead, starts[-1])
    assert ((out.double().reshape(c["rows"], hq, dim) - ref["out"]).abs() <= tol)[rows].all()
    assert ((lse.double() - ref["lse"]).abs() <= ltol)[rows].all()
    assert (out[starts[-1]:] == 3.0).all()


@pytest.mark.parametrize("lens,new,prefix,hq,hkv,dim,page,dtype", [
    ([32000, 24001], None, 0, 4, 1, 128, 128, BF),
    ([31999, 7], [3, 2], 0, 2, 1, 64, 16, F16),
    ([5003], [5003], 0, 1, 1, 128, 64, BF),
    ([12300, 12401, 12288], [1, 5, 2], 12288, 4, 1, 128, 64, BF),
    ([20000], [300], 0, 1, 1, 64, 256, BF),
])
def test_long_caches(lens, new, prefix, hq, hkv, dim, page, dtype):
    c = pc.batch(lens, new, hq, hkv, dim, page, dtype, seed=71, prefix=prefix)
    compare(c, *run(c))


@pytest.mark.parametrize("dim,hq", [(64, 3), (64, 5), (128, 7)])
def test_several_tiles_of_a_cluster(dim, hq):
    """max_q told too low: a cluster walks many tiles of odd heights; repeated, since
    a tile written too early is a matter of time."""
    c = pc.batch([300, 77], [61, 33], hq, 1, dim, 32, BF, seed=33, spare_cols=0)
    first = run(c, max_q=1)
    compare(c, *first)
    for _ in range(50):
        again = run(c, max_q=1)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_maximum_that_moves_at_every_unit():
    """In the kernel for many rows each unit's probabilities are then written twice; repeated."""
    c = pc.batch([1900], [260], 2, 1, 128, 64, BF, seed=9)
    c["q"][:] = 1.0
    for p in range(1900):
        c["k"][c["table"][0, p // 64], :, p % 64] = p / 64
    first = run(c)
    compare(c, *first)
    for _ in range(50):
        again = run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


class _Aside:
    """Stands in for the compiled calls: leaves every call to Python."""

    @staticmethod
    def append(*args):
        return None

    attention = append


@pytest.mark.parametrize("compiled", [True, False])
def test_compiled_calls_and_python_refuse_the_same(compiled, monkeypatch):
    """Whichever checks a call, what may not run is refused, by the same kind of error."""
    from breeze_b200.fused import paged

    paged._native()
    if not compiled:
        monkeypatch.setattr(paged, "_bound", _Aside)
    c = pc.to(pc.batch([40, 20], None, 4, 2, 64, 16, BF, seed=1), DEV)
    q, k, v, table, lens = (c[n] for n in ("q", "k", "v", "table", "lens"))
    cs = torch.ones(64, 64, dtype=BF, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    rows = torch.zeros(2, 8 * 64, dtype=BF, device=DEV)
    shared = [
        (dict(k_pages=k.half()), ValueError), (dict(v_pages=v.float()), ValueError), (dict(k_pages=k[0]), ValueError),
        (dict(v_pages=v[:, :1]), ValueError), (dict(k_pages=k.transpose(2, 3)), ValueError),
        (dict(k_pages=k[..., :32], v_pages=v[..., :32]), ValueError), (dict(k_pages=k[:, :, :8], v_pages=v[:, :, :8]), ValueError),
        (dict(k_pages=k[:0], v_pages=v[:0]), ValueError), (dict(k_pages=k.expand(2, *k.shape)[0][:1].expand(k.shape)), ValueError),
        (dict(k_pages=k.view(-1)[4:][:k[1:].numel()].view_as(k[1:]), v_pages=v[1:]), ValueError),  # 8-byte aligned
        (dict(page_table=table.long()), ValueError), (dict(page_table=table[0]), ValueError),
        (dict(page_table=table.repeat(1, 2)[:, ::2]), ValueError), (dict(page_table=table[:, :0]), ValueError),
        (dict(page_table=table[:1].expand(2, -1)), ValueError), (dict(seq_lens=lens.long()), ValueError),
        (dict(seq_lens=lens[:1]), ValueError), (dict(seq_lens=lens.repeat(2)[::2]), ValueError),
        (dict(seq_lens=lens.cpu()), RuntimeError), (dict(page_table=table.cpu()), RuntimeError),
        (dict(k_pages=k.cpu(), v_pages=v.cpu()), RuntimeError), (dict(q_starts=torch.zeros(2, **i32)), ValueError),
        (dict(q_starts=torch.zeros(3, device=DEV)), ValueError), (dict(q_starts=torch.zeros(3, dtype=torch.int32)), RuntimeError),
    ]
    attention = shared + [
        (dict(q=q.float()), ValueError), (dict(q=q[0]), ValueError), (dict(q=q[:, ::2]), ValueError), (dict(q=q[:1]), ValueError),
        (dict(q=q[:, :192]), ValueError), (dict(q=q[:, :100]), ValueError), (dict(q=q.cpu()), RuntimeError),
        (dict(q=q[:1].expand(2, -1)), ValueError), (dict(out=q.float()), ValueError), (dict(out=q[:, :128]), ValueError),
        (dict(out=q.cpu()), ValueError), (dict(out=torch.empty_like(q[:1]).expand(2, -1)), ValueError),
        (dict(lse=torch.empty(2, 4, dtype=BF, device=DEV)), ValueError), (dict(lse=torch.empty(2, 4)), ValueError),
        (dict(lse=torch.empty(4, 2, device=DEV).t()), ValueError), (dict(lse=torch.empty(2, 3, device=DEV)), ValueError),
        (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError),
        (dict(scale=float("inf")), ValueError), (dict(scale=1e39), ValueError), (dict(scale=3e38), ValueError),
        (dict(scale="1"), TypeError), (dict(max_q=-1), ValueError), (dict(max_q=2 ** 31), ValueError),
        (dict(max_q=2 ** 70), ValueError), (dict(max_q=1.5), TypeError), (dict(prefix_len=17), ValueError),
        (dict(prefix_len=-16), ValueError), (dict(prefix_len=2 ** 31), ValueError), (dict(prefix_len=2 ** 70), ValueError),
        (dict(prefix_len=16.0), TypeError), (dict(prefix_len=16 * 100), ValueError),
    ]
    append = shared + [
        (dict(qkv=rows.float()), ValueError), (dict(qkv=rows[:, :4 * 64]), ValueError), (dict(qkv=rows[:, :500]), ValueError),
        (dict(qkv=rows.cpu()), RuntimeError), (dict(qkv=rows[:1]), ValueError), (dict(cos=cs.half()), ValueError),
        (dict(cos=cs.half(), sin=cs.half()), ValueError), (dict(cos=cs[:, :32], sin=cs[:, :32]), ValueError),
        (dict(cos=cs[:0], sin=cs[:0]), ValueError), (dict(cos=cs[:32]), ValueError), (dict(sin=cs.cpu()), RuntimeError),
        (dict(cos=cs[:1].expand(64, -1), sin=cs[:1].expand(64, -1)), ValueError), (dict(q_norm_w=cs[0]), ValueError),
        (dict(q_norm_w=cs[0], k_norm_w=cs[0].float()), ValueError), (dict(q_norm_w=cs[0], k_norm_w=cs[:, 0]), ValueError),
        (dict(q_norm_w=cs[0].cpu(), k_norm_w=cs[0].cpu()), ValueError), (dict(out=rows), ValueError),
        (dict(out=rows[:, :256].float()), ValueError), (dict(eps=1e39), ValueError), (dict(eps=float("nan")), ValueError),
        (dict(eps=float("inf")), ValueError), (dict(eps="0"), TypeError),
    ]
    where = dict(k_pages=k, v_pages=v, page_table=table, seq_lens=lens)
    for call, good, bad in ((paged.prefix_attention, dict(where, q=q, prefix_len=16), attention),
                            (paged.paged_append, dict(where, qkv=rows, cos=cs, sin=cs), append)):
        for change, error in bad:
            with pytest.raises(error):
                call(**{**good, **change})
                pytest.fail(f"{call.__name__} took {sorted(change)}: {bad.index((change, error))}")


@pytest.mark.parametrize("lens,new,prefix,hq,dim", [
    ([90, 300], None, 0, 128, 128), ([300, 33], [1, 9], 0, 128, 64),    # a token is a box of queries
    ([90, 300], None, 0, 256, 64), ([130, 140], [3, 2], 128, 256, 64),  # a tile is one token
    ([70], [5], 0, 300, 64), ([200, 190], None, 128, 300, 128),         # a token goes on in the next tile
    ([700], [40], 0, 96, 64),
])
def test_many_query_heads_on_one_kv_head(lens, new, prefix, hq, dim, table_room):  # noqa: F811
    c = table_room(pc.batch(lens, new, hq, 1, dim, 32, BF, seed=81, prefix=prefix))
    compare(c, *run(c))


@pytest.mark.parametrize("what", ["append", "cluster", "narrow", "wide", "prefix"])
def test_a_first_call_inside_a_capture(what):
    """A process whose first paged call is captured: nothing that a capture forbids is left to the first call."""
    code = f"""
import torch
from breeze_b200 import _lib
from breeze_b200.fused import paged
from tests import paged_cases as pc
what = {what!r}
new = None if what in ("append", "cluster", "narrow") else [100, 60]
c = pc.batch([300, 200], new, 4, 2, 128, 64, torch.bfloat16, seed=1, prefix=128 if what == "prefix" else 0)
if what == "narrow":
    c["table"] = torch.nn.functional.pad(c["table"], (0, 1000), value=-1)
d = pc.to(c, "cuda")
where = (d["k"], d["v"], d["table"], d["lens"])
rows = torch.ones(2, 8 * 128, dtype=torch.bfloat16, device="cuda")
cs = torch.ones(512, 128, device="cuda")
def call():
    if what == "append":
        return paged.paged_append(rows, cs, cs, *where)
    if what == "prefix":
        return paged.prefix_attention(d["q"], *where, 128, q_starts=d["starts"], always=True)
    return paged.paged_attention(d["q"], *where, q_starts=d["starts"])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = call()
out.zero_()
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, call()) and out.abs().sum() > 0 and _lib.device_status(0) == 0
"""
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
