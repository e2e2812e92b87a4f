"""8-bit paged cache, far ends of its ranges: scores so large that fp32 steps over whole units, scales as far apart
and factors as small as they go. Tolerances stand beside each case."""

import math

import pytest
import torch

from oracle import paged8 as o8
from tests import paged_fp8_cases as pc
from tests.test_paged_fp8_gpu import DEV, _api, _clean_status, oracle, run, table_room, where  # noqa: F401

pytestmark = pytest.mark.gpu
BF, F16, F8, E8 = pc.BF, pc.F16, pc.F8, pc.E8
LOG2E = 1.4426950408889634

# one token per sequence, and rows for the kernels of few (12 per kv head) and of many (130)
FORMS = [([700, 260], None), ([700, 260], [6, 5]), ([700, 260], [40, 90])]


def fill(c, values):
    """Keys: the same value in every dim, values(b, p) at position p of sequence b."""
    k = torch.zeros(c["k"].shape)
    for b, n in enumerate(c["lens"].tolist()):
        for p in range(n):
            k[c["table"][b, p // c["page"]], :, p % c["page"]] = values(b, p)
    c["k"], c["ks"] = pc.quantise(k, c["used"], c["block"])


def visible(c):
    """Sequence and visible positions of every row."""
    lens = c["lens"].tolist()
    starts = list(range(len(lens) + 1)) if c["starts"] is None else c["starts"].tolist()
    for b, n in enumerate(lens):
        for r in range(starts[b], starts[b + 1]):
            yield r, b, n - starts[b + 1] + r + 1


def gathered(c, codes, scales, b, n):
    """(HKV, n, D) in 64 bits."""
    x = o8.values(codes, scales)[c["table"][b, :-(-n // c["page"])].long()]
    return x.transpose(0, 1).reshape(c["hkv"], -1, c["dim"])[:, :n]


LARGE = [7e5, 2.0 ** 22, 2.0 ** 24 + 2, 3.1e7, 2.0 ** 25, 1.3e8, 2.0 ** 28, 1e9, 7e9, 1e30, -2.0 ** 24, -3.1e7, -1e9, -7e9]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lens,new", FORMS)
@pytest.mark.parametrize("top", LARGE)
def test_one_large_score_takes_all(top, lens, new, dtype, table_room):
    """The largest score, `top` in base 2, is a seventh of |top| or more above the others: its probability is 1 whatever
    the scores' roundings, and the row is that position's value, exactly (four significant bits, sums of zeros)."""
    dim = 128
    c = table_room(pc.batch(lens, new, 4, 2, dim, 32, 16, dtype, seed=3, levels=2))
    best, sign = (1.75, 1.0) if top > 0 else (0.25, -1.0)
    c["q"][:] = sign
    at = [5, 130]
    others = [0.5, 0.75, 1.0, 1.25, 1.5]
    fill(c, lambda b, p: best if p == at[b] else others[(p * 7) % 5])
    scale = abs(top) / (best * dim * LOG2E)
    out, lse = run(c, scale=scale)
    o = out.double().reshape(c["rows"], 4, dim)
    for r, b, n in visible(c):
        want = gathered(c, c["v"], c["vs"], b, n)[:, at[b]].repeat_interleave(2, 0)
        assert torch.equal(o[r], want), r
    # a sum of `dim` equal terms, three roundings of the factor, the reference's, its part's and the last steps': 2^-23 each
    assert ((lse.double() - top / LOG2E).abs() <= (dim + 16) * 2.0 ** -23 * abs(top)).all()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lens,new", FORMS)
@pytest.mark.parametrize("top", LARGE)
def test_large_scores_that_are_all_the_same(top, lens, new, dtype, table_room):
    """Equal scores and equal exponents: the row is the mean of the values that it sees."""
    dim = 64
    c = table_room(pc.batch(lens, new, 4, 2, dim, 32, 32, dtype, seed=4))
    c["q"][:] = 1.0 if top > 0 else -1.0
    fill(c, lambda b, p: 1.0)
    g = torch.Generator().manual_seed(1)
    codes = (torch.randn(c["v"].shape, generator=g) * 100).clamp(-448, 448).masked_fill(~c["used"][:, None, :, None], math.nan)
    c["v"] = codes.to(F8)
    pc.bits(c["vs"])[:] = 119  # 2^-8
    out, _ = run(c, scale=abs(top) / (dim * LOG2E))
    o = out.double().reshape(c["rows"], 4, dim)
    u = torch.finfo(dtype).eps / 2
    for r, b, n in visible(c):
        v = gathered(c, c["v"], c["vs"], b, n).repeat_interleave(2, 0)
        want, size = v.mean(1), v.abs().mean(1)
        # one rounding of the result (at least fp16's smallest), the same weight at each position up to ex2's 2^-22 in
        # the sum of exponentials, n roundings of the sums and some at their joins
        assert ((o[r] - want).abs() <= u * want.abs() + 2.0 ** -25 + (n + 24) * 2.0 ** -23 * size).all(), r


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lens,new", FORMS)
@pytest.mark.parametrize("base", [2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, -2.0 ** 24])
def test_large_scores_that_rise_by_a_few_units(base, lens, new, dtype, table_room):
    """Scores of `base` that rise by 7 or 8 from one piece of 128 positions to the next, which a reference may lag
    behind: whatever the roundings, a row stays within the values that it sees."""
    dim = 64
    c = table_room(pc.batch(lens, new, 4, 2, dim, 32, 16, dtype, seed=5))
    half = abs(base) / 512  # two dims of keys of 256
    c["q"][:] = 0.0
    q = c["q"].view(c["rows"], 4, dim)
    parts = max(1, int(half // 2 ** 15))  # f16 queries hold 2^15
    q[:, :, :2 * parts] = math.copysign(half / parts, base)
    q[:, :, 60:] = 1.0
    k = torch.zeros(c["k"].shape)
    for b, n in enumerate(lens):
        for p in range(n):
            spot = k[c["table"][b, p // 32], :, p % 32]
            spot[:, :2 * parts] = 256.0
            rise = p // 128 * (7 + b)
            for d in range(60, 64):  # as the sum of four: codes have four bits, and a step of 2^-1 at most here
                step = min(rise, 15)
                spot[:, d], rise = step, rise - step
    c["k"], c["ks"] = pc.quantise(k, c["used"], 16)
    out, lse = run(c, scale=math.log(2))
    o = out.double().reshape(c["rows"], 4, dim)
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    for r, b, n in visible(c):
        v = gathered(c, c["v"], c["vs"], b, n).repeat_interleave(2, 0)
        slack = (torch.finfo(dtype).eps / 2 + 2.0 ** -10 + (n + 24) * 2.0 ** -23) * v.abs().amax(1)
        assert (o[r] <= v.amax(1) + slack).all() and (o[r] >= v.amin(1) - slack).all(), r


@pytest.mark.parametrize("lens,new", FORMS)
def test_a_small_factor_over_large_products(lens, new, table_room):
    """Products of 2^126, blocks of keys of 2^-60 and a scale of 1e-25: scores of 2^-16, so all positions count alike."""
    dim = 64
    c = table_room(pc.batch(lens, new, 4, 2, dim, 32, 16, BF, seed=6))
    c["q"][:] = 0.0
    c["q"].view(c["rows"], 4, dim)[:, :, 3] = 2.0 ** 118
    k = torch.zeros(c["k"].shape)
    k[..., 3] = torch.where(torch.rand(k.shape[:3], generator=torch.Generator().manual_seed(2)) < 0.5, 256.0, -256.0)
    k = k.masked_fill(~c["used"][:, None, :, None], math.nan)
    c["k"] = k.to(F8)
    pc.bits(c["ks"])[:] = 67
    out, lse = run(c, scale=1e-25)
    o = out.double().reshape(c["rows"], 4, dim)
    for r, b, n in visible(c):
        v = gathered(c, c["v"], c["vs"], b, n).repeat_interleave(2, 0)
        want, size = v.mean(1), v.abs().mean(1)
        # weights: 2^-15 for the scores, a factor of fp32's smallest step (2^-149 2^126), half a step of fp16 and the sums'
        tol = torch.finfo(BF).eps / 2 * want.abs() + (2.0 ** -14 + 2.0 ** -21 + 2.0 ** -11 + (n + 24) * 2.0 ** -23) * size
        assert ((o[r] - want).abs() <= tol).all(), r
        assert ((lse[r].double() - math.log(n)).abs() <= 2.0 ** -14 + (n + 24) * 2.0 ** -22).all(), r


def test_many_small_terms_beside_a_large_value():
    """One position whose values are 2^120 times the others', and 40000 others that hold 2^-21.5 of its probability each:
    together they are 1.3 % of the sum of exponentials, though each weight times 2^exponent is 2^-141.5 of the largest."""
    dim, page, length, batch = 64, 1024, 40000, 592
    pages = -(-length // page)
    k = torch.zeros(pages, 1, page, dim)
    k[..., 0], k[..., 1] = -20.0, -1.5
    k[0, :, 7] = 0.0
    k, ks = pc.quantise(k, torch.ones(pages, page, dtype=torch.bool), 128)
    v = torch.full((pages, 1, page, dim), 1.0)
    v[0, :, 7] = torch.arange(dim) % 8 + 8.0  # exact in four bits
    vs = torch.full((pages, 1, page // 128), 67, dtype=torch.uint8)
    vs[0, 0, 0] = 187
    q = torch.zeros(batch, dim, dtype=BF)
    q[:, :2] = 1.0
    table = torch.arange(pages, dtype=torch.int32).expand(batch, pages).contiguous()  # pages that all of them read
    lens = torch.full((batch,), length, dtype=torch.int32)
    lse = torch.empty(batch, 1, device=DEV)
    d = [t.to(DEV) for t in (q, pc.bits(k), pc.bits(v.to(F8)), pc.bits(ks), vs, table, lens)]
    out = _api().paged_attention_fp8(d[0], d[1].view(F8), d[2].view(F8), d[3].view(E8), d[4].view(E8), *d[5:], scale=math.log(2),
                                     lse=lse)
    torch.cuda.synchronize()
    # the other positions of the first block share its exponent, their values are small beside its own
    total = 1 + (length - 1) * 2.0 ** -21.5
    near = 127 * 2.0 ** -21.5
    want = (v[0, 0, 7].double() + near) / total * 2.0 ** 60
    # scores: (dim + 9) 2^-23 of 21.5; sums of n terms of like size, the largest aside
    score = (dim + 9) * 2.0 ** -23 * 22.5 * math.log(2)
    slack = score + (length + 8) * 2.0 ** -23 * (total - 1) + 2.0 ** -20
    assert ((lse.double().cpu() - math.log(total)).abs() <= slack).all()
    # one rounding of the result, the weights' in fp16 (here a power of two: none for the largest)
    assert ((out.double().cpu() - want).abs() <= want * (torch.finfo(BF).eps / 2 + 2.0 ** -11 + 2 * slack)).all()


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("block", [16, 64])
def test_a_rejected_draft_leaves_its_blocks_scale(block, ragged):
    """A drafted token with large entries is taken back: its block keeps the scale that it needed, older and later codes
    are those of that scale, until the block is written from its first position again."""
    hkv, dim, page = 2, 64, 64
    g = torch.Generator().manual_seed(block + ragged)
    x = torch.randn(14, 3 * hkv, dim, generator=g)
    x[6] *= 3000.0  # the draft
    x = x.to(BF)
    k, v = (torch.full((2, hkv, page, dim), 0x7F, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
    ks, vs = (torch.full((2, hkv, page // block), 255, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2))
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    one, zero = torch.ones(128, dim, device=DEV), torch.zeros(128, dim, device=DEV)

    def add(rows, at):
        for r in [rows] if ragged else [[i] for i in rows]:
            lens.fill_(at + len(r))
            at += len(r)
            starts = torch.tensor([0, len(r)], dtype=torch.int32, device=DEV) if ragged else None
            _api().paged_append_fp8(x[r].reshape(len(r), -1).to(DEV), one, zero, k, v, ks, vs, table, lens, q_starts=starts)

    def check(rows, seen):
        """Rows in the cache, after a scale that the rows `seen` needed."""
        starts = torch.tensor([0, len(rows)], dtype=torch.int32, device=DEV)
        back = _api().paged_read_fp8(k, v, ks, vs, table, lens, q_starts=starts, rows=len(rows), dtype=torch.float32)
        for got, want, scales in ((back[0], x[:, hkv:2 * hkv], ks), (back[1], x[:, 2 * hkv:], vs)):
            e = torch.tensor([o8.exponent(float(t)) for t in want[seen].double().abs().amax((0, 2))])
            assert torch.equal(o8.scales_of(scales.cpu())[1, :, 0].long(), e)
            # half a step of four significant bits, then, where the code became subnormal, half of 2^(e - 9) at each
            # rescaling, which at least doubles it: 2^(e - 9) in all
            tol = want[rows].double().abs() * 2.0 ** -4 + torch.exp2(e.double() - 9)[:, None]
            assert ((got.cpu().double() - want[rows].double()).abs() <= tol).all()

    add([0, 1, 2, 3, 4, 5, 6], 0)
    check([0, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5, 6])
    lens.fill_(6)
    check([0, 1, 2, 3, 4, 5], [6])
    add([7, 8], 6)
    check([0, 1, 2, 3, 4, 5, 7, 8], [6])
    add([9, 10, 11, 12, 13], 0)  # the stream begins anew
    check([9, 10, 11, 12, 13], [9, 10, 11, 12, 13])


@pytest.mark.parametrize("lens,new", FORMS + [([130] * 120, [60] * 120)])  # (many tiles: thread blocks have them whole)
@pytest.mark.parametrize("top", [3.0, 1e9])
def test_outputs_where_the_queries_are(top, lens, new, table_room):
    c = table_room(pc.batch(lens, new, 4, 2, 64, 32, 16, BF, seed=3, levels=2))
    c["q"][:] = 1.0
    fill(c, lambda b, p: 1.75 if p == 5 else 0.5)
    scale = top / (1.75 * 64 * LOG2E)
    out, _ = run(c, scale=scale)
    d = pc.to({k: c[k] for k in ("q", "k", "v", "ks", "vs", "table", "lens")}, DEV)
    starts = None if c["starts"] is None else c["starts"].to(DEV)
    assert _api().paged_attention_fp8(d["q"], *where(d), q_starts=starts, scale=scale, out=d["q"]) is d["q"]
    torch.cuda.synchronize()
    assert torch.equal(d["q"].cpu(), out)


def test_large_scores_over_a_long_cache():
    """Tiles of 190 thousand positions whose rows all have large scores take longer than other waits may: they are answered."""
    from breeze_b200 import _lib

    hkv, dim, page, new, length = 8, 128, 1024, 4800, 190000
    pages = -(-length // page)
    k = torch.full((pages, hkv, page, dim), 0.5, device=DEV)
    k[0, :, 5] = 1.75
    g = torch.Generator(device=DEV).manual_seed(3)
    v = torch.randint(0, 256, k.shape, generator=g, device=DEV, dtype=torch.uint8)
    v[(v & 0x7F) == 0x7F] = 0
    ks, vs = (torch.full((pages, hkv, page // 128), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    q = torch.ones(new, hkv * dim, dtype=BF, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([length], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, new], dtype=torch.int32, device=DEV)
    out = _api().paged_attention_fp8(q, k.to(F8), v.view(F8), ks.view(E8), vs.view(E8), table, lens, q_starts=starts,
                                     scale=1e9 / (1.75 * dim * LOG2E))
    torch.cuda.synchronize()
    assert _lib.device_status(0) == 0
    want = v.view(F8)[0, :, 5].float().to(BF).reshape(-1)
    assert torch.equal(out, want.expand(new, -1))
