"""DecodeStack over a paged cache held in 8 bits."""

import pytest
import torch

from breeze_b200.fused import stack as S
from oracle import paged as op
from oracle import paged8 as o8
from tests.paged_fp8_cases import E8, F8, bits

BF = torch.bfloat16


def _small(device, n_layers=2, seed=0):
    return S.synthetic_stack("int8", n_layers, device, seed=seed, hidden=256, qkv=768, inter=512, head=384)


def test_shapes_and_counts_cpu():
    layers, head, ln_f = _small("cpu")
    kw = dict(rows=3, attention=True, kv_len=128, page_size=32, kv_dtype=F8)
    st = S.DecodeStack(layers, head, ln_f, **kw)
    assert st.launches == 7 * 2 + 1
    assert st.k_pages[0].shape == (12, 2, 32, 128) and st.k_pages[0].dtype == F8
    assert st.v_scales[1].shape == (12, 2, 1) and st.v_scales[1].dtype == E8 and (st.v_scales[1].float() == 1).all()
    assert st.kv_bytes == 2 * 2 * 2 * (3 * 128 * 128 + 3 * 128 // 32)
    st = S.DecodeStack(layers, head, ln_f, **kw, kv_block=16, prefix_len=64)
    assert st.k_scales[0].shape == (8, 2, 2) and st.launches == 7 * 2 + 1
    assert st.kv_bytes == 2 * 2 * 2 * ((64 + 3 * 64) * 128 + (64 + 3 * 64) // 16)
    st = S.DecodeStack(layers, head, ln_f, rows=3, attention=True, kv_len=128, page_size=32, kv_dtype=BF)
    assert st.k_pages[0].dtype == BF and st.kv_block is None


def test_refusals_cpu():
    layers, head, ln_f = _small("cpu")
    for kw in (dict(kv_dtype=F8), dict(page_size=32, kv_dtype=torch.float16), dict(page_size=32, kv_block=32),
               dict(page_size=32, kv_dtype=F8, kv_block=64), dict(page_size=32, kv_dtype=F8, kv_block=8),
               dict(page_size=64, kv_dtype=F8, kv_block=48)):
        with pytest.raises(ValueError):
            S.DecodeStack(layers, head, ln_f, rows=3, attention=True, kv_len=128, **kw)


def _pages(st, li=-1):
    return [t.cpu() for t in (st.k_pages[li], st.v_pages[li], st.k_scales[li], st.v_scales[li])]


def _check_last_layer(st, table, lens, before):
    """The last layer's append and attention against the oracle, on the qkv and caches they read."""
    hkv, dim, hq, block, page = st.hkv, st.head_dim, st.hq, st.kv_block, st.page_size
    l = st.layers[-1]
    live = [r for r, n in enumerate(lens) if n > 0]
    fake = torch.zeros(before[0].shape[0], hkv, page, dim)
    q, written, terms = op.append(st.qkv.cpu(), st.cos.cpu(), st.sin.cpu(), fake, fake, table, lens, None, l.q_norm.cpu(),
                                  l.k_norm.cpu(), st.eps)
    u, slack = torch.finfo(BF).eps / 2, (dim / 2 + 8) * 2.0 ** -24
    got = st.q.cpu().double().reshape(st.rows, hq, dim)
    # one rounding of the result, under (dim / 2 + 8) fp32 roundings before it
    assert ((got[live] - q[live]).abs() <= u * q[live].abs() + slack * terms[live, :hq]).all()
    after = _pages(st)
    values = [o8.values(after[i], after[2 + i]) for i in (0, 1)]
    for (pg, slot), (t, *kv) in written.items():
        for i in (0, 1):
            e = o8.scales_of(after[2 + i])[pg, :, slot // block].double()[:, None]
            err = slack * terms[t, hq:] if i == 0 else 0.0
            assert (kv[i].abs() <= 448 * torch.exp2(e) + err).all()
            # half a step of four significant bits, or of the subnormal codes'
            tol = torch.maximum(kv[i].abs() * 2.0 ** -4, torch.exp2(e - 10))
            assert ((values[i][pg, :, slot] - kv[i]).abs() <= tol + err).all()
    # k and v as a block's older positions had them, but for codes that became subnormal
    for i in (0, 1):
        old = o8.values(before[i], before[2 + i])
        for t, n in enumerate(lens):
            for p in range(max(0, n - 1)):
                pg, slot = table[t][p // page], p % page
                e = o8.scales_of(after[2 + i])[pg, :, slot // block].double()[:, None]
                assert ((values[i][pg, :, slot] - old[pg, :, slot]).abs() <= torch.exp2(e - 10)).all()
    ref = o8.attention(st.q.cpu(), (after[0], after[1]), (after[2], after[3]), table, lens, None)
    tol, _ = o8.attention_bounds(ref, dim, BF)
    out = st.attn_out.cpu().double().reshape(st.rows, hq, dim)
    assert ((out - ref["out"]).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 64])
def test_uneven_streams_follow_the_oracle_as_they_grow(prefix):
    """Eager steps, then a captured one replayed, with lengths (one row unused)
    and caches advancing; the graph's logits are the eager step's bits."""
    g = torch.Generator().manual_seed(3)
    layers, head, ln_f = _small("cuda")
    rows = 5
    st = S.DecodeStack(layers, head, ln_f, rows=rows, attention=True, kv_len=256, page_size=32, prefix_len=prefix, kv_dtype=F8,
                       kv_block=16)
    ang = torch.arange(256)[:, None] * 1e4 ** (-torch.arange(0, 128, 2) / 128)
    st.cos.copy_(torch.cat([ang, ang], 1).cos())
    st.sin.copy_(torch.cat([ang, ang], 1).sin())
    for t in st.k_pages + st.v_pages:
        bits(t).copy_(bits((torch.randn(t.shape, generator=g) * 64).clamp(-448, 448).to(F8)))
    for t in st.k_scales + st.v_scales:
        bits(t).copy_(torch.randint(119, 122, t.shape, generator=g))
    if not prefix:  # any pages will do
        st.page_table.copy_(torch.randperm(st.page_table.numel(), generator=g).reshape(st.page_table.shape))
    table = st.page_table.tolist()
    lens = [70, 200, 0, 129, 256 - 8]
    st.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    for step in range(6):
        if step == 3:
            st.capture()
        st.x.copy_(torch.randn(rows, 256, generator=g))
        before = _pages(st)
        st.run() if step < 3 else st.replay()
        torch.cuda.synchronize()
        _check_last_layer(st, table, lens, before)
        if step >= 3:
            logits = st.logits.clone()
            st.run()  # the same step again: it rewrites the same slots
            torch.cuda.synchronize()
            assert torch.equal(logits, st.logits)
        lens = [n + 1 if n else 0 for n in lens]
        st.seq_lens += (st.seq_lens > 0).int()
    from breeze_b200 import _lib

    assert _lib.device_status(0) == 0


@pytest.mark.gpu
def test_a_prompt_moves_from_a_16_bit_cache_and_back():
    """Rows of a 16-bit stack's cache written into an 8-bit one by an append without norm and rotation, read back, and
    written into another 16-bit cache: half a step of four significant bits of each value, or of its block's largest."""
    from breeze_b200.fused import paged, paged_fp8

    g = torch.Generator().manual_seed(5)
    hkv, dim, page, n = 2, 128, 32, 77
    k, v = (torch.randn(n, hkv, dim, generator=g).to(BF) for _ in range(2))
    table, lens = torch.tensor([[3, 1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    kp, vp = (torch.zeros(4, hkv, page, dim, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2))
    ks, vs = (torch.zeros(4, hkv, 2, dtype=torch.uint8, device="cuda").view(E8) for _ in range(2))
    one, zero = torch.ones(n, dim, device="cuda"), torch.zeros(n, dim, device="cuda")
    qkv = torch.cat([k, k, v], 1).reshape(n, -1).cuda()
    paged_fp8.paged_append_fp8(qkv, one, zero, kp, vp, ks, vs, table, lens, q_starts=starts)
    kk, vv = paged_fp8.paged_read_fp8(kp, vp, ks, vs, table, lens, q_starts=starts, rows=n)
    k16, v16 = (torch.zeros(4, hkv, page, dim, dtype=BF, device="cuda") for _ in range(2))
    paged.paged_append(torch.cat([kk, kk, vv], 1).reshape(n, -1), one, zero, k16, v16, table, lens, q_starts=starts)
    torch.cuda.synchronize()
    for want, got in ((k, k16), (v, v16)):
        x = op.gather(got.cpu(), table[0].tolist(), n).transpose(0, 1)
        top = torch.stack([want.double()[p - p % 16:p - p % 16 + 16].abs().amax((0, 2)) for p in range(n)])[..., None]
        # subnormal codes: half of 2^-9 of a scale that is at most 1 / 224 of the block's largest
        assert ((x - want.double()).abs() <= torch.maximum(want.double().abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)).all()
