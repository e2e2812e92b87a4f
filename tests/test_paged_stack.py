"""DecodeStack over a paged cache: streams of unequal length in one step."""

import pytest
import torch

from breeze_b200.fused import stack as S
from oracle import paged as op

BF = torch.bfloat16


def _small(device, n_layers=2, seed=0):
    return S.synthetic_stack("int8", n_layers, device, seed=seed, hidden=256, qkv=768, inter=512, head=384)


def test_shapes_and_counts_cpu():
    layers, head, ln_f = _small("cpu")
    st = S.DecodeStack(layers, head, ln_f, rows=3, attention=True, kv_len=128, page_size=32)
    assert st.launches == 7 * 2 + 1
    assert st.k_pages[0].shape == (12, 2, 32, 128) and st.page_table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]]
    assert st.kv_bytes == 2 * 2 * (3 * 128) * 2 * 128 * 2
    st = S.DecodeStack(layers, head, ln_f, rows=3, attention=True, kv_len=128, page_size=32, num_pages=5)  # a pool
    assert st.k_pages[0].shape[0] == 5 and st.page_table.tolist() == [[-1] * 4] * 3 and st.seq_lens.tolist() == [0, 0, 0]
    st = S.DecodeStack(layers, head, ln_f, rows=3, attention=True, kv_len=128, page_size=32, prefix_len=64, num_pages=11)
    assert st.launches == 8 * 2 + 1
    assert st.k_pages[0].shape[0] == 11 and st.page_table.tolist() == [[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 6, 7]]
    assert st.kv_bytes == 2 * 2 * (64 + 3 * 64) * 2 * 128 * 2
    st.seq_lens.copy_(torch.tensor([70, 0, 128]))
    assert st.kv_bytes == 2 * 2 * (64 + 6 + 64) * 2 * 128 * 2


def test_refusals_cpu():
    layers, head, ln_f = _small("cpu")
    for kw in (dict(page_size=32), dict(attention=True, prefix_len=32), dict(attention=True, page_size=32, kv_len=100),
               dict(attention=True, page_size=32, kv_len=128, prefix_len=40),
               dict(attention=True, page_size=32, kv_len=128, prefix_len=160),
               dict(attention=True, page_size=32, kv_len=128, num_pages=0),
               dict(attention=True, page_size=32, kv_len=128, prefix_len=64, num_pages=2)):
        with pytest.raises(ValueError):
            S.DecodeStack(layers, head, ln_f, rows=3, **kw)


def _check_last_layer(st, table, lens, before):
    """The last layer's append and attention against the oracle, on the qkv and caches they read."""
    hkv, dim, hq = st.hkv, st.head_dim, st.hq
    l = st.layers[-1]
    live = [r for r, n in enumerate(lens) if n > 0]
    q, written, terms = op.append(st.qkv.cpu(), st.cos.cpu(), st.sin.cpu(), *before, table, lens, None, l.q_norm.cpu(),
                                  l.k_norm.cpu(), st.eps)
    u = torch.finfo(BF).eps / 2
    got = st.q.cpu().double().reshape(st.rows, hq, dim)
    # one rounding of the result, under (dim / 2 + 8) fp32 roundings before it
    assert ((got[live] - q[live]).abs() <= u * q[live].abs() + (dim / 2 + 8) * 2.0 ** -24 * terms[live, :hq]).all()
    k, v = st.k_pages[-1].cpu(), st.v_pages[-1].cpu()
    for (page, slot), (t, kk, vv) in written.items():
        assert ((k[page, :, slot].double() - kk).abs() <= u * kk.abs() + (dim / 2 + 8) * 2.0 ** -24 * terms[t, hq:]).all()
        assert torch.equal(v[page, :, slot], vv.to(BF))
    ref = op.attention(st.q.cpu(), k, v, table, lens, None)
    tol, _ = op.attention_bounds(ref, dim, BF)
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
    st = S.DecodeStack(layers, head, ln_f, rows=rows, attention=True, kv_len=256, page_size=32, prefix_len=prefix)
    ang = torch.arange(256)[:, None] * 1e4 ** (-torch.arange(0, 128, 2) / 128)
    st.cos.copy_(torch.cat([ang, ang], 1).cos())
    st.sin.copy_(torch.cat([ang, ang], 1).sin())
    for t in st.k_pages + st.v_pages:
        t.copy_(torch.randn(t.shape, generator=g))
    if not prefix:  # any pages will do
        st.page_table.copy_(torch.randperm(st.page_table.numel(), generator=g).reshape(st.page_table.shape))
    table = st.page_table.tolist()
    lens = [70, 200, 0, 129, 256 - 8]
    st.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    for step in range(3):
        st.x.copy_(torch.randn(rows, 256, generator=g))
        before = (st.k_pages[-1].cpu(), st.v_pages[-1].cpu())
        st.run()
        torch.cuda.synchronize()
        _check_last_layer(st, table, lens, before)
        lens = [n + 1 if n else 0 for n in lens]
        st.seq_lens += (st.seq_lens > 0).int()
    st.capture()
    for step in range(3):
        st.x.copy_(torch.randn(rows, 256, generator=g))
        before = (st.k_pages[-1].cpu(), st.v_pages[-1].cpu())
        st.replay()
        torch.cuda.synchronize()
        _check_last_layer(st, table, lens, before)
        logits = st.logits.clone()
        st.run()  # the same step again: it rewrites the same slots
        torch.cuda.synchronize()
        assert torch.equal(logits, st.logits)
        lens = [n + 1 if n else 0 for n in lens]
        st.seq_lens += (st.seq_lens > 0).int()
    from breeze_b200 import _lib

    assert _lib.device_status(0) == 0


@pytest.mark.gpu
def test_even_streams_agree_with_the_static_cache():
    """All rows at one position: the paged stack and the static-cache stack of
    the same weights, logits within 1e-2 of the largest (the paged step rounds
    the rotated q to bf16, the static one keeps it in fp32)."""
    layers, head, ln_f = _small("cuda")
    dense = S.DecodeStack(layers, head, ln_f, rows=4, attention=True, kv_len=128)
    pg = S.DecodeStack(layers, head, ln_f, rows=4, attention=True, kv_len=128, page_size=64)
    g = torch.Generator().manual_seed(5)
    for i in range(2):
        for c, p in ((dense.k_cache[i], pg.k_pages[i]), (dense.v_cache[i], pg.v_pages[i])):
            c.copy_(torch.randn(c.shape, generator=g))
            p.copy_(c.reshape(4, 2, 2, 64, 128).transpose(1, 2).reshape(8, 2, 64, 128))
    x = torch.randn(4, 256, generator=g).to(BF)
    dense.pos.fill_(90)
    pg.seq_lens.fill_(91)
    dense.x.copy_(x)
    pg.x.copy_(x)
    a, b = dense.run().clone(), pg.run().clone()
    torch.cuda.synchronize()
    assert (a - b).abs().max() <= 1e-2 * a.abs().max()
