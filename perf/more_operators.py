"""The operators of a paged KV cache held in 8 bits and what they cost: cases, plain forms and exact values.

Three operators of serving with such a cache, as breeze_b200.fused.paged_fp8 offers them:

  append   paged_append_fp8: new tokens' q / k / v rows -> per-head RMSNorm, rotary
           positions, k and v quantised block by block into their pages, q returned
  attend   paged_attention_fp8: softmax(q k^T) v over the caches of a ragged batch
  read     paged_read_fp8: the last positions of each sequence back as 16-bit rows

Layout: k_pages / v_pages (pages, kv heads, page size, head dim) e4m3 codes;
k_scales / v_scales (pages, kv heads, page size / block) e8m0, a power of two for
each block of positions and head; page_table (batch, pages of the longest sequence)
int32, -1 where a sequence has no page; seq_lens (batch) int32, the new tokens
included. The rows of sequence b are rows q_starts[b] .. q_starts[b + 1], its last
positions; without q_starts every sequence has one.

A block's scale is 2^e with the least e from -60 to 60 for which its largest
magnitude is at most 448 2^e. Where tokens are added behind others of the same block,
e does not shrink, and where it grows the codes there are divided by the power of two.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed():
    base = dict(dtype="bf16", heads=16, kv_heads=16, dim=128, page=64, block=64, batch=1, lo=1, hi=1, new=1)
    return [
        # one CFG pair (cond, uncond) of a stream: the decode step's append, where latency counts
        dict(base, name="append_pair", op="append", batch=2, lo=200, hi=600),
        # a busy server's decode step: one new token in each of 160 streams of uneven length
        dict(base, name="append_decode_160", op="append", heads=32, kv_heads=8, block=32, batch=160, lo=25, hi=5000),
        # prompts of seven streams written in one go (half precision, small heads, ragged, short blocks)
        dict(base, name="append_prompts_f16", op="append", dtype="f16", heads=20, kv_heads=4, dim=64, page=32, block=16,
             batch=7, lo=700, hi=4400, new=1900),
        # one CFG pair's decode step over a prompt and some audio frames: latency
        dict(base, name="attend_pair", op="attend", batch=2, lo=250, hi=650),
        # decode step of a mixed batch, lengths from a few tokens to some thousands
        dict(base, name="attend_decode_64", op="attend", heads=32, kv_heads=8, block=32, batch=64, lo=11, hi=7000),
        # long contexts: six streams of about 50 thousand tokens
        dict(base, name="attend_long_6", op="attend", heads=32, kv_heads=8, page=128, block=128, batch=6, lo=40000, hi=60000),
        # multi-token verify: up to six drafted tokens per stream, small heads, half precision, short pages
        dict(base, name="attend_verify_f16", op="attend", dtype="f16", heads=15, kv_heads=3, dim=64, page=16, block=16,
             batch=29, lo=60, hi=2900, new=6),
        # a chunk of prompts beside running streams: ragged new tokens, causal
        dict(base, name="attend_chunk_mixed", op="attend", heads=32, kv_heads=8, batch=7, lo=900, hi=5200, new=1100),
        # one long prompt in a single call
        dict(base, name="attend_prompt_6500", op="attend", kv_heads=8, lo=6500, hi=6500, new=6500),
        # one stream's prompt copied out of the cache
        dict(base, name="read_prompt", op="read", lo=410, hi=410, new=410),
        # the whole caches of 24 streams copied out, to move them to a 16-bit cache
        dict(base, name="read_streams_24", op="read", heads=32, kv_heads=8, page=128, block=32, batch=24, lo=900, hi=9000,
             new=9000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "read"])
    dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    if kv * group > 48:
        group = 2
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    batch = _log_int(rng, 1, 16 if kind == "prompt" else 200)
    new = 1 if kind == "decode" else rng.randint(2, 8) if kind == "verify" else _log_int(rng, 9, 4000)
    # cache rows of the batch are bounded, so that a case costs no more than the largest listed one
    hi = _log_int(rng, 1, max(2, min(50000, (200000 if kind != "prompt" else 40000) // batch)))
    hi = max(hi, new)
    if kind == "prompt" and op == "attend":  # score entries of the padded batch, too
        new = min(new, max(2, 500_000_000 // (hi * kv * group * batch)))
    lo = max(new, int(hi * rng.choice([0.05, 0.5, 1.0])))
    return dict(op=op, dtype=rng.choice(["bf16", "f16"]), heads=kv * group, kv_heads=kv, dim=dim, page=page, block=block,
                batch=batch, lo=min(lo, hi), hi=hi, new=new)


def lengths(case):
    """Cache lengths (new tokens included) and rows of every sequence: the longest first."""
    rng = random.Random("lengths %d %d %d %d" % (case["batch"], case["lo"], case["hi"], case["new"]))
    lens = [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]
    if case["new"] == 1:
        return lens, [1] * len(lens)
    if case["op"] == "read" and case["new"] == case["hi"]:
        return lens, lens  # all there is
    new = [case["new"]] + [_log_int(rng, 1, case["new"]) for _ in lens[1:]]
    return lens, [min(n, length) for n, length in zip(new, lens)]


def _power(e):
    """2^e in fp32, exactly, for whole e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponent(top):
    """Least e from -60 to 60 with top <= 448 2^e: top = m 2^x with m from 1/2 to 1, and 448 is 7/8 of 2^9."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 9 + (m > 0.875).int(), -60).clamp(-60, 60)


def _codes(x):
    """e4m3 codes of values that are scaled already; what is infinite is NaN."""
    return torch.where(x.isfinite(), x.clamp(-448, 448), math.nan).to(F8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = DTYPES[case["dtype"]], "cuda"
    heads, kv, dim, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    lens, new = lengths(case)
    order = torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed)).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    cols = -(-max(lens) // page)
    need = torch.tensor([-(-n // page) for n in lens], device=dev)
    pages = int(need.sum()) + 3  # three pages nobody uses
    ids = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    taken = torch.arange(cols, device=dev) < need[:, None]
    table = torch.full((len(lens), cols), -1, dtype=torch.int32, device=dev)
    table[taken] = ids[:pages - 3]
    rows = sum(new)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    def cache():
        """Normal values, some channels of a head several times the others, a level of its own for each block."""
        channel = torch.exp2(1.5 * torch.randn(kv, 1, 1, dim, generator=g, device=dev).clamp(min=0))
        level = torch.exp2(0.5 * torch.randn(pages, kv, page // block, 1, 1, generator=g, device=dev))
        x = normal(pages, kv, page // block, block, dim)
        e = _exponent((x.abs().float() * channel).amax((3, 4)) * level[..., 0, 0])
        codes = _codes(x * (channel * level * _power(-e)[..., None, None])).view(pages, kv, page, dim)
        return codes, (e + 127).to(torch.uint8).view(E8)

    state = dict(case=case, max_q=max(new), page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                 q_starts=None, rows=rows)
    state["k_pages"], state["k_scales"] = cache()
    state["v_pages"], state["v_scales"] = cache()
    if case["new"] > 1:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if case["op"] == "append":
        state["qkv"] = normal(rows, (heads + 2 * kv) * dim)
        state["q_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=dev)).to(dt)
        state["k_norm"] = torch.exp2(1.5 * torch.randn(dim, generator=g, device=dev).clamp(min=0)).to(dt)
        freq = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
        ang = torch.arange(max(lens), dtype=torch.float64, device=dev)[:, None] * freq
        ang = torch.cat([ang, ang], -1)
        state["cos"], state["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    elif case["op"] == "attend":
        state["q"] = normal(rows, heads * dim) * 0.75  # keys of a few units: scores of a few units
    return state


def _rows(state):
    """Sequence and index within its rows of every row, rows of every sequence."""
    rows = state["rows"]
    if state["q_starts"] is None:
        seq = torch.arange(rows, device="cuda")
        return seq, torch.zeros_like(seq), torch.ones_like(state["seq_lens"])
    starts = state["q_starts"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, row - starts[seq], (starts[1:] - starts[:-1]).int()


def _store(pages, scales, x, page, pos, page0, pos0):
    """x (rows, kv heads, dim) into position pos of page `page`; sequence b's first row goes to pos0[b] of page0[b]."""
    size, per = pages.shape[2], scales.shape[2]
    block = size // per
    held, exps = pages.view(torch.uint8), scales.view(torch.uint8)
    slot, slot0 = pos % size, pos0 % size
    # largest finite magnitude of the new tokens of every block
    mag = torch.where(x.isfinite(), x, 0).abs().amax(-1)
    top = torch.zeros(pages.shape[0] * per, x.shape[1], device=x.device)
    top.index_reduce_(0, page * per + slot // block, mag, "amax")
    e = _exponent(top).view(-1, per, x.shape[1])
    # blocks that hold older tokens: their scale does not shrink, and their codes follow it
    kept = slot0 % block
    was, need = exps[page0, :, slot0 // block].int() - 127, e[page0, slot0 // block]
    now = torch.where(kept[:, None] > 0, torch.maximum(was, need), need)
    e[page0, slot0 // block] = now
    at = (slot0 - kept)[:, None] + torch.arange(block, device=x.device)
    old = held[page0[:, None], :, at]
    moved = _codes(old.view(F8).float() * _power(was - now)[:, None, :, None]).view(torch.uint8)
    held[page0[:, None], :, at] = torch.where((at < slot0[:, None])[..., None, None], moved, old)
    mine = e[page, slot // block]
    held[page, :, slot] = _codes(x * _power(-mine)[..., None]).view(torch.uint8)
    exps[page, :, slot // block] = (mine + 127).to(torch.uint8)


def _plain_append(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    qkv, table = state["qkv"], state["page_table"]
    rows = qkv.shape[0]
    seq, index, count = _rows(state)
    pos0 = (state["seq_lens"] - count).long()
    pos = pos0[seq] + index
    x = qkv.view(rows, heads + 2 * kv, dim)
    f = x[:, :heads + kv].float()
    gain = torch.cat([state["q_norm"].float().expand(heads, dim), state["k_norm"].float().expand(kv, dim)])
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * gain
    turned = torch.cat([-f[..., dim // 2:], f[..., :dim // 2]], -1)
    f = f * state["cos"][pos].float()[:, None] + turned * state["sin"][pos].float()[:, None]
    where = (table[seq, pos // page].long(), pos, table.gather(1, (pos0 // page)[:, None])[:, 0].long(), pos0)
    _store(state["k_pages"], state["k_scales"], f[:, heads:], *where)
    _store(state["v_pages"], state["v_scales"], x[:, heads + kv:].float(), *where)
    return (f[:, :heads].to(qkv.dtype).reshape(rows, heads * dim), state["k_pages"], state["k_scales"], state["v_pages"],
            state["v_scales"])


def _plain_attention(state):
    case = state["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    q, table, lens, longest = state["q"], state["page_table"], state["seq_lens"], state["max_q"]
    rows, batch, group = q.shape[0], table.shape[0], heads // kv
    seq, index, count = _rows(state)
    which = table.clamp(min=0).long()

    def gathered(pages, scales):
        x = pages.view(torch.uint8)[which].view(F8).float()  # batch, column, kv, slot, dim
        s = scales.view(torch.uint8)[which].view(E8).float()
        x = (x.view(*s.shape, -1, dim) * s[..., None, None]).view(x.shape)
        return x.transpose(1, 2).reshape(batch, kv, -1, dim)

    k, v = gathered(state["k_pages"], state["k_scales"]), gathered(state["v_pages"], state["v_scales"])
    padded = torch.zeros(batch, longest, heads, dim, device=q.device)
    padded[seq, index] = q.view(rows, heads, dim).float() * dim ** -0.5
    padded = padded.view(batch, longest, kv, group, dim).transpose(1, 2).reshape(batch, kv, longest * group, dim)
    score = (padded @ k.transpose(2, 3)).view(batch, kv, longest, group, -1)
    seen = (lens - count).long()[:, None] + torch.arange(1, longest + 1, device=q.device)
    hidden = torch.arange(k.shape[2], device=q.device) >= seen[:, :, None]
    score = score.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(batch, kv, longest * group, -1) @ v).view(batch, kv, longest, group, dim) / total
    out = out.transpose(1, 2).reshape(batch, longest, heads * dim)[seq, index].to(q.dtype)
    lse = (top + total.log()).squeeze(-1).transpose(1, 2).reshape(batch, longest, heads)[seq, index]
    return out, lse


def _plain_read(state):
    case, table = state["case"], state["page_table"]
    page, block = case["page"], case["block"]
    seq, index, count = _rows(state)
    pos = (state["seq_lens"] - count)[seq].long() + index
    where, slot = table[seq, pos // page].long(), pos % page

    def back(pages, scales):
        x = pages.view(torch.uint8)[where, :, slot].view(F8).float()
        return (x * scales.view(torch.uint8)[where, :, slot // block].view(E8).float()[..., None]).to(DTYPES[case["dtype"]])

    return back(state["k_pages"], state["k_scales"]), back(state["v_pages"], state["v_scales"])


def run(state):
    case = state["case"]
    if own:
        from breeze_b200.fused import paged_fp8

        where = (state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"], state["page_table"], state["seq_lens"])
        if case["op"] == "append":
            q = paged_fp8.paged_append_fp8(state["qkv"], state["cos"], state["sin"], *where, q_starts=state["q_starts"],
                                           q_norm_w=state["q_norm"], k_norm_w=state["k_norm"], eps=1e-6)
            return q, state["k_pages"], state["k_scales"], state["v_pages"], state["v_scales"]
        if case["op"] == "attend":
            lse = torch.empty(state["rows"], case["heads"], device="cuda")
            return paged_fp8.paged_attention_fp8(state["q"], *where, q_starts=state["q_starts"], max_q=state["max_q"], lse=lse), lse
        return paged_fp8.paged_read_fp8(*where, q_starts=state["q_starts"], rows=state["rows"], dtype=DTYPES[case["dtype"]])
    return {"append": _plain_append, "attend": _plain_attention, "read": _plain_read}[case["op"]](state)


def work(case):
    lens, new = lengths(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    rows = sum(new)
    if case["op"] == "append":
        # qkv read, q (2 bytes) and the codes (1 byte) written, one cos / sin row per token, a scale per block, lengths
        # and table entries
        blocks = sum(-(-n // case["block"]) for n in new)
        return {"bytes": rows * ((2 * heads + 2 * kv) * dim * 2 + 2 * kv * dim + 2 * dim * 2) + blocks * 2 * kv + len(lens) * 8,
                "flops": rows * (heads + 2 * kv) * dim * 8}
    if case["op"] == "read":
        blocks = sum(-(-n // case["block"]) for n in new)
        return {"bytes": rows * 2 * kv * dim * 3 + blocks * 2 * kv + len(lens) * 8, "flops": rows * 2 * kv * dim}
    blocks = sum(-(-n // case["block"]) for n in lens)
    table = sum(-(-n // case["page"]) for n in lens) * 4
    pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lens))
    return {"bytes": (sum(lens) * dim + blocks) * kv * 2 + rows * heads * (dim * 2 * 2 + 4) + table + len(lens) * 4,
            "flops": pairs * heads * dim * 4}


def _nearest(x):
    """64-bit values to the nearest e4m3 value, ties to even: steps of 2^-9 up to 2^-6, of an eighth of the power above."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    lens, table = s["seq_lens"].tolist(), s["page_table"].tolist()
    batch, group = len(lens), heads // kv
    starts = list(range(batch + 1)) if s["q_starts"] is None else s["q_starts"].tolist()
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        ks, vs = s["k_scales"].double(), s["v_scales"].double()
        qkv = s["qkv"].double().view(-1, heads + 2 * kv, dim)
        q = torch.empty(qkv.shape[0], heads, dim, dtype=torch.float64, device="cuda")
        half = dim // 2

        def blocks_of(codes, scales, x, b, first):
            """The rows x (n, kv, dim) of sequence b from position `first`, one block's part after the other: parts of
            one position in the block are done together, over all whole blocks."""
            p = first
            while p < first + x.shape[0]:
                o = p % block
                n = min(block - o, first + x.shape[0] - p)
                runs = 1 if o or n < block else (first + x.shape[0] - p) // block
                part = x[p - first:p - first + runs * n].view(runs, n, kv, dim)
                at = torch.arange(runs, device="cuda") * block + p
                pg = torch.tensor(table[b], device="cuda")[at // page]
                sl = at % page - o
                top = part.abs().amax((1, 3))
                scale = torch.exp2(torch.ceil(torch.log2(top / 448).clamp(-60, 60)))
                if o:
                    before = scales[pg, :, sl // block]
                    scale = torch.maximum(scale, before)
                    codes[pg[0], :, sl[0]:sl[0] + o] = _nearest(codes[pg[0], :, sl[0]:sl[0] + o] * (before / scale)[0, :, None, None])
                scales[pg, :, sl // block] = scale
                inside = sl[:, None] + o + torch.arange(n, device="cuda")
                codes[pg[:, None], :, inside] = _nearest((part / scale[:, None, :, None]).clamp(-448, 448))
                p += runs * n

        for b in range(batch):
            n = starts[b + 1] - starts[b]
            if n == 0:
                continue
            first = lens[b] - n
            x = qkv[starts[b]:starts[b + 1]]
            cos, sin = s["cos"][first:lens[b]].double()[:, None], s["sin"][first:lens[b]].double()[:, None]

            def turn(h, gain):
                h = h / (h.square().sum(-1, keepdim=True) / dim + 1e-6).sqrt() * gain.double()
                a, c = h[..., :half], h[..., half:]
                return torch.cat([a * cos[..., :half] - c * sin[..., :half], c * cos[..., half:] + a * sin[..., half:]], -1)

            q[starts[b]:starts[b + 1]] = turn(x[:, :heads], s["q_norm"])
            blocks_of(kp, ks, turn(x[:, heads:heads + kv], s["k_norm"]), b, first)
            blocks_of(vp, vs, x[:, heads + kv:].contiguous(), b, first)
        return q.reshape(-1, heads * dim), kp, ks, vp, vs

    def values(codes, scales, ids, length):
        """(kv, length, dim) of the pages `ids` in order, in 64 bits."""
        x = codes[ids].double().view(len(ids), kv, page // block, block, dim) * scales[ids].double()[..., None, None]
        return x.view(len(ids), kv, page, dim).transpose(0, 1).reshape(kv, -1, dim)[:, :length]

    if case["op"] == "read":
        parts = []
        for b in range(batch):
            ids = torch.tensor(table[b][:-(-lens[b] // page)], device="cuda")
            first = lens[b] - (starts[b + 1] - starts[b])
            parts.append([values(s[x + "_pages"], s[x + "_scales"], ids, lens[b])[:, first:].transpose(0, 1) for x in "kv"])
        return tuple(torch.cat(x) for x in zip(*parts))
    rows = s["q"].shape[0]
    q = s["q"].double().view(rows, kv, group, dim)
    out = torch.zeros(rows, kv, group, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(rows, kv, group, dtype=torch.float64, device="cuda")
    for b in range(batch):
        a, z, length = starts[b], starts[b + 1], lens[b]
        ids = torch.tensor(table[b][:-(-length // page)], device="cuda")
        k, v = (values(s[x + "_pages"], s[x + "_scales"], ids, length) for x in "kv")
        for r in range(a, z, 512):  # blocks of rows bound the score matrix
            e = min(r + 512, z)
            score = torch.einsum("thgd,hsd->thgs", q[r:e], k) / math.sqrt(dim)
            last = length - (z - torch.arange(r, e, device="cuda"))  # the row's own position
            score.masked_fill_((torch.arange(length, device="cuda") > last[:, None])[:, None, None], -math.inf)
            out[r:e] = torch.einsum("thgs,hsd->thgd", torch.softmax(score, -1), v)
            lse[r:e] = torch.logsumexp(score, -1)
    return out.reshape(rows, heads * dim), lse.reshape(rows, heads)
