"""The paged-cache operators and what they cost: cases, plain forms and exact values.

Three operators of serving with a paged KV cache, as breeze_b200.fused.paged offers them:

  append   paged_append: new tokens' q / k / v rows -> per-head RMSNorm, rotary
           positions, k and v written into their pages, q returned
  paged    paged_attention: softmax(q k^T) v over the paged caches of a ragged batch
  prefix   prefix_attention: the same for a batch whose sequences begin with the
           same pages, which are read once for the whole batch

Layout: k_pages / v_pages (pages, kv heads, page size, head dim); page_table
(batch, pages of the longest sequence) int32, -1 where a sequence has no page;
seq_lens (batch) int32, the new tokens included. The new tokens of sequence b
are rows q_starts[b] .. q_starts[b + 1] of q; without q_starts every sequence
has one new token.
"""

import math
import random
import sys
from pathlib import Path

import torch

# where the package lives in this repository
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "breeze-tts-2_b200"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    base = dict(dtype="bf16", heads=16, kv_heads=16, dim=128, page=64, batch=1, lo=1, hi=1, new=1, prefix=0)
    return [
        # one CFG pair (cond, uncond) of a stream: the decode step's append, where latency counts
        dict(base, name="append_pair", op="append", batch=2, lo=300, hi=700),
        # a busy server's decode step: one new token in each of 200 streams of uneven length
        dict(base, name="append_decode_200", op="append", heads=32, kv_heads=8, batch=200, lo=30, hi=4000),
        # prompts of six streams written in one go (half precision, small heads, ragged)
        dict(base, name="append_prompts_f16", op="append", dtype="f16", heads=24, kv_heads=8, dim=64, page=16, batch=6,
             lo=900, hi=5000, new=2100),
        # one CFG pair's decode step over a prompt and some audio frames: latency
        dict(base, name="paged_pair", op="paged", batch=2, lo=300, hi=700),
        # decode step of a mixed batch, lengths from a few tokens to some thousands
        dict(base, name="paged_decode_48", op="paged", heads=32, kv_heads=8, batch=48, lo=17, hi=6000),
        # long contexts: eight streams of about 30 thousand tokens
        dict(base, name="paged_long_8", op="paged", heads=32, kv_heads=8, batch=8, lo=24000, hi=32000, page=128),
        # multi-token verify: up to five drafted tokens per stream, small heads, half precision, short pages
        dict(base, name="paged_verify_f16", op="paged", dtype="f16", heads=12, kv_heads=4, dim=64, page=16, batch=33,
             lo=40, hi=3100, new=5),
        # a chunk of prompts beside running streams: ragged new tokens, causal
        dict(base, name="paged_chunk_mixed", op="paged", heads=32, kv_heads=8, batch=9, lo=700, hi=4500, new=1300),
        # one long prompt in a single call
        dict(base, name="paged_prompt_7000", op="paged", heads=16, kv_heads=8, batch=1, lo=7000, hi=7000, new=7000),
        # four streams that share a short voice prompt
        dict(base, name="prefix_4", op="prefix", batch=4, lo=520, hi=800, prefix=512),
        # many streams behind one long system and voice prompt
        dict(base, name="prefix_96_long", op="prefix", heads=32, kv_heads=8, batch=96, lo=12300, hi=12900, prefix=12288),
        # drafted tokens of streams that share a prompt (half precision, odd head count)
        dict(base, name="prefix_verify_f16", op="prefix", dtype="f16", heads=20, kv_heads=4, dim=64, page=32, batch=24,
             lo=2100, hi=2700, new=4, prefix=2048),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "prefix"])
    dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    if kv * group > 48:
        group = 2
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    batch = _log_int(rng, 1, 16 if kind == "prompt" else 200)
    new = 1 if kind == "decode" else rng.randint(2, 8) if kind == "verify" else _log_int(rng, 9, 4000)
    # cache rows of the batch are bounded, so that a case costs no more than the largest listed one
    hi = _log_int(rng, 1, max(2, min(32000, (200000 if kind != "prompt" else 40000) // batch)))
    prefix = 0
    if op == "prefix":
        prefix = page * _log_int(rng, 1, max(1, 12288 // page))
        hi = prefix + new + min(hi, 2000)
        if kind == "prompt":
            new, batch = min(new, 600), min(batch, 4)
    hi = max(hi, new)
    if kind == "prompt":  # score entries of the padded batch, too
        new = min(new, max(2, 500_000_000 // (hi * kv * group * batch)))
    lo = max(new + prefix, int(hi * rng.choice([0.05, 0.5, 1.0])))
    return dict(op=op, dtype=rng.choice(["bf16", "f16"]), heads=kv * group, kv_heads=kv, dim=dim, page=page,
                batch=batch, lo=min(lo, hi), hi=hi, new=new, prefix=prefix)


def lengths(case):
    """Cache lengths (new tokens included) and new tokens of every sequence: the longest first."""
    rng = random.Random("lengths %d %d %d %d" % (case["batch"], case["lo"], case["hi"], case["new"]))
    lens = [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]
    if case["new"] == 1:
        return lens, [1] * len(lens)
    new = [case["new"]] + [_log_int(rng, 1, case["new"]) for _ in lens[1:]]
    return lens, [min(n, length - case["prefix"]) if case["prefix"] else min(n, length) for n, length in zip(new, lens)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = DTYPES[case["dtype"]], "cuda"
    heads, kv, dim, page, prefix = case["heads"], case["kv_heads"], case["dim"], case["page"], case["prefix"]
    lens, new = lengths(case)
    order = torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed)).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    cols, shared = -(-max(lens) // page), prefix // page
    need = [-(-n // page) - shared for n in lens]
    pages = shared + sum(need)
    ids = torch.randperm(pages + 3, generator=g, device=dev).to(torch.int32)  # three pages nobody uses
    table = torch.full((len(lens), cols), -1, dtype=torch.int32, device=dev)
    at = shared
    for b, n in enumerate(need):
        table[b, :shared] = ids[:shared]
        table[b, shared:shared + n] = ids[at:at + n]
        at += n
    rows = sum(new)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    state = dict(case=case, max_q=max(new), k_pages=normal(pages + 3, kv, page, dim), v_pages=normal(pages + 3, kv, page, dim),
                 page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), q_starts=None)
    if case["new"] > 1:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if case["op"] == "append":
        state["qkv"] = normal(rows, (heads + 2 * kv) * dim)
        state["q_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=dev)).to(dt)
        state["k_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=dev)).to(dt)
        freq = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
        ang = torch.arange(max(lens), dtype=torch.float64, device=dev)[:, None] * freq
        ang = torch.cat([ang, ang], -1)
        state["cos"], state["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    else:
        state["q"] = normal(rows, heads * dim) * 1.5  # normed heads: scores of a few units
    return state


def _rows(state, rows):
    """Sequence and index within its new tokens of every row."""
    if state["q_starts"] is None:
        seq = torch.arange(rows, device="cuda")
        return seq, torch.zeros_like(seq), torch.ones_like(state["seq_lens"])
    starts = state["q_starts"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, row - starts[seq], (starts[1:] - starts[:-1]).int()


def _plain_append(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    qkv, kp, vp = state["qkv"], state["k_pages"], state["v_pages"]
    rows = qkv.shape[0]
    seq, index, count = _rows(state, rows)
    pos = (state["seq_lens"] - count)[seq].long() + index
    x = qkv.view(rows, heads + 2 * kv, dim)
    f = x[:, :heads + kv].float()
    gain = torch.cat([state["q_norm"].float().expand(heads, dim), state["k_norm"].float().expand(kv, dim)])
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * gain
    turned = torch.cat([-f[..., dim // 2:], f[..., :dim // 2]], -1)
    f = (f * state["cos"][pos].float()[:, None] + turned * state["sin"][pos].float()[:, None]).to(qkv.dtype)
    where = state["page_table"][seq, pos // page].long()
    kp[where, :, pos % page] = f[:, heads:]
    vp[where, :, pos % page] = x[:, heads + kv:]
    return f[:, :heads].reshape(rows, heads * dim), kp, vp


def _plain_attention(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q, table, lens, longest = state["q"], state["page_table"], state["seq_lens"], state["max_q"]
    rows, batch, group = q.shape[0], table.shape[0], heads // kv
    seq, index, count = _rows(state, rows)
    which = table.clamp(min=0).long()
    k = state["k_pages"][which].transpose(1, 2).reshape(batch, kv, -1, dim).float()
    v = state["v_pages"][which].transpose(1, 2).reshape(batch, kv, -1, dim).float()
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


def run(state):
    case = state["case"]
    if own:
        from breeze_b200.fused import paged

        where = (state["k_pages"], state["v_pages"], state["page_table"], state["seq_lens"])
        if case["op"] == "append":
            q = paged.paged_append(state["qkv"], state["cos"], state["sin"], *where, q_starts=state["q_starts"],
                                   q_norm_w=state["q_norm"], k_norm_w=state["k_norm"], eps=1e-6)
            return q, state["k_pages"], state["v_pages"]
        lse = torch.empty(state["q"].shape[0], case["heads"], device=state["q"].device)
        if case["op"] == "paged":
            return paged.paged_attention(state["q"], *where, q_starts=state["q_starts"], max_q=state["max_q"], lse=lse), lse
        return paged.prefix_attention(state["q"], *where, case["prefix"], q_starts=state["q_starts"],
                                      max_q=state["max_q"], lse=lse), lse
    return _plain_append(state) if case["op"] == "append" else _plain_attention(state)


def work(case):
    lens, new = lengths(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    rows = sum(new)
    if case["op"] == "append":
        # qkv read, q and the cache rows written, one cos / sin row per token, lengths and table entries
        return {"bytes": rows * (2 * (heads + 2 * kv) * dim * 2 + 2 * dim * 2) + len(lens) * 8,
                "flops": rows * (heads + kv) * dim * 8}
    cached = sum(lens) - (len(lens) - 1) * case["prefix"]  # the shared prefix once
    table = sum(-(-n // case["page"]) for n in lens) * 4
    pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lens))
    return {"bytes": cached * kv * dim * 2 * 2 + rows * heads * (dim * 2 * 2 + 4) + table + len(lens) * 4,
            "flops": pairs * heads * dim * 4}


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens, table = s["seq_lens"].tolist(), s["page_table"].tolist()
    batch, group = len(lens), heads // kv
    starts = list(range(batch + 1)) if s["q_starts"] is None else s["q_starts"].tolist()
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        qkv = s["qkv"].double().view(-1, heads + 2 * kv, dim)
        q = torch.empty(qkv.shape[0], heads, dim, dtype=torch.float64, device="cuda")
        half = dim // 2
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
            k, v = turn(x[:, heads:heads + kv], s["k_norm"]), x[:, heads + kv:]
            pos = torch.arange(first, lens[b], device="cuda")
            at = torch.tensor(table[b], device="cuda")[pos // page]
            kp[at, :, pos % page] = k
            vp[at, :, pos % page] = v
        return q.reshape(-1, heads * dim), kp, vp
    rows = s["q"].shape[0]
    q = s["q"].double().view(rows, kv, group, dim)
    out = torch.zeros(rows, kv, group, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(rows, kv, group, dtype=torch.float64, device="cuda")
    for b in range(batch):
        a, z, length = starts[b], starts[b + 1], lens[b]
        ids = torch.tensor(table[b][:-(-length // page)], device="cuda")
        k = s["k_pages"][ids].transpose(0, 1).reshape(kv, -1, dim)[:, :length].double()
        v = s["v_pages"][ids].transpose(0, 1).reshape(kv, -1, dim)[:, :length].double()
        for r in range(a, z, 512):  # blocks of rows bound the score matrix
            e = min(r + 512, z)
            score = torch.einsum("thgd,hsd->thgs", q[r:e], k) / math.sqrt(dim)
            last = length - (z - torch.arange(r, e, device="cuda"))  # the row's own position
            score.masked_fill_((torch.arange(length, device="cuda") > last[:, None])[:, None, None], -math.inf)
            out[r:e] = torch.einsum("thgs,hsd->thgd", torch.softmax(score, -1), v)
            lse[r:e] = torch.logsumexp(score, -1)
    return out.reshape(rows, heads * dim), lse.reshape(rows, heads)
