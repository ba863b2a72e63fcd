"""The attention layer of a serving step beyond plain causal attention over one pool, as cases that can be timed: new keys
and values rotated (by one position per token, or by time, height and width) on their way into the paged cache, attention
with a sliding window and visible first tokens over that cache, and attention of batches whose sequences share a prefix.

A case is a dict of plain values.  `listed()` names twelve; `draw(rng)` gives others of the same ranges; `prepare` makes what
a program holds before the call; `run` makes one pass, in elementary tensor operations or (`own`) through the package;
`exact` is the same in 64 bits, written apart from both."""
import json
import math
import os
import random
import sys

import torch

own = False

PAGE = 256
HD = 128

_ctx = None


def context():
    """One context per process, as a serving program keeps it."""
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "exllamav3-rs_b200"))      # the package of the tree it is run in
        import exl3b200
        _ctx = exl3b200.Ctx(0, workspace_bytes=1 << 30)
    return _ctx


# ---------------------------------------------------------------------------------------------------------------- cases
# Every case has `decode` sequences of one row and `chunks` sequences of `chunk_len` rows.

def _append(name, decode, chunks, chunk_len, ctx_lo, ctx_hi, nq, nkv, n_freq=64, axes=1, order="sections", norm=False, mode="neox"):
    return dict(name=name, op="append", decode=decode, chunks=chunks, chunk_len=chunk_len, ctx_lo=ctx_lo, ctx_hi=ctx_hi, nq=nq, nkv=nkv,
                n_freq=n_freq, axes=axes, order=order, norm=norm, mode=mode)


def _window(name, decode, chunks, chunk_len, ctx_lo, ctx_hi, window, sinks, nq, nkv):
    return dict(name=name, op="window", decode=decode, chunks=chunks, chunk_len=chunk_len, ctx_lo=ctx_lo, ctx_hi=ctx_hi, window=window,
                sinks=sinks, nq=nq, nkv=nkv)


def _prefix(name, decode, chunks, chunk_len, groups, prefix_lo, prefix_hi, tail_lo, tail_hi, nq, nkv):
    return dict(name=name, op="prefix", decode=decode, chunks=chunks, chunk_len=chunk_len, groups=groups, prefix_lo=prefix_lo,
                prefix_hi=prefix_hi, tail_lo=tail_lo, tail_hi=tail_hi, nq=nq, nkv=nkv)


def listed():
    return [
        # one token of one conversation with a small model: the smallest call, where only latency counts
        _append("append-1row", 1, 0, 0, 700, 700, 16, 8),
        # a decode step of 64 users, some of them far into long documents, of a model that normalises its heads
        _append("append-decode-64", 64, 0, 0, 128, 131072, 40, 8, norm=True),
        # continuous batching of an image model: 28 users decode while three prompts with pictures are read in odd pieces
        _append("append-images-mixed", 28, 3, 327, 512, 16384, 40, 8, axes=3, norm=True),
        # four long prompts with pictures, axes interleaved over the frequencies: the largest
        _append("append-images-prefill", 0, 4, 2048, 1, 4096, 40, 8, axes=3, order="interleaved"),
        # one token of one conversation, a short window: the smallest attention call
        _window("window-1row", 1, 0, 0, 700, 700, 128, 4, 16, 8),
        # decode of 128 users with a window of a few thousand tokens; pages behind the windows have been let go
        _window("window-decode-128", 128, 0, 0, 128, 32768, 4096, 4, 40, 8),
        # continuous batching: 28 users decode while four prompts are read in odd pieces
        _window("window-mixed", 28, 4, 251, 512, 16384, 1024, 4, 40, 8),
        # four prompts read in large pieces, the largest contraction over a window
        _window("window-prefill", 0, 4, 2048, 1024, 16384, 4096, 64, 40, 8),
        # four users of one short system prompt on a small model
        _prefix("prefix-decode-4", 4, 0, 0, 1, 512, 512, 20, 300, 16, 8),
        # 64 users of one long system prompt with tool descriptions
        _prefix("prefix-decode-64", 64, 0, 0, 1, 8192, 8192, 16, 1024, 40, 8),
        # speculative verification of 32 sequences that share one of two documents
        _prefix("prefix-verify-32", 0, 32, 8, 2, 8192, 16384, 64, 2048, 64, 8),
        # eight questions of 128 tokens about one document are read at once
        _prefix("prefix-questions-8", 0, 8, 128, 1, 32768, 32768, 1, 300, 40, 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 8), (40, 8), (40, 8), (32, 4), (64, 8), (28, 4), (12, 2), (6, 6), (32, 1), (9, 3)]


def _rows(rng, most):
    """(decode, chunks, chunk_len) with no more than `most` rows"""
    mode = rng.choice(["decode", "decode", "verify", "mixed", "chunks"])
    if mode == "decode":
        return _log_int(rng, 1, min(128, most)), 0, 0
    if mode == "verify":
        n = rng.randint(2, 12)
        return 0, _log_int(rng, 1, max(1, min(48, most // n))), n
    decode = _log_int(rng, 1, 40) if mode == "mixed" else 0
    n = rng.randint(1, 4)
    return decode, n, _log_int(rng, 13, max(14, (most - decode) // n))


def _draw_append(rng):
    nq, nkv = rng.choice(HEADS)
    decode, chunks, chunk_len = _rows(rng, 8192 * 48 // max(48, nq + nkv))
    lo = _log_int(rng, 1, 4096)
    axes = rng.choice([1, 1, 3, 3, 2])
    c = _append(None, decode, chunks, chunk_len, lo, lo * _log_int(rng, 1, 32), nq, nkv, rng.choice([64, 64, 64, 48, 32, 16]), axes,
                rng.choice(["sections", "interleaved"]), rng.random() < 0.5, rng.choice(["neox", "neox", "neox", "gptj"]))
    del c["name"]
    return c


def _draw_window(rng):
    nq, nkv = rng.choice(HEADS)
    window = _log_int(rng, 16, 8192)
    sinks = rng.choice([0, 1, 4, 4, 16, rng.randint(0, 300)])
    rows = max(64, min(8192, 8192 * 4096 * 40 // (window * nq)))
    while True:
        decode, chunks, chunk_len = _rows(rng, rows)
        seqs = decode + chunks
        if seqs * (window + sinks) * nkv <= 128 * 4100 * 8 and (decode * 1 + chunks * chunk_len) <= rows:
            break
    lo = _log_int(rng, 1, 4096)
    c = _window(None, decode, chunks, chunk_len, lo, min(65536, lo * _log_int(rng, 1, 32)), window, sinks, nq, nkv)
    del c["name"]
    return c


def _draw_prefix(rng):
    nq, nkv = rng.choice(HEADS)
    while True:
        lo = PAGE * _log_int(rng, 1, 64)
        hi = min(32768, lo * rng.randint(1, 4))
        tail_lo = _log_int(rng, 1, 128)
        tail_hi = tail_lo * _log_int(rng, 1, 24)
        decode, chunks, chunk_len = _rows(rng, 1024)
        groups = rng.choice([1, 1, 1, 2, 3])
        seqs, rows = decode + chunks, decode + chunks * chunk_len
        if groups <= seqs and rows * hi * nq <= 1024 * 32768 * 40 and seqs * (hi + tail_hi + chunk_len) * nkv <= 64 * 9216 * 8:
            break
    c = _prefix(None, decode, chunks, chunk_len, groups, lo, hi, tail_lo, tail_hi, nq, nkv)
    del c["name"]
    return c


def draw(rng):
    return rng.choice([_draw_append, _draw_window, _draw_prefix])(rng)


# ----------------------------------------------------------------------------------------------------------- batch shapes

def _spread(r, lo, hi, n):
    """n whole numbers spread over the logarithm of [lo, hi], in a mixed-up order"""
    a, b = math.log(lo), math.log(hi)
    v = [int(math.exp(a + (b - a) * (i + r.random()) / n) + 1e-9) for i in range(n)]
    r.shuffle(v)
    return v


def _lengths(case):
    """What belongs to the case: every sequence's rows and cached tokens; for groups their first sequences and prefixes."""
    q = [1] * case["decode"] + [case["chunk_len"]] * case["chunks"]
    r = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    r.shuffle(q)
    if case["op"] != "prefix":
        return q, _spread(r, case["ctx_lo"], case["ctx_hi"], len(q)), None, None
    n, g = len(q), case["groups"]
    start = [i * n // g for i in range(g + 1)]
    prefix = [PAGE * max(1, x // PAGE) for x in _spread(r, case["prefix_lo"], case["prefix_hi"], g)]
    tail = _spread(r, case["tail_lo"], case["tail_hi"], n)
    ctx = [prefix[i] + tail[b] for i in range(g) for b in range(start[i], start[i + 1])]
    return q, ctx, start, prefix


def _ragged(q):
    return len(set(q)) > 1


def _freq_axis(case):
    """the axis whose position turns each frequency"""
    n, axes = case["n_freq"], case["axes"]
    if case["order"] == "interleaved":
        return [i % axes for i in range(n)]
    first = n // 4 if axes == 3 else n // axes                       # time takes a quarter, height and width share the rest
    rest = (n - first + max(1, axes - 1) - 1) // max(1, axes - 1)
    return [0 if i < first or axes == 1 else 1 + (i - first) // rest for i in range(n)]


# ------------------------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.float16)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pools(pages, nkv, g):
    pair = [torch.empty((pages, PAGE, nkv, HD), dtype=torch.float16, device="cuda") for _ in range(2)]
    for t, std in zip(pair, (1.0, 0.5)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 1 << 28):
            flat[i:i + (1 << 28)].normal_(0.0, std, generator=g)
    return pair


def _table(needed, width, seed):
    """Block table [sequences, width] from every sequence's needed logical pages, which get pages of the pool in a mixed-up
    order; other entries are -1, as after a program has let those pages go."""
    total = sum(len(n) for n in needed)
    perm = list(range(total + 1))
    random.Random(seed).shuffle(perm)
    rows, at = [], 0
    for n in needed:
        row = [-1] * width
        for p in n:
            row[p] = perm[at]
            at += 1
        rows.append(row)
    return rows, total + 1


def _image_positions(r, rows, base, axes):
    """Positions of one sequence's rows: runs of text, where all axes count on together, and pictures, whose rows stand on
    a grid of height and width at one time."""
    out, at, now = [], 0, base
    while at < rows:
        n = min(rows - at, r.randint(1, 200))
        out += [[now + i] * axes for i in range(n)]
        at, now = at + n, now + n
        if axes > 1 and at < rows:
            h, w = r.randint(2, 24), r.randint(2, 24)
            cells = [[now] + [now + y if a % 2 else now + x for a in range(1, axes)] for y in range(h) for x in range(w)][:rows - at]
            out += cells
            at, now = at + len(cells), now + max(h, w)
    return out


def prepare(case, seed):
    q, ctx, start, prefix = _lengths(case)
    nq, nkv, rows, g = case["nq"], case["nkv"], sum(q), _gen(seed)
    lead = (rows,) if _ragged(q) else (len(q), q[0])
    cu = [0]
    for x in q:
        cu.append(cu[-1] + x)
    total = [c + x for c, x in zip(ctx, q)]
    width = max((t + PAGE - 1) // PAGE for t in total)
    s = dict(op=case["op"], q=_normal(lead + (nq, HD), g, 1.5), seqlens=_i32(ctx), cu_q=_i32(cu) if _ragged(q) else None, cu=_i32(cu),
             max_q=max(q), rows=rows, scale=1.0 / math.sqrt(HD))
    if case["op"] == "append":
        needed = [range(c // PAGE, (t + PAGE - 1) // PAGE) for c, t in zip(ctx, total)]
        table, pages = _table(needed, width, seed)
        r = random.Random(seed + 1)
        pos = [p for b, x in enumerate(q) for p in _image_positions(r, x, ctx[b], case["axes"])]
        n = case["n_freq"]
        s |= dict(k=_normal(lead + (nkv, HD), g, 1.5), v=_normal(lead + (nkv, HD), g, 0.5), pools=_pools(pages, nkv, g), table=_i32(table),
                  inv_freq=(1e6 ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda(), mode=case["mode"],
                  positions=None if case["axes"] == 1 else _i32(pos).t().contiguous(), freq_axis=None if case["axes"] == 1 else bytes(_freq_axis(case)),
                  q_norm=None, k_norm=None, eps=1e-6, out_q=torch.zeros(lead + (nq, HD), dtype=torch.float16, device="cuda"))
        s["axis"] = torch.tensor(_freq_axis(case), device="cuda")
        if case["norm"]:
            s |= dict(q_norm=_normal((HD,), g, 0.1) + 1, k_norm=_normal((HD,), g, 0.1) + 1)
        return s
    s["o"] = torch.zeros(lead + (nq, HD), dtype=torch.float16, device="cuda")
    if case["op"] == "window":
        needed = []
        for c, x, t in zip(ctx, q, total):
            first = max(0, c + 1 - case["window"]) // PAGE
            sink = range(min((min(case["sinks"], t) + PAGE - 1) // PAGE, first))
            needed.append(list(sink) + list(range(first, (t + PAGE - 1) // PAGE)))
        table, pages = _table(needed, width, seed)
        return s | dict(pools=_pools(pages, nkv, g), table=_i32(table), window=case["window"], sinks=case["sinks"])
    # every group's prefix stands in pages that its sequences share
    needed = [range(prefix[i] // PAGE, (total[b] + PAGE - 1) // PAGE) for i in range(len(prefix)) for b in range(start[i], start[i + 1])]
    table, pages = _table(list(needed) + [range(p // PAGE) for p in prefix], max(width, max(prefix) // PAGE), seed)
    for i, p in enumerate(prefix):
        for b in range(start[i], start[i + 1]):
            table[b][:p // PAGE] = table[len(q) + i][:p // PAGE]
    return s | dict(pools=_pools(pages, nkv, g), table=_i32(table[:len(q)]), group_start=_i32(start), prefix_lens=_i32(prefix),
                    longest=max(total))


# ---------------------------------------------------------------------------------------------------------- the plain form

def _sequences(s):
    """sequence of every packed row and its number in it"""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], row, right=True) - 1
    return b, row.long() - s["cu"][b].long()


def _plain_append(s):
    b, i = _sequences(s)
    at = s["seqlens"][b].long() + i
    page = s["table"][b, at // PAGE].long()
    where = page * PAGE + at % PAGE
    n, axes = s["inv_freq"].numel(), s["axis"]
    pos = at[:, None].expand(-1, n) if s["positions"] is None else s["positions"].t()[:, axes]
    angle = pos.double() * s["inv_freq"].double()                    # far positions need more than 32 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, w):
        x = x.reshape(s["rows"], -1, HD).float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float()
        if s["mode"] == "neox":
            u, v = x[..., :n], x[..., n:2 * n]
            return torch.cat([u * cos - v * sin, v * cos + u * sin, x[..., 2 * n:]], -1).to(torch.float16)
        u, v = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        return torch.cat([torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2), x[..., 2 * n:]], -1).to(torch.float16)

    kc, vc = s["pools"]
    kc.view(-1, *kc.shape[2:])[where] = rotated(s["k"], s["k_norm"])
    vc.view(-1, *vc.shape[2:])[where] = s["v"].reshape(s["rows"], -1, HD)
    return [rotated(s["q"], s["q_norm"]).view(s["q"].shape), kc, vc]


def _plain_attention(s, pos, real):
    """Attention of every sequence's rows over its keys at logical positions pos [sequences, keys], of which those that are
    `real` exist, under the mask of the operator."""
    bsz, qm, (kc, vc) = s["table"].shape[0], s["max_q"], s["pools"]
    nkv = kc.shape[2]
    group = s["q"].shape[-2] // nkv
    page = torch.where(real, s["table"].gather(1, torch.where(real, pos, 0) // PAGE), 0).long()
    where = page * PAGE + pos % PAGE
    k, v = (t.view(-1, nkv, HD)[where].permute(0, 2, 1, 3).float() for t in (kc, vc))              # [sequences, kv heads, keys, HD]
    b, i = _sequences(s)
    rows = torch.zeros((bsz, qm), dtype=torch.long, device="cuda")
    rows[b, i] = torch.arange(s["rows"], device="cuda")
    q = s["q"].reshape(s["rows"], nkv, group, HD)[rows].permute(0, 2, 3, 1, 4).float()             # [sequences, kv heads, group, rows, HD]
    at = s["seqlens"][:, None].long() + torch.arange(qm, device="cuda")
    seen = real[:, None] & (pos[:, None] <= at[..., None])
    if s["op"] == "window":
        seen &= (pos[:, None] > at[..., None] - s["window"]) | (pos[:, None] < s["sinks"])
    score = torch.matmul(q.reshape(bsz, nkv, group * qm, HD), k.transpose(2, 3)).view(bsz, nkv, group, qm, -1) * s["scale"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp_(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(bsz, nkv, group * qm, -1), v).view(bsz, nkv, group, qm, HD) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4)[b, i].to(torch.float16).view(s["q"].shape)


def _plain_window(s):
    cached, ql = s["seqlens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    total = (cached + ql)[:, None]
    sink = torch.arange(s["sinks"], device="cuda").expand(cached.numel(), -1)
    first = torch.clamp(cached + 1 - s["window"], min=s["sinks"])[:, None]
    near = first + torch.arange(s["window"] + s["max_q"] - 1, device="cuda")
    pos = torch.cat([sink, near], 1)
    return _plain_attention(s, pos, pos < total)


def _plain_prefix(s):
    ql = (s["cu"][1:] - s["cu"][:-1]).long()
    pos = torch.arange(s["longest"], device="cuda").expand(ql.numel(), -1)
    return _plain_attention(s, pos, pos < (s["seqlens"].long() + ql)[:, None])


def run(s):
    if own:
        ctx = context()
        kc, vc = s["pools"]
        if s["op"] == "append":
            ctx.rope_append_paged(s["q"], s["k"], s["v"], kc, vc, s["table"], s["seqlens"], s["inv_freq"], out_q=s["out_q"], cu_q=s["cu_q"],
                                  max_q_len=s["max_q"], positions=s["positions"], freq_axis=s["freq_axis"], q_norm=s["q_norm"],
                                  k_norm=s["k_norm"], norm_eps=s["eps"], rope_mode={"gptj": 1, "neox": 2}[s["mode"]])
            return [s["out_q"], kc, vc]
        if s["op"] == "window":
            ctx.window_attn_paged(s["q"], kc, vc, s["table"], s["seqlens"], s["o"], s["window"], sinks=s["sinks"], sm_scale=s["scale"],
                                  cu_q=s["cu_q"], max_q_len=s["max_q"])
            return s["o"]
        ctx.prefix_attn_paged(s["q"], kc, vc, s["table"], s["seqlens"], s["group_start"], s["prefix_lens"], s["o"], sm_scale=s["scale"],
                              cu_q=s["cu_q"], max_q_len=s["max_q"])
        return s["o"]
    if s["op"] == "append":
        return _plain_append(s)
    return _plain_window(s) if s["op"] == "window" else _plain_prefix(s)


# ---------------------------------------------------------------------------------------------------- what a pass requires

def work(case):
    q, ctx, start, prefix = _lengths(case)
    nq, nkv, rows = case["nq"], case["nkv"], sum(q)
    tok = nkv * HD * 4                                               # keys and values of a token
    if case["op"] == "append":
        # queries and keys in and out, values moved; a few operations per rotated value
        return {"bytes": rows * (4 * nq * HD + 2 * tok + 4 * case["axes"]), "flops": 6.0 * rows * (nq + nkv) * HD}
    nbytes, pairs = 4.0 * rows * nq * HD, 0
    for b, (x, c) in enumerate(zip(q, ctx)):
        if case["op"] == "window":
            w, n = case["window"], case["sinks"]
            near = [min(w, c + i + 1) for i in range(x)]
            pairs += sum(k + min(n, c + i + 1 - k) for i, k in enumerate(near))
            first = max(0, c + 1 - w)
            nbytes += tok * (c + x - first + min(n, first))
        else:
            pairs += x * c + x * (x + 1) // 2
            nbytes += tok * (c + x)
    if case["op"] == "prefix":
        nbytes -= sum(tok * p * (start[i + 1] - start[i] - 1) for i, p in enumerate(prefix))      # a prefix is read once
    return {"bytes": nbytes, "flops": 4.0 * HD * nq * pairs}


# ------------------------------------------------------------------------------------------------- the definition in 64 bits

def _exact_append(case, s):
    q_lens, ctx, _, _ = _lengths(case)
    n, nkv = case["n_freq"], case["nkv"]
    table = s["table"].tolist()
    token = [table[b][(c + i) // PAGE] * PAGE + (c + i) % PAGE for b, (c, x) in enumerate(zip(ctx, q_lens)) for i in range(x)]
    own_pos = torch.tensor([c + i for c, x in zip(ctx, q_lens) for i in range(x)], device="cuda", dtype=torch.float64)
    angle = torch.empty((len(token), n), dtype=torch.float64, device="cuda")
    for f, a in enumerate(_freq_axis(case)):
        angle[:, f] = (own_pos if s["positions"] is None else s["positions"][a].double()) * s["inv_freq"][f].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x, w):
        x = x.reshape(len(token), -1, HD).double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / HD + s["eps"]).sqrt() * w.double()
        out = x.clone()
        a, b = (slice(0, n), slice(n, 2 * n)) if case["mode"] == "neox" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
        out[..., a], out[..., b] = z.real, z.imag
        return out

    kc, vc = (t.double().view(-1, nkv, HD) for t in s["pools"])
    kc[token], vc[token] = turned(s["k"], s["k_norm"]), s["v"].reshape(-1, nkv, HD).double()
    return [turned(s["q"], s["q_norm"]).view(s["q"].shape), kc.view(s["pools"][0].shape), vc.view(s["pools"][1].shape)]


def _exact_attention(case, s):
    q_lens, ctx, _, _ = _lengths(case)
    nq, nkv = case["nq"], case["nkv"]
    q = s["q"].reshape(-1, nkv, nq // nkv, HD).double()
    out, at = torch.empty_like(q), 0
    for b, (x, c) in enumerate(zip(q_lens, ctx)):
        keys = torch.arange(c + x, device="cuda")
        if case["op"] == "window":
            keys = keys[(keys >= c + 1 - case["window"]) | (keys < case["sinks"])]
        token = s["table"][b].long()[keys // PAGE] * PAGE + keys % PAGE
        me = torch.arange(c, c + x, device="cuda")[:, None]
        hidden = keys[None] > me
        if case["op"] == "window":
            hidden |= (keys[None] <= me - case["window"]) & (keys[None] >= case["sinks"])
        for h in range(nkv):
            k, v = (t.view(-1, nkv, HD)[token, h].double() for t in s["pools"])
            score = torch.einsum("igd,kd->gik", q[at:at + x, h], k) / math.sqrt(HD)
            prob = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[at:at + x, h] = torch.einsum("gik,kd->igd", prob, v)
        at += x
    return out.view(s["q"].shape)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)
