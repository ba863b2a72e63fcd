"""Attention over spans of the paged cache (window_attn_paged, prefix_attn_paged) against the definition in 64 bits, and its refusals."""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "exllamav3-rs_b200", "libexl3b200.so")
PAGE, HD = 256, 128
BIG = 1 << 30


# --------------------------------------------------------------------------------------------------------- inputs and oracle

class Batch:
    """A batch over pools that hold NaN wherever no row of the batch sees a key: what is masked may hold anything.  Table entries
    without a visible key are `unused`."""

    def __init__(self, q_lens, cached, nq, nkv, window=BIG, sinks=0, groups=None, prefix=None, copies=False, seed=0, extra_rows=0, unused=-1, q_std=1.5,
                 pages=None, drop=(), width=0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        self.q_lens, self.cached, self.nq, self.nkv, self.window, self.sinks = q_lens, cached, nq, nkv, window, sinks
        self.groups, self.prefix = groups, prefix
        bsz = len(q_lens)
        total = [c + x for c, x in zip(cached, q_lens)]
        width = max(max((t + PAGE - 1) // PAGE for t in total), 1, width, *[(p + PAGE - 1) // PAGE for p in (prefix or [0])])
        self.seen = [np.zeros(width * PAGE, bool) for _ in range(bsz)]         # positions that some row sees
        for b, (x, c) in enumerate(zip(q_lens, cached)):
            for p in range(c, c + x):
                self.seen[b][max(0, p + 1 - window):p + 1] = True
                self.seen[b][:min(sinks, p + 1)] = True
        self.table = np.full((bsz, width), unused, np.int32)
        self.first = list(range(bsz))                                          # whose table has the sequence's prefix
        self.shared = [0] * bsz
        for i, p in enumerate(prefix or []):
            for b in range(groups[i], groups[i + 1]):
                if cached[b] >= p:
                    self.first[b], self.shared[b] = groups[i], p
            if groups[i + 1] > groups[i]:
                self.seen[groups[i]][:p] |= any(q_lens[b] and self.shared[b] for b in range(groups[i], groups[i + 1]))
        self.pages = pages or sum(int(s.reshape(-1, PAGE).any(1).sum()) for s in self.seen) + 2
        free = list(range(self.pages) if pages else r.permutation(self.pages))
        for b in range(bsz):
            for n in np.nonzero(self.seen[b].reshape(-1, PAGE).any(1))[0]:
                if self.first[b] != b and (n + 1) * PAGE <= self.shared[b]:
                    if copies:
                        continue                                               # not read: through the first sequence's table
                    self.table[b, n] = self.table[self.first[b], n]
                else:
                    self.table[b, n] = free.pop()
        for b, n in drop:
            self.table[b, n] = unused
        self.k, self.v = (torch.full((self.pages, PAGE, nkv, HD), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
        for b in range(bsz):
            pos = np.nonzero(self.seen[b])[0]
            page = self.table[b, pos // PAGE]
            ok = (page >= 0) & (page < self.pages)
            at = torch.from_numpy(page[ok].astype(np.int64) * PAGE + pos[ok] % PAGE).cuda()
            for t, std in ((self.k, 1.0), (self.v, 0.5)):
                flat = t.view(-1, nkv, HD)
                new = (torch.randn((at.numel(), nkv, HD), device="cuda", generator=g) * std).half()
                if self.first[b] != b:                                         # a partly shared page: the prefix's tokens are copies
                    share = torch.from_numpy(pos[ok] < self.shared[b]).cuda()
                    src = self._where(self.first[b], pos[ok])
                    new = torch.where(share[:, None, None], flat[src], new)
                flat[at] = new
        rows = sum(q_lens)
        self.rows, self.extra = rows, extra_rows
        self.q = (torch.randn((rows + extra_rows, nq, HD), device="cuda", generator=g) * q_std).half()
        self.o = torch.full_like(self.q, 7.0)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
        self.bt = torch.from_numpy(self.table).cuda()
        self.sl = torch.tensor(cached, dtype=torch.int32, device="cuda")

    def _where(self, b, pos):
        import torch
        page = np.maximum(self.table[b, pos // PAGE], 0).astype(np.int64)
        return torch.from_numpy(page * PAGE + pos % PAGE).cuda()

    def exact(self, scale=None):
        """(output, bound on a kernel's distance from it), both in 64 bits.

        The bound.  A score is a sum of 128 products in fp32: off by at most d = 2 * 136 * 2^-24 * scale * sum |q||k| (any order, and
        twice that for the scaling and the exponential's argument), so a weight by a factor of e^(2d) against the largest.  Weights are
        rounded to fp16 where they enter the second product (2^-11 of each, at least 2^-25 absolute, the largest being 1 or more), which
        sums n of them in fp32 (2 n 2^-24).  The result is rounded to fp16 once (2^-11, or half of the smallest step)."""
        import torch
        scale = scale or 1.0 / math.sqrt(HD)
        G = self.nq // self.nkv
        q = self.q[:self.rows].double().view(self.rows, self.nkv, G, HD)
        out, tol = torch.zeros_like(q), torch.zeros_like(q)
        row = 0
        for b, (x, c) in enumerate(zip(self.q_lens, self.cached)):
            pos = np.nonzero(self.seen[b])[0]
            own = pos if self.first[b] == b else pos[pos >= self.shared[b]]
            tab = np.concatenate([self.table[self.first[b], np.arange(self.shared[b]) // PAGE] if self.first[b] != b else np.empty(0, np.int32),
                                  self.table[b, own // PAGE]])
            pos = np.concatenate([np.arange(self.shared[b]) if self.first[b] != b else np.empty(0, np.int64), own]).astype(np.int64)
            there = (tab >= 0) & (tab < self.pages)
            pos, tab = pos[there], tab[there].astype(np.int64)
            if x == 0 or pos.size == 0:
                row += x
                continue
            at = torch.from_numpy(tab * PAGE + pos % PAGE).cuda()
            k, v = self.k.view(-1, self.nkv, HD)[at].double(), self.v.view(-1, self.nkv, HD)[at].double()
            pos_t = torch.from_numpy(pos).cuda()
            me = torch.arange(c, c + x, device="cuda")[:, None]
            see = (pos_t[None] <= me) & ((pos_t[None] > me - self.window) | (pos_t[None] < self.sinks))
            for h in range(self.nkv):
                qq = q[row:row + x, h]
                s = torch.einsum("igd,kd->igk", qq, k[:, h]) * scale
                d = (2 * 136 * 2.0 ** -24 * scale * torch.einsum("igd,kd->igk", qq.abs(), k[:, h].abs())).masked_fill(~see[:, None], 0.0).amax(-1, keepdim=True)
                s = s.masked_fill(~see[:, None], -math.inf)
                top = s.amax(-1, keepdim=True)
                w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                n = see.sum(-1).clamp(min=1)[:, None, None].double()
                l = w.sum(-1, keepdim=True)
                w = w / torch.where(l == 0, 1.0, l)
                o = torch.einsum("igk,kd->igd", w, v[:, h])
                a = torch.einsum("igk,kd->igd", w, v[:, h].abs())
                vmax = v[:, h].abs().amax()
                out[row:row + x, h] = o
                tol[row:row + x, h] = o.abs() * 2.0 ** -11 + 2.0 ** -25 + a * (2.0 ** -11 + 4 * d + 4 * n * 2.0 ** -24 + 2.0 ** -20) + n * 2.0 ** -25 * vmax / torch.clamp(l, min=1.0)
            row += x
        return out.view(self.rows, self.nq, HD), tol.view(self.rows, self.nq, HD)

    def check(self, got, scale=None):
        import torch
        want, tol = self.exact(scale)
        over = ((got[:self.rows].double() - want).abs() / tol).nan_to_num(nan=math.inf)
        over = torch.where(got[:self.rows].isfinite(), over, torch.full_like(over, math.inf))
        assert over.numel() == 0 or over.max().item() <= 1.0, (over.max().item(), np.unravel_index(over.argmax().item(), over.shape))
        assert bool((got[self.rows:] == 7.0).all()), "rows behind the last sequence were written"


def window(ctx, b, **kw):
    ctx.window_attn_paged(b.q, b.k, b.v, b.bt, b.sl, b.o, b.window, sinks=b.sinks, cu_q=b.cu, max_q_len=max(max(b.q_lens), 1), **kw)
    ctx.poll_status()
    return b.o


def prefix(ctx, b, **kw):
    import torch
    start, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (b.groups, b.prefix))
    ctx.prefix_attn_paged(b.q, b.k, b.v, b.bt, b.sl, start, lens, b.o, cu_q=b.cu, max_q_len=max(max(b.q_lens), 1), **kw)
    ctx.poll_status()
    return b.o


# ------------------------------------------------------------------------------------------------------------------- windows

WINDOWS = [
    # one token with nothing in front of it; with one; at the edges of tiles and pages
    ([1], [0], 8, 0, 16, 8), ([1], [1], 1, 0, 16, 8), ([1], [63], 64, 0, 16, 8), ([1], [64], 64, 4, 16, 8), ([1], [255], 256, 0, 40, 8),
    ([1], [256], 256, 1, 40, 8), ([1], [127], 1000, 4, 64, 8), ([1], [700], 128, 4, 16, 8),
    # a window of one key, with and without first tokens; first tokens that reach into the window or past it
    ([5], [300], 1, 0, 40, 8), ([5], [300], 1, 3, 40, 8), ([3], [100], 64, 60, 16, 8), ([3], [100], 64, 500, 16, 8), ([40], [0], 16, 4, 16, 8),
    # head ratios: none shared, odd, more than a row block
    ([1, 3], [500, 77], 200, 4, 6, 6), ([1, 2, 9], [500, 1000, 3], 333, 5, 9, 3), ([2, 1], [70, 900], 128, 4, 32, 1), ([7, 30], [600, 20], 100, 9, 28, 4),
    ([1], [400], 100, 2, 128, 1), ([3, 1], [400, 90], 100, 2, 100, 1), ([40, 1, 2], [300, 90, 1000], 333, 2, 17, 1), ([90], [300], 333, 2, 33, 1),
    # ragged: sequences without rows, decode rows beside chunks, many short ones, one after a long window
    ([0, 1, 0, 130, 1, 0], [10, 2000, 0, 513, 0, 99], 512, 4, 40, 8), ([1] * 40, list(range(0, 4000, 100)), 1024, 4, 16, 8),
    ([1, 64, 1, 2, 333], [3000, 100, 5, 1500, 1], 256, 70, 32, 4), ([1, 1], [9000, 5], 8192, 300, 40, 8), ([300], [1000], 5000, 0, 16, 2),
    ([257], [255], 63, 1, 16, 8), ([129], [0], 129, 0, 5, 1), ([64, 64], [4096, 4095], 4096, 64, 16, 8), ([1] * 300, [20] * 300, 16, 2, 16, 8),
    ([2] * 1200, [30] * 1200, 16, 2, 16, 8),
    # both classes large enough that they run side by side
    ([1, 251, 1, 251] * 2 + [1] * 24, [600 + 137 * i for i in range(32)], 1024, 4, 40, 8), ([1] * 90 + [300] * 2, [5 * i for i in range(92)], 4096, 0, 9, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(WINDOWS)))
def test_window_shapes(ctx, case):
    q_lens, cached, w, sinks, nq, nkv = WINDOWS[case]
    b = Batch(q_lens, cached, nq, nkv, w, sinks, seed=case, extra_rows=3)
    b.check(window(ctx, b))


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,cached", [(1, [5, 900, 256]), (4, [0, 3, 700]), (33, [64, 1, 2000])])
def test_window_rectangular(ctx, q_len, cached):
    b = Batch([q_len] * 3, cached, 40, 8, 200, 4, seed=q_len)
    q, o = b.q.view(3, q_len, 40, HD), b.o.view(3, q_len, 40, HD)
    ctx.window_attn_paged(q, b.k, b.v, b.bt, b.sl, o, 200, sinks=4)
    b.check(b.o)


@pytest.mark.gpu
@pytest.mark.parametrize("unused", [-1, -2 ** 31, 2 ** 31 - 1, 100000])
@pytest.mark.parametrize("q_lens", [[1, 2], [1, 50]])
def test_window_entries_outside_the_pool(ctx, unused, q_lens):
    """keys of visible entries outside the pool are left out; a row all of whose keys are gone gives zeros"""
    b = Batch(q_lens, [600, 300], 16, 8, 400, 4, unused=unused, drop=[(0, 1), (1, 0)])
    b.check(window(ctx, b))
    b = Batch(q_lens, [100, 90], 16, 8, 400, 4, unused=unused, drop=[(0, 0), (1, 0)])
    assert bool((window(ctx, b) == 0).all())


@pytest.mark.gpu
def test_window_lengths_out_of_range(ctx):
    """positions behind the table see what the table has; negative ones nothing"""
    import torch
    b = Batch([1, 20], [500, 470], 16, 8, 300, 4, seed=3)
    b.sl.copy_(torch.tensor([-5, 470]))
    got = window(ctx, b).clone()
    assert bool((got[0] == 0).all())
    want, tol = b.exact()
    assert bool(((got[1:].double() - want[1:]).abs() <= tol[1:]).all())
    for far in (5000, 2 ** 31 - 1):
        b.sl.copy_(torch.tensor([far, 470]))
        got = window(ctx, b)
        assert bool(got[0].isfinite().all())               # its first tokens: the window is behind the table
        assert bool(((got[1:].double() - want[1:]).abs() <= tol[1:]).all())


@pytest.mark.gpu
def test_sequences_with_more_rows_than_declared_are_left_out(ctx):
    import torch
    b = Batch([1, 40, 2], [100, 300, 50], 16, 8, 64, 4, seed=5)
    ctx.window_attn_paged(b.q, b.k, b.v, b.bt, b.sl, b.o, 64, sinks=4, cu_q=b.cu, max_q_len=2)
    want, tol = b.exact()
    assert bool((b.o[1:41] == 7.0).all())
    keep = torch.tensor([0, 41, 42])
    assert bool(((b.o[keep].double() - want[keep]).abs() <= tol[keep]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("q_std", [0.0, 8.0])
def test_window_scales(ctx, scale, q_std):
    """equal scores, and scores of hundreds"""
    b = Batch([1, 3, 70], [900, 10, 2000], 40, 8, 700, 4, seed=8, q_std=q_std)
    b.check(window(ctx, b, sm_scale=scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens", [[1], [60]])
def test_window_offsets_past_32_bits(ctx, q_lens):
    """pages whose elements stand behind 2^31, and bytes behind 2^32"""
    import torch
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs two pools of 4.4 GB")
    b = Batch(q_lens, [3000], 16, 8, 2500, 4, seed=9, pages=8400)
    assert int(b.table.max()) * PAGE * 8 * HD > 2 ** 31
    b.check(window(ctx, b))
    del b
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------------------ shared prefixes

PREFIXES = [
    # rows, cached, heads, groups, prefixes
    ([1], [300], 16, 8, [0, 1], [256]), ([1, 1], [256, 256], 16, 8, [0, 2], [256]), ([1, 1, 1, 1], [530, 812, 600, 700], 16, 8, [0, 4], [512]),
    ([1] * 5, [2100, 2049, 3000, 2048, 2200], 40, 8, [0, 5], [2048]), ([8] * 6, [1100, 1030, 1500, 1024, 1040, 2000], 64, 8, [0, 6], [1024]),
    # prefixes that end inside a page or a tile, or after one token
    ([1, 2, 1], [1000, 1300, 900], 40, 8, [0, 3], [900]), ([1, 1], [5, 700], 16, 8, [0, 2], [1]), ([3, 70], [333, 400], 28, 4, [0, 2], [333]),
    # several groups, sequences of no group in front, between and behind, empty groups, groups of one, prefixes of nothing
    ([1] * 9, [600, 700, 300, 1200, 1300, 50, 800, 0, 40], 40, 8, [1, 3, 5, 5, 7], [256, 1024, 512, 0]),
    ([1, 0, 5, 1, 90, 1], [600, 700, 900, 1200, 1300, 300], 32, 4, [0, 3, 5], [512, 1024]),
    # sequences that have not cached the whole prefix, the first one among them where nobody else needs its table
    ([1, 1, 1], [1100, 300, 1024], 40, 8, [0, 3], [1024]), ([2, 40, 1], [700, 10, 3], 16, 8, [0, 3], [640]), ([1, 1], [100, 200], 16, 8, [0, 2], [512]),
    # chunks of many rows, head ratios
    ([130, 1, 257], [2500, 2048, 3000], 40, 8, [0, 3], [2048]), ([1, 9, 1], [800, 900, 1000], 6, 6, [0, 3], [768]), ([1, 2], [800, 900], 32, 1, [0, 2], [768]),
    ([1] * 70, [520 + 7 * i for i in range(70)], 9, 3, [0, 70], [512]), ([1] * 3, [5000, 6000, 20000], 16, 8, [0, 3], [4864]), ([1, 1], [0, 3], 16, 8, [0], []),
    ([2] * 1100, [300] * 1100, 16, 8, [0, 500, 1100], [256, 256]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("width", [0, 9000])
@pytest.mark.parametrize("copies", [False, True])
@pytest.mark.parametrize("case", range(len(PREFIXES)))
def test_prefix_shapes(ctx, case, copies, width):
    """narrow tables, of which a few sequences read a prefix each, and wide ones, which may hold long prefixes"""
    q_lens, cached, nq, nkv, groups, lens = PREFIXES[case]
    if width and len(q_lens) > 100:
        width = 500
    b = Batch(q_lens, cached, nq, nkv, groups=groups, prefix=lens, copies=copies, seed=case, extra_rows=2, width=width)
    b.check(prefix(ctx, b))


@pytest.mark.gpu
def test_prefix_rectangular_and_plain_causal(ctx):
    """the same as bighead_attn_paged over the same tables, whatever the groups"""
    import torch
    b = Batch([4] * 6, [700, 800, 1024, 900, 1500, 768], 40, 8, groups=[0, 6], prefix=[512], seed=1)
    q = b.q.view(6, 4, 40, HD)
    outs = []
    for start, lens in (([0, 6], [512]), ([0, 2, 6], [512, 256]), ([0], []), ([6, 6], [512])):
        o = torch.zeros_like(q)
        ctx.prefix_attn_paged(q, b.k, b.v, b.bt, b.sl, torch.tensor(start, dtype=torch.int32, device="cuda"),
                              torch.tensor(lens, dtype=torch.int32, device="cuda"), o)
        b.check(o.view(24, 40, HD))
        outs.append(o)
    # bighead_attn_paged sees the keys of this call as appended: the pools have them already, so it appends them again as they are
    pos = (b.sl[:, None].long() + torch.arange(4, device="cuda"))
    at = torch.gather(b.bt.long(), 1, pos // PAGE) * PAGE + pos % PAGE
    k, v = (t.view(-1, 8, HD)[at].contiguous() for t in (b.k, b.v))
    o = torch.zeros_like(q)
    b.k.nan_to_num_(nan=0.0), b.v.nan_to_num_(nan=0.0)
    ctx.bighead_attn_paged(q, k, v, b.k, b.v, b.bt, b.sl, o)
    b.check(o.view(24, 40, HD))


@pytest.mark.gpu
def test_prefix_lengths_are_read_at_replay(ctx):
    """a captured call goes by the lengths, tables and groups of its replay"""
    import torch
    import exl3b200
    b = Batch([1] * 8, [900 + 10 * i for i in range(8)], 40, 8, groups=[0, 8], prefix=[768], seed=2)
    start, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (b.groups, b.prefix))
    lens_now, sl_now = torch.zeros_like(lens), torch.zeros_like(b.sl)
    w = Batch([1] * 8, [900 + 10 * i for i in range(8)], 40, 8, 300, 4, seed=2)
    graph = exl3b200.CudaGraph(ctx)
    torch.cuda.synchronize()
    graph.capture_begin()
    s = graph.side_stream()
    ctx.prefix_attn_paged(b.q, b.k, b.v, b.bt, sl_now, start, lens_now, b.o, cu_q=b.cu, max_q_len=1, stream=s)
    ctx.window_attn_paged(w.q, w.k, w.v, w.bt, sl_now, w.o, 300, sinks=4, cu_q=w.cu, max_q_len=1, stream=s)
    graph.capture_end()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
    lens_now.copy_(lens), sl_now.copy_(b.sl)
    torch.cuda.synchronize()
    for _ in range(3):
        b.o.fill_(7.0), w.o.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b.check(b.o)
        w.check(w.o)


@pytest.mark.gpu
def test_classes_side_by_side_in_a_graph(ctx):
    """a call that forks to a second stream and joins, captured and replayed, and eager calls right behind one another"""
    import torch
    import exl3b200
    b = Batch([1] * 28 + [251] * 4, [600 + 137 * i for i in range(32)], 40, 8, 1024, 4, seed=12)
    call = lambda s=None: ctx.window_attn_paged(b.q, b.k, b.v, b.bt, b.sl, b.o, 1024, sinks=4, cu_q=b.cu, max_q_len=251, stream=s)  # noqa: E731
    for _ in range(5):
        call()
    b.check(b.o)
    first = b.o.clone()
    graph = exl3b200.CudaGraph(ctx)
    torch.cuda.synchronize()
    graph.capture_begin()
    for _ in range(2):
        call(graph.side_stream())
    graph.capture_end()
    for _ in range(3):
        b.o.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.o, first)
    ctx.poll_status()


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call(ctx):
    import torch
    b = Batch([1] * 20 + [40], [100 * i for i in range(1, 22)], 40, 8, 1500, 4, seed=4)
    first = window(ctx, b).clone()
    p = Batch([1] * 12 + [30], [1200 + 50 * i for i in range(13)], 40, 8, groups=[0, 13], prefix=[1024], seed=4)
    first_p = prefix(ctx, p).clone()
    for _ in range(10):
        assert torch.equal(window(ctx, b), first)
        assert torch.equal(prefix(ctx, p), first_p)


@pytest.mark.gpu
def test_two_contexts_on_two_streams(ctx):
    """calls side by side, a context and a stream each"""
    import torch
    import exl3b200
    other = exl3b200.Ctx(0, workspace_bytes=64 << 20)
    a = Batch([1] * 24, [3000 + 10 * i for i in range(24)], 40, 8, 2000, 4, seed=6)
    b = Batch([1] * 24, [3000 + 10 * i for i in range(24)], 40, 8, groups=[0, 24], prefix=[2816], seed=7)
    start, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (b.groups, b.prefix))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        ctx.window_attn_paged(a.q, a.k, a.v, a.bt, a.sl, a.o, 2000, sinks=4, cu_q=a.cu, max_q_len=1, stream=s1)
        other.prefix_attn_paged(b.q, b.k, b.v, b.bt, b.sl, start, lens, b.o, cu_q=b.cu, max_q_len=1, stream=s2)
    torch.cuda.synchronize()
    a.check(a.o)
    b.check(b.o)
    other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,mb", [(32, 90), (25, 84), (12, 72)])
def test_prefix_with_little_scratch(rows, mb):
    """partial sums of 20 sequences' prefixes: a place per row and head has room once (prefixes stay whole), twice, and three times"""
    import exl3b200
    place = 20 * rows * 40 * 528
    assert (mb << 18) // place == {32: 1, 25: 2, 12: 3}[rows]
    small = exl3b200.Ctx(0, workspace_bytes=mb << 20)
    b = Batch([rows] * 20, [2000 + 30 * i for i in range(20)], 40, 8, groups=[0, 11, 20], prefix=[1900, 1000], seed=21)
    b.check(prefix(small, b))
    small.close()


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 1]])
def test_too_little_scratch_is_refused(q_lens):
    import exl3b200
    small = exl3b200.Ctx(0, workspace_bytes=1 << 20)
    b = Batch(q_lens, [100, 300], 16, 8, 64, 4, groups=[0, 2], prefix=[64], seed=22)
    for call in (window, prefix):
        with pytest.raises(exl3b200.Exl3Error, match="scratch"):
            call(small, b)
    assert bool((b.o == 7.0).all())
    small.close()


@pytest.mark.gpu
def test_empty_calls(ctx):
    import torch
    f = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ctx.window_attn_paged(f(0, 16, HD), f(2, PAGE, 8, HD), f(2, PAGE, 8, HD), i(0, 1), i(0), f(0, 16, HD), 5, cu_q=i(1), max_q_len=1)
    ctx.window_attn_paged(f(2, 0, 16, HD), f(2, PAGE, 8, HD), f(2, PAGE, 8, HD), i(2, 1), i(2), f(2, 0, 16, HD), 5)
    ctx.prefix_attn_paged(f(2, 0, 16, HD), f(2, PAGE, 8, HD), f(2, PAGE, 8, HD), i(2, 1), i(2), i(1), i(0), f(2, 0, 16, HD))
    o = f(3, 16, HD) + 7                                   # no sequence has rows
    ctx.window_attn_paged(f(3, 16, HD), f(2, PAGE, 8, HD), f(2, PAGE, 8, HD), i(2, 1), i(2), o, 5, cu_q=i(3), max_q_len=1)
    assert bool((o == 7).all())


# ------------------------------------------------------------------------------------------------------------------- refusals

def _lib():
    if not os.path.exists(LIB):
        sys.path.insert(0, ROOT)
        import __graft_entry__
        __graft_entry__.build()
    import exl3b200
    return exl3b200.lib()


GOOD = dict(q=4096, k=4096, v=4096, bt=4096, sl=4096, cu=0, o=4096, bsz=2, q_len=1, rows=2, nq=16, nkv=8, hd=128, pages=4, pps=2, scale=0.0,
            window=8, sinks=0, gs=4096, pl=4096, groups=1)
BAD = [(dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(bt=0), -1), (dict(sl=0), -1), (dict(o=0), -1), (dict(q=4098), -1), (dict(o=4104), -1),
       (dict(k=4100), -1), (dict(v=4100), -1), (dict(bsz=-1), -1), (dict(q_len=-1), -1), (dict(rows=3), -1), (dict(rows=-1), -1), (dict(nq=0), -1),
       (dict(nkv=0), -1), (dict(nq=12), -1), (dict(hd=64), -2), (dict(pages=0), -1), (dict(pps=0), -1), (dict(pps=1 << 23), -1), (dict(scale=-1.0), -1),
       (dict(scale=math.nan), -1), (dict(scale=math.inf), -1), (dict(bsz=1 << 30, rows=1 << 30), -2), (dict(bsz=8193, rows=8193), -2),
       (dict(nq=8 * 128, rows=1 << 21, cu=4096), -1), (dict(nq=8 * 129), -2)]
WIDE = [(dict(bsz=1024, rows=1024, pps=1 << 17, window=1 << 30), -2),
        (dict(rows=1 << 24, q_len=1 << 24, cu=4096, nq=64, nkv=8, pps=1 << 12, window=1 << 30), -2)]     # 2^31 key tiles and more
BAD_WINDOW = [(dict(window=0), -1), (dict(window=-3), -1), (dict(sinks=-1), -1)]
BAD_PREFIX = [(dict(groups=-1), -1), (dict(groups=3), -1), (dict(gs=0), -1), (dict(pl=0), -1)]


def _call(lib, which, ctx, **change):
    a = {**GOOD, **change}
    tail = [a[n] for n in ("o", "bsz", "q_len", "rows", "nq", "nkv", "hd", "pages", "pps")]
    head = [ctx, None] + [a[n] for n in ("q", "k", "v", "bt", "sl", "cu")]
    if which == "window":
        return lib.exl3_window_attn_paged(*head, *tail, a["window"], a["sinks"], a["scale"])
    return lib.exl3_prefix_attn_paged(*head, a["gs"], a["pl"], a["groups"], *tail, a["scale"])


@pytest.mark.parametrize("which", ["window", "prefix"])
def test_refusals_on_the_host(which):
    """every bad argument is refused before anything is launched: on a machine without a GPU, with a context that is only memory"""
    lib = _lib()
    assert _call(lib, which, None) == -1
    fake = C.create_string_buffer(1 << 16)
    C.memset(fake, 0xff, 4)                                # a device that never is the current one
    for change, code in BAD + WIDE + (BAD_WINDOW if which == "window" else BAD_PREFIX):
        assert _call(lib, which, fake, **change) == code, change
    assert _call(lib, which, fake) == -1 and b"device" in lib.exl3_last_error(fake)


def test_refusals_of_the_wrapper():
    import torch
    import exl3b200
    c = exl3b200.Ctx.__new__(exl3b200.Ctx)
    c._h, c.device = None, 0
    t = torch.zeros((2, 1, 16, HD), dtype=torch.float16)
    with pytest.raises(exl3b200.Exl3Error, match="CUDA"):
        c.window_attn_paged(t, t, t, t, t, t, 5)
    with pytest.raises(exl3b200.Exl3Error, match="CUDA"):
        c.prefix_attn_paged(t, t, t, t, t, t, t, t)


@pytest.mark.gpu
def test_wrapper_checks_shapes(ctx):
    import torch
    import exl3b200
    f = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(q=f(2, 1, 16, HD), k_cache=f(2, PAGE, 8, HD), v_cache=f(2, PAGE, 8, HD), block_table=i(2, 1), cache_seqlens=i(2), o=f(2, 1, 16, HD), window=4)
    ctx.window_attn_paged(**good)
    for change in (dict(q=f(3, 1, 16, HD)), dict(q=f(2, 16, HD)), dict(o=f(2, 1, 8, HD)), dict(k_cache=f(2, 128, 8, HD), v_cache=f(2, 128, 8, HD)),
                   dict(v_cache=f(3, PAGE, 8, HD)), dict(cache_seqlens=i(3)), dict(block_table=i(2, 1).long()), dict(q=f(2, 1, 16, HD).float()),
                   dict(cu_q=i(4)), dict(q=f(2, 1, HD, 16).transpose(2, 3))):
        with pytest.raises(exl3b200.Exl3Error):
            ctx.window_attn_paged(**{**good, **change})
    del good["window"]
    for gs, pl in ((i(2), i(2)), (i(4), i(3))):
        with pytest.raises(exl3b200.Exl3Error):
            ctx.prefix_attn_paged(**good, group_start=gs, prefix_lens=pl)


# --------------------------------------------------------------------------------------------------------- scores far from 0

@pytest.mark.gpu
@pytest.mark.parametrize("dims", [1, 128])
@pytest.mark.parametrize("size", [2.0 ** 6, 2.0 ** 9, 2.0 ** 12, 2.0 ** 14])
@pytest.mark.parametrize("q_lens,groups", [([1, 1], None), ([60, 1], None), ([130], None), ([1] * 4, [0, 4]), ([1, 40], [0, 2])])
def test_scores_of_any_size(ctx, q_lens, groups, size, dims):
    """Every third key has the largest score, the others 0: the output is the mean of the former's values.  All products and sums are exact in
    fp32 (queries and keys of three significant bits, 128 equal products), so the weights of equal scores are equal whatever the scores are.
    What is left: rounding of a weight to fp16 (2^-11), fp32 sums of n weights and of the parts (2 n 2^-24 and less than 2^-20), rounding of
    the result (2^-11, or half of the smallest step)."""
    import torch
    cached = [900 + 200 * i for i in range(len(q_lens))]
    b = Batch(q_lens, cached, 40, 8, groups=groups, prefix=[700] if groups else None, width=9000 if groups else 0, seed=3)
    r = np.random.default_rng(1)
    b.q.zero_()
    b.q[..., :dims] = torch.from_numpy(r.integers(4, 8, (b.rows, 40, 1)) * (size / 2)).half().cuda()
    mark = torch.zeros(b.pages * PAGE, dtype=torch.bool, device="cuda")
    for i, t in enumerate(b.table):
        mark[(torch.from_numpy(t[t >= 0].astype(np.int64) * PAGE).cuda()[:, None] + torch.arange(0, PAGE, 3, device="cuda")).flatten()] = True
    mark = mark.view(b.pages, PAGE, 1, 1)
    live = b.k.isfinite()
    b.k.copy_(torch.where(live, (mark & (torch.arange(HD, device="cuda") < dims)) * (1.75 * size), math.nan))
    got = prefix(ctx, b) if groups else window(ctx, b)
    row = 0
    for i, (x, c) in enumerate(zip(q_lens, cached)):
        for j in range(x):
            pos = np.arange(c + j + 1)
            pos = pos[(pos % PAGE) % 3 == 0]
            page = np.where(pos < b.shared[i], b.table[b.first[i], pos // PAGE], b.table[i, pos // PAGE]).astype(np.int64)
            v = b.v.view(-1, 8, HD)[torch.from_numpy(page * PAGE + pos % PAGE).cuda()].double()
            want, mean = (t.mean(0).repeat_interleave(5, 0) for t in (v, v.abs()))
            tol = want.abs() * 2.0 ** -11 + mean * (2.0 ** -11 + 4 * pos.size * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -25
            diff = (got[row].double() - want).abs()
            assert bool((diff <= tol).all()), (i, j, (diff / tol).nan_to_num(nan=math.inf).max().item())
            row += 1


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_lens,groups", [([1, 1], None), ([60, 1], None), ([130], None), ([1] * 4, [0, 4]), ([1, 40], [0, 2])])
def test_scores_that_grow_from_key_to_key(ctx, q_lens, groups, sign):
    """Scores around +-8192 in units of the exponent (times log2 e), growing by two units per 128 keys and passing that size at another key in every row.
    Scores are whole numbers below 2^17, exact in fp32; an exponent has up to four roundings of half a step of 8192, 2^-12 each, a weight so 2^-10, twice
    as numerator and denominator; the rest as in `exact`."""
    import torch
    cached = [1400 + 60 * i for i in range(len(q_lens))]
    b = Batch(q_lens, cached, 40, 8, groups=groups, prefix=[700] if groups else None, width=9000 if groups else 0, seed=4)
    b.q.zero_()
    b.q[..., 0], b.q[..., 1], b.q[..., 2] = 32.0, 1.0, 1.0
    b.q[..., 3] = torch.arange(b.rows, device="cuda")[:, None].half()
    for i in range(len(q_lens)):
        pos = np.nonzero(b.seen[i])[0]
        pos = pos[b.table[i, pos // PAGE] >= 0]
        k = torch.zeros((pos.size, 1, HD), dtype=torch.float16, device="cuda")
        k[..., 0], k[..., 1] = 2004.0 * sign, torch.from_numpy(pos // 8).cuda().half()[:, None]
        k[..., 2], k[..., 3] = 18.0 if sign > 0 else -205.0, 1.0
        b.k.view(-1, 8, HD)[b._where(i, pos)] = k
    got = prefix(ctx, b) if groups else window(ctx, b)
    row = 0
    for i, (x, c) in enumerate(zip(q_lens, cached)):
        for j in range(x):
            pos = np.arange(c + j + 1)
            page = np.where(pos < b.shared[i], b.table[b.first[i], pos // PAGE], b.table[i, pos // PAGE]).astype(np.int64)
            at = torch.from_numpy(page * PAGE + pos % PAGE).cuda()
            k, v = b.k.view(-1, 8, HD)[at].double(), b.v.view(-1, 8, HD)[at].double()
            w = torch.softmax((k @ b.q[row, 0].double()) / math.sqrt(HD), 0)[..., None]
            want, mean = ((w * t).sum(0).repeat_interleave(5, 0) for t in (v, v.abs()))
            n = pos.size
            tol = want.abs() * 2.0 ** -11 + mean * (2.0 ** -9 + 2.0 ** -11 + 4 * n * 2.0 ** -24 + 2.0 ** -20) + n * 2.0 ** -25 * v.abs().max() + 2.0 ** -25
            diff = (got[row].double() - want).abs()
            assert bool((diff <= tol).all()), (i, j, (diff / tol).nan_to_num(nan=math.inf).max().item())
            row += 1


class _Tensor:
    """what the wrappers look at, without a GPU"""

    def __init__(self, dtype, *shape, device=0):
        import torch
        self.dtype, self.shape, self.device, self.is_cuda = dtype, torch.Size(shape), device, True

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return 4096


class _Library:
    """takes the calls of the three operators and keeps their arguments"""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.mark.parametrize("op", ["window", "prefix", "append", "append_q"])
def test_wrappers_refuse_other_devices_and_numbers_beyond_an_int(op, monkeypatch):
    """An address of another device would be taken for this one's, and a number of more than 32 bits would be cut: 2^32 + 5 is no window of 5."""
    import torch
    import exl3b200
    from exl3b200 import ffi
    f, i = torch.float16, torch.int32
    rows = dict(q=(f, 2, 16, HD), block_table=(i, 2, 3), cache_seqlens=(i, 2), cu_q=(i, 3))
    span = dict(rows, k_cache=(f, 4, PAGE, 8, HD), v_cache=(f, 4, PAGE, 8, HD), o=(f, 2, 16, HD))
    append = dict(rows, k=(f, 2, 8, HD), v=(f, 2, 8, HD), out_q=(f, 2, 16, HD), inv_freq=(torch.float32, 64), positions=(i, 3, 2), q_norm=(f, HD), k_norm=(f, HD))
    call, tensors, numbers = {
        "window": ("window_attn_paged", span, dict(window=8, sinks=4)),
        "prefix": ("prefix_attn_paged", dict(span, group_start=(i, 2), prefix_lens=(i, 1)), {}),
        "append": ("rope_append_paged", dict(append, k_cache=(f, 4, PAGE, 8, HD), v_cache=(f, 4, PAGE, 8, HD)), dict(rope_mode=2)),
        "append_q": ("rope_append_paged_q", dict(append, qk=(i, 4, PAGE, 128), sk=(f, 4, PAGE, 32), qv=(i, 4, PAGE, 128), sv=(f, 4, PAGE, 32)), dict(rope_mode=2)),
    }[op]
    numbers["max_q_len"] = 2
    library = _Library()
    monkeypatch.setattr(ffi, "lib", lambda: library)
    c = exl3b200.Ctx.__new__(exl3b200.Ctx)
    c._h, c.device = None, 0
    good = {n: _Tensor(*t) for n, t in tensors.items()}
    getattr(c, call)(**good, **numbers, stream=0)
    assert len(library.calls) == 1
    for n, t in tensors.items():
        with pytest.raises(exl3b200.Exl3Error, match="device"):
            getattr(c, call)(**{**good, n: _Tensor(*t, device=1)}, **numbers, stream=0)
    for n in numbers:
        for x in (2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1):
            with pytest.raises(exl3b200.Exl3Error, match=call):
                getattr(c, call)(**good, **{**numbers, n: x}, stream=0)
    for n, t in dict(block_table=(i, 6), **({} if "append" in op else dict(k_cache=(f, 4, PAGE, 8 * HD)))).items():
        with pytest.raises(exl3b200.Exl3Error, match=call):
            getattr(c, call)(**{**good, n: _Tensor(*t)}, **numbers, stream=0)
    assert len(library.calls) == 1


# ------------------------------------------------------------------------------------- captured calls whose batch changes

def _states(which):
    """(most rows of a sequence, heads, window, states): batches of one call's sizes, each sequences' rows, cached tokens, groups and prefixes"""
    r = np.random.default_rng(len(which))
    lens = lambda n, lo, hi: [int(x) for x in r.integers(lo, hi, n)]  # noqa: E731
    if which == "decode":                                  # prefix kernel, stream, join
        return 1, (40, 8), BIG, [([1] * 8, lens(8, 0, 900), [0, 4, 8], [0, 0]), ([1] * 8, lens(8, 5000, 6000), [0, 8, 8], [4999, 0]),
                                 ([1, 0] * 4, lens(8, 300, 900), [1, 2, 7], [256, 129]), ([0] * 8, lens(8, 300, 900), [0, 4, 8], [256, 129]),
                                 ([1] * 8, lens(8, 300, 900), [0, 3, 8], [1, 300])]
    if which == "mixed":                                   # and the sequences of many rows on tcgen05
        return 70, (40, 8), BIG, [([1, 40, 1, 3, 9, 1], lens(6, 300, 900), [0, 3, 6], [256, 300]), ([70, 1, 0, 1, 2, 1], lens(6, 3000, 4000), [0, 6, 6], [2900, 0]),
                                  ([1] * 6, lens(6, 0, 900), [0, 2, 4], [0, 0]), ([60, 3, 3, 3, 3, 3], lens(6, 128, 900), [2, 4, 6], [128, 100]),
                                  ([1, 40, 1, 3, 9, 1], lens(6, 300, 900), [0, 0, 6], [9, 257])]
    if which == "many":                                    # more sequences than a launch of the stream takes
        return 20, (16, 8), BIG, [([1] * 1100, lens(1100, 64, 300), [0, 600, 1100], [64, 60]), ([1] * 1070 + [20] + [0] * 29, lens(1100, 200, 500), [0, 1100, 1100], [200, 0]),
                                  ([0] * 40 + [1] * 1060, lens(1100, 0, 300), [0, 500, 1100], [0, 0]), ([20, 13] + [1] * 1060 + [0] * 38, lens(1100, 130, 300), [3, 900, 1050], [128, 1])]
    return 251, (40, 8), 1024, [([1] * 28 + [251] * 4, lens(32, 300, 6000), None, None), ([251, 1, 1, 100] + [1] * 28, lens(32, 0, 2000), None, None),
                                ([1] * 32, lens(32, 0, 6000), None, None), ([0] * 28 + [251, 0, 250, 4], lens(32, 2000, 6000), None, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["decode", "mixed", "many", "window"])
def test_batches_that_change_between_replays(ctx, which):
    """Wide tables, so that prefixes are read together: the prefix kernel, the kernels over own keys and the join as nodes of one graph.  Rows, lengths,
    tables, groups and prefixes of every replay are others; each state comes twice, once behind each other one."""
    import torch
    import exl3b200
    most, (nq, nkv), w, states = _states(which)
    total = max(sum(s[0]) for s in states) + 2
    batches = [Batch(q, c, nq, nkv, w, 4 if w != BIG else 0, groups=g, prefix=p, seed=i, extra_rows=total - sum(q), pages=2600 if which == "many" else 900,
                     width=300) for i, (q, c, g, p) in enumerate(states)]
    now = {n: torch.zeros_like(getattr(batches[0], n)) for n in ("q", "k", "v", "bt", "sl", "cu", "o")}
    if w == BIG:
        groups = [[torch.tensor(x, dtype=torch.int32, device="cuda") for x in (b.groups, b.prefix)] for b in batches]
        start, lens = (torch.zeros_like(x) for x in groups[0])
    graph = exl3b200.CudaGraph(ctx)
    torch.cuda.synchronize()
    before = ctx.launch_count()
    graph.capture_begin()
    args = [now[n] for n in ("q", "k", "v", "bt", "sl")]
    kw = dict(cu_q=now["cu"], max_q_len=most, stream=graph.side_stream())
    for _ in range(2):                                     # the second call behind the first one's join
        if w == BIG:
            ctx.prefix_attn_paged(*args, start, lens, now["o"], **kw)
        else:
            ctx.window_attn_paged(*args, now["o"], w, sinks=4, **kw)
    graph.capture_end()
    assert ctx.launch_count() - before == 2 * {"decode": 3, "mixed": 4, "many": 5, "window": 2}[which]
    order = [i for a in range(len(batches)) for b in range(a) for i in (a, b)]
    for i in order:
        for n, t in now.items():
            t.copy_(getattr(batches[i], n))
        if w == BIG:
            start.copy_(groups[i][0]), lens.copy_(groups[i][1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        batches[i].check(now["o"])
    ctx.poll_status()


# ---------------------------------------------------------------------------------------- both classes of a batch side by side

LOPSIDED = [
    # short contexts beside a chunk far into a document, the other way round, chunks at the beginning of theirs, few rows in all
    ([1] * 40 + [256], [200] * 40 + [8000], 4096, 40, 8), ([1] * 30 + [300] * 3, [5000] * 30 + [0, 3, 9], 2048, 32, 8), ([300] * 3 + [1] * 30, [1] * 33, 4096, 40, 8),
    ([1] * 100 + [20] * 8, [3000] * 100 + [9, 700] * 4, 2048, 40, 8), ([1] * 60 + [400, 2], [31 * i for i in range(62)], 2048, 12, 2), ([0] * 30 + [251] * 4 + [1] * 30, [999] * 64, 1024, 9, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(LOPSIDED)))
def test_classes_of_unlike_lengths_side_by_side(ctx, case):
    import torch
    q_lens, cached, w, nq, nkv = LOPSIDED[case]
    b = Batch(q_lens, cached, nq, nkv, w, 4, seed=case, extra_rows=3, width=max(w // PAGE, 40))
    first = window(ctx, b).clone()
    b.check(first)
    for _ in range(3):
        assert torch.equal(window(ctx, b), first)


@pytest.mark.gpu
@pytest.mark.parametrize("few,many", [((40, 200), (1, 256, 16384)), ((120, 150), (4, 1024, 6000))])
def test_side_by_side_is_no_detour(ctx, few, many):
    """Decode rows with short contexts beside chunks with full windows: the classes' split of the SMs goes by lengths.  Split by the window, such calls took
    1.5 to 2.1 times as long as the two classes in calls of their own; half as much again is the bound."""
    import torch
    q = [1] * few[0] + [many[1]] * many[0]
    batches = [Batch(x, c, 40, 8, 4096, 4, seed=1) for x, c in ((q, [few[1]] * few[0] + [many[2]] * many[0]), ([1] * few[0], [few[1]] * few[0]), ([many[1]] * many[0], [many[2]] * many[0]))]

    def us(b):
        times = []
        for _ in range(12):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(10):
                ctx.window_attn_paged(b.q, b.k, b.v, b.bt, b.sl, b.o, b.window, sinks=4, cu_q=b.cu, max_q_len=max(b.q_lens))
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end) * 100)
        return sorted(times[2:])[2]

    both, alone = us(batches[0]), [us(b) for b in batches[1:]]
    assert both < 1.5 * sum(alone), (both, alone)
