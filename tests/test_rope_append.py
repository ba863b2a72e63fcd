"""rope_append_paged / rope_append_paged_q: rotation, head norm and append in one launch, against the definition in 64 bits; a run of the
attention layer's operators together; refusals."""
import ctypes as C
import math

import numpy as np
import pytest

from tests.test_span_attention import HD, PAGE, _lib


class Case:
    def __init__(self, q_lens, cached, nq, nkv, n_freq=64, axes=0, mode=2, norm=False, seed=0, extra_rows=0, cbias=0.0, attn_factor=1.0, far=0, std=1.5):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        n = lambda *s, k=1.0: (torch.randn(s, device="cuda", generator=g) * k).half()  # noqa: E731
        self.q_lens, self.cached, self.nq, self.nkv, self.mode, self.cbias, self.attn_factor = q_lens, cached, nq, nkv, mode, cbias, attn_factor
        self.rows, bsz = sum(q_lens), len(q_lens)
        total = self.rows + extra_rows
        width = max(max((c + x + PAGE - 1) // PAGE for c, x in zip(cached, q_lens)), 1)
        self.table = np.full((bsz, width), -1, np.int32)
        need = [(b, p) for b, (c, x) in enumerate(zip(cached, q_lens)) for p in range(c // PAGE, (c + x + PAGE - 1) // PAGE)]
        for (b, p), page in zip(need, r.permutation(len(need) + 2)):
            self.table[b, p] = page
        self.pages = len(need) + 2
        self.q, self.k, self.v = n(total, nq, HD, k=std), n(total, nkv, HD, k=std), n(total, nkv, HD)
        self.kc, self.vc = n(self.pages, PAGE, nkv, HD), n(self.pages, PAGE, nkv, HD)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
        self.bt, self.sl = torch.from_numpy(self.table).cuda(), torch.tensor(cached, dtype=torch.int32, device="cuda")
        self.inv_freq = (1e4 ** (-torch.arange(n_freq, dtype=torch.float64) / max(n_freq, 1))).float().cuda()
        self.positions = torch.randint(0, far or 3000, (axes, total), device="cuda", generator=g).int() if axes else None
        self.freq_axis = bytes(int(x) for x in r.integers(0, axes, n_freq)) if axes > 1 else None
        self.q_norm, self.k_norm = (n(HD, k=0.2), n(HD, k=0.2)) if norm else (None, None)
        self.place = np.concatenate([np.arange(c, c + x) for c, x in zip(cached, q_lens)] + [np.empty(0, int)]).astype(np.int64)
        seq = np.repeat(np.arange(bsz), q_lens)
        page = self.table[seq, self.place // PAGE] if self.rows else np.empty(0, int)
        self.slot = np.where(page >= 0, page.astype(np.int64) * PAGE + self.place % PAGE, -1)

    def kw(self):
        return dict(cu_q=self.cu, max_q_len=max(max(self.q_lens), 1), positions=self.positions, freq_axis=self.freq_axis, q_norm=self.q_norm,
                    k_norm=self.k_norm, norm_eps=1e-6, norm_constant_bias=self.cbias, rope_mode=self.mode, attn_factor=self.attn_factor)

    def exact(self, x, w):
        """(rotated rows, bound on a kernel's distance).  The sum of squares is off by 128 * 2^-24 relative, what is made of it and the
        product with the weight by a few more roundings; cos and sin by 2^-22 (the angle, reduced in 64 bits, is rounded to fp32 in half
        turns), the rotation by three roundings of each product: together under 2^-16 of |u| + |v|.  Then one rounding to fp16."""
        import torch
        x = x[:self.rows].double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (w.double() + self.cbias)
        n = self.inv_freq.numel()
        y, mag = x.clone(), x.abs()
        if self.mode != 0:
            pos = torch.from_numpy(self.place).cuda().double()[:, None].expand(-1, n)
            if self.positions is not None:
                axis = torch.tensor(list(self.freq_axis or bytes(n)), device="cuda")
                pos = self.positions[:, :self.rows].double()[axis].t()
            a = (pos * self.inv_freq.double())[:, None]
            u, v = (slice(0, n), slice(n, 2 * n)) if self.mode == 2 else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
            y[..., u] = (x[..., u] * a.cos() - x[..., v] * a.sin()) * self.attn_factor
            y[..., v] = (x[..., v] * a.cos() + x[..., u] * a.sin()) * self.attn_factor
            both = (x[..., u].abs() + x[..., v].abs()) * abs(self.attn_factor)
            mag[..., u], mag[..., v] = both, both
        return y, y.abs() * 2.0 ** -11 + mag * 2.0 ** -16 + 2.0 ** -25

    def run(self, ctx, in_place=False, **kw):
        import torch
        out = self.q if in_place else torch.full_like(self.q, 7.0)
        ctx.rope_append_paged(self.q, self.k, self.v, self.kc, self.vc, self.bt, self.sl, self.inv_freq, out_q=None if in_place else out,
                              **{**self.kw(), **kw})
        return out

    def check(self, ctx, in_place=False, **kw):
        import torch
        kc, vc, q = self.kc.clone(), self.vc.clone(), self.q.clone()
        wq, tq = self.exact(q, self.q_norm)
        wk, tk = self.exact(self.k, self.k_norm)
        out = self.run(ctx, in_place, **kw)
        assert bool(((out[:self.rows].double() - wq).abs() <= tq).all())
        assert torch.equal(out[self.rows:], q[self.rows:] if in_place else torch.full_like(q[self.rows:], 7.0))
        ok = torch.from_numpy(self.slot >= 0).cuda()
        at = torch.from_numpy(self.slot).cuda()[ok]
        got = self.kc.view(-1, self.nkv, HD)
        assert bool(((got[at].double() - wk[ok]).abs() <= tk[ok]).all())
        kc.view(-1, self.nkv, HD)[at] = got[at]
        vc.view(-1, self.nkv, HD)[at] = self.v[:self.rows][ok]
        assert torch.equal(self.kc, kc) and torch.equal(self.vc, vc), "the pools changed elsewhere, or the values are not the values"


SHAPES = [
    # rows, cached, heads
    ([1], [0], 16, 8), ([1], [255], 16, 8), ([1], [256], 40, 8), ([1], [131071], 16, 8), ([1] * 64, list(range(0, 64 * 50, 50)), 40, 8),
    ([0, 3, 0, 300, 1], [9, 250, 7, 511, 1023], 40, 8), ([2048, 1], [100, 5], 9, 3), ([1, 5], [10, 20], 1, 1), ([2400], [1], 6, 6), ([700], [3], 28, 4),
    ([1] * 3, [5, 6, 7], 65, 13), ([2501], [0], 40, 8), ([1] * 700, [4] * 700, 16, 8), ([1] * 1300 + [5], [4] * 1301, 2, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("axes", [0, 1, 3])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_shapes(ctx, case, axes, norm):
    c = Case(*SHAPES[case], axes=axes, norm=norm, seed=case, extra_rows=2, cbias=0.5 if norm else 0.0)
    c.check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("mode,n_freq", [(2, 64), (2, 48), (2, 8), (2, 16), (1, 64), (1, 1), (1, 33), (0, 64), (0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_modes(ctx, mode, n_freq, in_place):
    for rows in ([1, 40], [3000]):
        c = Case(rows, [500, 3][:len(rows)], 40, 8, n_freq=n_freq, mode=mode, seed=n_freq, norm=True, extra_rows=1, attn_factor=1.25, axes=2 if n_freq > 1 else 0)
        c.check(ctx, in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [100000, 2 ** 24, 2 ** 31 - 1])
def test_far_positions(ctx, far):
    Case([50, 1], [10, 900], 16, 8, axes=3, seed=far % 97, far=far).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("std", [0.0, 1e-4, 300.0])
def test_magnitudes(ctx, std):
    Case([9, 1], [10, 900], 16, 8, norm=True, seed=3, std=std).check(ctx)
    Case([9, 1], [10, 900], 16, 8, seed=3, std=std).check(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("entry", [-1, -2 ** 31, 1 << 20, 2 ** 31 - 1])
def test_rows_without_a_slot_are_rotated_only(ctx, entry):
    c = Case([40, 1], [250, 100], 40, 8, seed=1)
    c.table[0, 1] = entry
    c.bt[0, 1] = entry
    c.slot[6:40] = -1
    c.check(ctx)
    c = Case([40, 1], [250, 100], 40, 8, seed=1, axes=1)   # behind the table
    c.sl[0] = 5000
    c.slot[:40] = -1
    c.check(ctx)
    c.sl[0] = -3                                           # in front of it: rows at -3, -2, -1 are not appended
    c.slot[3:40] = c.table[0, 0] * PAGE + np.arange(37)
    c.slot[:3] = -1
    c.check(ctx)


@pytest.mark.gpu
def test_rectangular_keys_alone_and_rows_that_are_left_out(ctx):
    import torch
    c = Case([3, 3], [250, 100], 40, 8, seed=2, norm=True)
    q, k, v = c.q.view(2, 3, 40, HD), c.k.view(2, 3, 8, HD), c.v.view(2, 3, 8, HD)
    out = torch.zeros_like(q)
    a = c.run(ctx)
    kc, vc = c.kc.clone(), c.vc.clone()
    ctx.rope_append_paged(q, k, v, c.kc, c.vc, c.bt, c.sl, c.inv_freq, out_q=out, q_norm=c.q_norm, k_norm=c.k_norm)
    assert torch.equal(out.view(6, 40, HD), a) and torch.equal(c.kc, kc) and torch.equal(c.vc, vc)
    c.kc.zero_(), c.vc.zero_()
    ctx.rope_append_paged(None, k, v, c.kc, c.vc, c.bt, c.sl, c.inv_freq, k_norm=c.k_norm)
    at = torch.from_numpy(c.slot).cuda()
    assert torch.equal(c.kc.view(-1, 8, HD)[at], kc.view(-1, 8, HD)[at])
    # a sequence with more rows than declared is left out whole
    c = Case([1, 5, 2], [250, 100, 3], 40, 8, seed=2)
    before = c.kc.clone()
    out = c.run(ctx, max_q_len=2)
    assert bool((out[1:6] == 7.0).all()) and bool((out[[0, 6, 7]] != 7.0).any(-1).all())
    at = torch.from_numpy(c.slot[1:6]).cuda()
    assert torch.equal(c.kc.view(-1, 8, HD)[at], before.view(-1, 8, HD)[at])


@pytest.mark.gpu
@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (8, 8), (6, 3), (2, 5)])
@pytest.mark.parametrize("rows", [[1, 1, 7], [2600], [0, 300, 1]])
@pytest.mark.parametrize("nkv", [8, 3])
def test_quantised_pools(ctx, k_bits, v_bits, rows, nkv):
    """the codes are those that quant_cache_paged makes of the rotated keys and of the values"""
    import torch
    c = Case(rows, [250, 100, 3][:len(rows)], 5 * nkv, nkv, seed=k_bits, norm=True, extra_rows=1, axes=3)
    out = c.run(ctx)
    groups = nkv * 4
    pools = []
    for _ in range(2):
        g = torch.Generator(device="cuda").manual_seed(5)
        codes = [torch.randint(-2 ** 31, 2 ** 31 - 1, (c.pages, PAGE, groups * b), device="cuda", generator=g, dtype=torch.int64).int() for b in (k_bits, v_bits)]
        scales = [torch.rand((c.pages, PAGE, groups), device="cuda", generator=g).half() for _ in range(2)]
        pools.append((codes[0], scales[0], codes[1], scales[1]))
    qk, sk, qv, sv = pools[0]
    # its new keys as packed rows, out of the fp16 pool
    keys = torch.zeros_like(c.k)
    keys[:c.rows] = c.kc.view(-1, nkv, HD)[torch.from_numpy(c.slot).cuda()]
    ctx.quant_cache_paged(keys, qk, sk, c.v, qv, sv, c.sl, c.bt, cu_q=c.cu, seq_len=max(rows))
    got = torch.full_like(c.q, 7.0)
    ctx.rope_append_paged_q(c.q, c.k, c.v, *[pools[1][i] for i in (0, 1, 2, 3)], c.bt, c.sl, c.inv_freq, out_q=got, **c.kw())
    assert torch.equal(got, out)
    for a, b in zip(pools[0], pools[1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_layer_of_a_decode_loop(ctx):
    """Rotation and append, then attention with a window or over a shared prefix, token after token from one captured step, against the
    same in 64 bits from the tokens alone."""
    import torch
    import exl3b200
    nq, nkv, W, S, bsz, steps, P = 40, 8, 150, 4, 3, 5, 256
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(s, device="cuda", generator=g).half()  # noqa: E731
    inv_freq = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    bt = torch.tensor([[0, 1, 2], [0, 3, 4], [0, 5, 6]], dtype=torch.int32, device="cuda")
    kc, vc = n(7, PAGE, nkv, HD) * math.nan, n(7, PAGE, nkv, HD) * math.nan
    lens = [300, 256, 411]
    raw = [[n(c + steps, h, HD) for h in (nq, nkv, nkv)] for c in lens]
    for b in range(1, bsz):                                # the same first page
        raw[b][1][:P], raw[b][2][:P] = raw[0][1][:P], raw[0][2][:P]
    zero = torch.zeros(bsz, dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    packed = [torch.cat([raw[b][i][:lens[b]] for b in range(bsz)]) for i in range(3)]
    ctx.rope_append_paged(packed[0], packed[1], packed[2], kc, vc, bt, zero, inv_freq, cu_q=cu, max_q_len=max(lens))
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v = (torch.zeros((bsz, 1, h, HD), dtype=torch.float16, device="cuda") for h in (nq, nkv, nkv))
    qr, ow, op = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    start, plen = torch.tensor([0, bsz], dtype=torch.int32, device="cuda"), torch.tensor([P], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = exl3b200.CudaGraph(ctx)
    graph.capture_begin()
    s = graph.side_stream()
    ctx.rope_append_paged(q, k, v, kc, vc, bt, sl, inv_freq, out_q=qr, stream=s)
    ctx.window_attn_paged(qr, kc, vc, bt, sl, ow, W, sinks=S, stream=s)
    ctx.prefix_attn_paged(qr, kc, vc, bt, sl, start, plen, op, stream=s)
    graph.capture_end()

    def rotated(x, pos):
        a = pos.double()[:, None, None] * inv_freq.double()
        u, w = x.double()[..., :64], x.double()[..., 64:]
        return torch.cat([u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin()], -1)

    for t in range(steps):
        for b in range(bsz):
            q[b, 0], k[b, 0], v[b, 0] = (raw[b][i][lens[b] + t] for i in range(3))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        sl += 1
        for b in range(bsz):
            p = lens[b] + t
            pos = torch.arange(p + 1, device="cuda")
            kk, vv = rotated(raw[b][1][:p + 1], pos), raw[b][2][:p + 1].double()
            qq = rotated(raw[b][0][p:p + 1], pos[p:])[0].view(nkv, nq // nkv, HD)
            score = torch.einsum("hgd,khd->hgk", qq, kk) / math.sqrt(HD)
            # query and key are rounded to fp16 on the way: a score is off by 2 * 2^-11 * |q||k| scale at most
            d = 2.0 ** -10 * (torch.einsum("hgd,khd->hgk", qq.abs(), kk.abs()) / math.sqrt(HD)).amax(-1)[..., None] * 1.02
            for o, see in ((ow, (pos > p - W) | (pos < S)), (op, pos >= 0)):
                w = torch.softmax(score.masked_fill(~see, -math.inf), -1)
                want, mean = torch.einsum("hgk,khd->hgd", w, vv), torch.einsum("hgk,khd->hgd", w, vv.abs())
                tol = want.abs() * 2.0 ** -11 + mean * (torch.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -13) + 2.0 ** -20
                assert bool(((o[b, 0].view(nkv, nq // nkv, HD).double() - want).abs() <= tol).all())
    ctx.poll_status()


# ------------------------------------------------------------------------------------------------------------------- refusals

GOOD = dict(q=4096, out_q=0, k=4096, v=4096, inv=4096, pos=0, qn=0, kn=0, kc=4096, vc=4096, sk=0, sv=0, bt=4096, sl=4096, cu=0, eps=1e-6, cb=0.0,
            af=1.0, n_freq=64, axes=1, mode=2, bsz=2, seq=1, rows=2, nq=16, nkv=8, hd=128, pages=4, pps=2, kb=0, vb=0, fa=b"")
BAD = [(dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(inv=0), -1), (dict(kc=0), -1), (dict(vc=0), -1), (dict(bt=0), -1), (dict(sl=0), -1),
       (dict(q=4100), -1), (dict(out_q=4100), -1), (dict(k=4104), -1), (dict(v=4104), -1), (dict(kc=4104), -1), (dict(vc=4104), -1), (dict(qn=4098), -1),
       (dict(kn=4098), -1), (dict(n_freq=0), -1), (dict(n_freq=65), -1), (dict(n_freq=12), -2), (dict(mode=7), -1), (dict(hd=64), -2), (dict(bsz=-1), -1),
       (dict(seq=-1), -1), (dict(rows=3), -1), (dict(rows=-1), -1), (dict(nq=-1), -1), (dict(nkv=0), -1), (dict(pages=0), -1), (dict(pps=0), -1),
       (dict(axes=3), -1), (dict(pos=4096, axes=0), -1), (dict(pos=4096, axes=3, fa=bytes([0, 1, 3] * 22)[:64]), -1), (dict(fa=bytes([1] * 64)), -1),
       (dict(kb=4, vb=4), -1)]
QUANT = dict(kb=4, vb=8, sk=4096, sv=4096)
BAD_QUANT = [(dict(sk=0), -1), (dict(sv=0), -1), (dict(sk=4100), -1), (dict(kb=1), -1), (dict(vb=9), -1), (dict(kb=0), -1), (dict(kc=4104), -1)]


def _call(lib, ctx, **change):
    import exl3b200.ffi as ffi
    return lib.exl3_rope_append_paged(ctx, None, ffi._ROPE_APPEND.pack(*{**GOOD, **change}.values()))


def test_refusals_on_the_host():
    lib = _lib()
    assert _call(lib, None) == -1
    fake = C.create_string_buffer(1 << 16)
    C.memset(fake, 0xff, 4)                                # a device that never is the current one
    assert lib.exl3_rope_append_paged(fake, None, None) == -1
    for change, code in BAD + [({**QUANT, **x}, code) for x, code in BAD_QUANT]:
        assert _call(lib, fake, **change) == code, change
    for change in ({}, QUANT):
        assert _call(lib, fake, **change) == -1 and b"device" in lib.exl3_last_error(fake)


@pytest.mark.gpu
def test_wrapper_checks_shapes(ctx):
    import torch
    import exl3b200
    f = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(q=f(2, 1, 16, HD), k=f(2, 1, 8, HD), v=f(2, 1, 8, HD), k_cache=f(2, PAGE, 8, HD), v_cache=f(2, PAGE, 8, HD), block_table=i(2, 1),
                cache_seqlens=i(2), inv_freq=torch.ones(64, device="cuda"))
    ctx.rope_append_paged(**good)
    for change in (dict(q=f(2, 2, 16, HD)), dict(v=f(2, 1, 4, HD)), dict(k=f(2, 8, HD)), dict(k_cache=f(2, PAGE, 4, HD)), dict(v_cache=f(3, PAGE, 8, HD)),
                   dict(cache_seqlens=i(3)), dict(positions=i(3, 3)), dict(positions=i(3, 2), freq_axis=bytes(3)), dict(out_q=f(2, 1, 8, HD)),
                   dict(q_norm=f(64)), dict(inv_freq=f(64)), dict(freq_axis=[1] * 64)):
        with pytest.raises(exl3b200.Exl3Error):
            ctx.rope_append_paged(**{**good, **change})


# ---------------------------------------------------------------------------------------------------------------- many rows
# From 32 rows per SM on a block takes eight rows, two of them in work.

def _ragged(rows, seed):
    """sequences of 0 to 13 rows, so that borders and empty ones fall inside a block of eight, then a long one up to `rows`"""
    r = np.random.default_rng(seed)
    q = [int(x) for x in r.integers(0, 14, 150)]
    q += [rows - sum(q), 0, 3, 0]
    q[150] -= 3
    return q, [int(x) for x in r.integers(0, 700, len(q))]


def _many(extra):
    import torch
    return 32 * torch.cuda.get_device_properties(0).multi_processor_count + extra


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [-3, 0, 1, 7])
@pytest.mark.parametrize("heads,mode,n_freq,axes,norm,in_place", [
    ((40, 8), 2, 64, 0, True, False), ((40, 8), 2, 48, 3, False, True), ((9, 3), 1, 33, 2, True, True), ((2, 1), 2, 64, 0, False, True), ((65, 13), 1, 64, 0, True, False),
    ((7, 7), 0, 0, 0, True, True), ((28, 4), 2, 8, 1, False, False)])
def test_many_rows(ctx, extra, heads, mode, n_freq, axes, norm, in_place):
    """around the row count from which a block has eight rows; two rows behind the last sequence"""
    q, cached = _ragged(_many(extra - 2), abs(extra + n_freq))
    c = Case(q, cached, *heads, n_freq=n_freq, axes=axes, mode=mode, norm=norm, seed=extra + 3, extra_rows=2, cbias=0.5 if norm else 0.0, attn_factor=1.25)
    c.table[3, :] = c.bt[3] = -1                           # and a sequence without pages
    at = sum(q[:3])
    c.slot[at:at + q[3]] = -1
    c.check(ctx, in_place)


@pytest.mark.gpu
def test_many_rows_that_are_left_out_and_rectangular(ctx):
    import torch
    rows = _many(5)
    q, cached = _ragged(rows, 5)
    c = Case(q, cached, 12, 2, seed=9)
    before = c.kc.clone()
    out = c.run(ctx, max_q_len=13)                         # the long sequence has more rows than declared
    a, b = sum(q[:150]), sum(q[:151])
    assert bool((out[a:b] == 7.0).all()) and bool((out[:a] != 7.0).any(-1).all()) and bool((out[b:] != 7.0).any(-1).all())
    at = torch.from_numpy(c.slot[a:b]).cuda()
    assert torch.equal(c.kc.view(-1, 2, HD)[at], before.view(-1, 2, HD)[at])
    n = (rows + 10) // 11
    c = Case([11] * n, [(37 * i) % 500 for i in range(n)], 12, 2, seed=10, norm=True)
    out = c.run(ctx)
    kc, vc = c.kc.clone(), c.vc.clone()
    c.kc.zero_(), c.vc.zero_()
    got = torch.empty_like(c.q).view(n, 11, 12, HD)
    ctx.rope_append_paged(c.q.view(n, 11, 12, HD), c.k.view(n, 11, 2, HD), c.v.view(n, 11, 2, HD), c.kc, c.vc, c.bt, c.sl, c.inv_freq, out_q=got,
                          q_norm=c.q_norm, k_norm=c.k_norm)
    at = torch.from_numpy(c.slot).cuda()
    assert torch.equal(got.view(-1, 12, HD), out)
    for x, y in ((c.kc, kc), (c.vc, vc)):
        assert torch.equal(x.view(-1, 2, HD)[at], y.view(-1, 2, HD)[at])


@pytest.mark.gpu
@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (8, 3), (2, 5)])
@pytest.mark.parametrize("nkv", [8, 3, 1])
@pytest.mark.parametrize("extra", [0, 7])
def test_many_rows_to_quantised_pools(ctx, extra, nkv, k_bits, v_bits):
    import torch
    q, cached = _ragged(_many(extra - 1), extra + nkv)
    c = Case(q, cached, 2 * nkv, nkv, seed=k_bits, norm=True, extra_rows=1, axes=3)
    out = c.run(ctx)
    pools = []
    for _ in range(2):
        g = torch.Generator(device="cuda").manual_seed(5)
        codes = [torch.randint(-2 ** 31, 2 ** 31 - 1, (c.pages, PAGE, nkv * 4 * b), device="cuda", generator=g, dtype=torch.int64).int() for b in (k_bits, v_bits)]
        scales = [torch.rand((c.pages, PAGE, nkv * 4), device="cuda", generator=g).half() for _ in range(2)]
        pools.append((codes[0], scales[0], codes[1], scales[1]))
    qk, sk, qv, sv = pools[0]
    keys = torch.zeros_like(c.k)                           # its new keys as packed rows, out of the fp16 pool
    keys[:c.rows] = c.kc.view(-1, nkv, HD)[torch.from_numpy(c.slot).cuda()]
    ctx.quant_cache_paged(keys, qk, sk, c.v, qv, sv, c.sl, c.bt, cu_q=c.cu, seq_len=max(q))
    got = torch.full_like(c.q, 7.0)
    ctx.rope_append_paged_q(c.q, c.k, c.v, *pools[1], c.bt, c.sl, c.inv_freq, out_q=got, **c.kw())
    assert torch.equal(got, out)
    for a, b in zip(*pools):
        assert torch.equal(a, b)
