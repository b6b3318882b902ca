"""Paged 8-bit caches at the edges of their calls, on the GPU: layouts whose strides say nothing, counts of zero or beyond
the rows, scores far below zero, scales that fall while scores rise, softcap in fp32, and warps that read many strips.

The reference is attention in 64 bits over what the codes stand for, on the device, one sequence at a time (`exact`).
Tolerances are the framework's bars, rel_rms 3e-4 (fp16), 2.5e-3 (bf16), 1e-5 (fp32), and 1e-5 of an LSE's rms, unless a test
says otherwise."""
import math

import pytest
import torch

import fable_attn as fa

pytestmark = pytest.mark.gpu
TDT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CDT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}
BAR = {"fp16": 3e-4, "bf16": 2.5e-3, "fp32": 1e-5}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return i32(out)


def rel(a, b):
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


class Pool:
    """A random paged cache: pages in no order, every slot full of codes, scales about 3 / Q."""

    def __init__(self, seed, lens, heads, dim, page, block, code):
        self.gen = g = torch.Generator("cuda").manual_seed(seed)
        self.page, self.block, self.code, self.heads, self.dim = page, block, code, heads, dim
        per = [(n + page - 1) // page for n in lens]
        n = sum(per) + 2
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32).cpu()
        self.table = torch.zeros(len(lens), max(max(per), 1), dtype=torch.int32)
        at = 0
        for z, p in enumerate(per):
            self.table[z, :p] = order[at:at + p]
            at += p
        self.bt = self.table.cuda()
        x = lambda: (torch.randn(n, page, heads, dim, generator=g, device="cuda") * (QMAX[code] / 3)).clamp(-QMAX[code], QMAX[code])
        self.k, self.v = ((x().round() if code == "int8" else x()).to(CDT[code]) for _ in range(2))
        self.ks, self.vs = (torch.randn(n, heads, page // block, generator=g, device="cuda").mul(0.5).exp() * (3 / QMAX[code])
                            for _ in range(2))

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def values(self, which, z, n):
        """fp64 (n, heads, dim): what the first n positions of sequence z stand for."""
        c, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        pages = self.bt[z, :(n + self.page - 1) // self.page].long()
        x = c.view(torch.int8)[pages].view(c.dtype).float().double()
        return (x * s[pages].double().repeat_interleave(self.block, 2).transpose(1, 2)[..., None]).flatten(0, 1)[:n]

    def blocks_of(self, z, n):
        """[(page, block in it)] of the first n positions of sequence z, in order."""
        return [(int(p), j) for p in self.table[z, :(n + self.page - 1) // self.page] for j in range(self.page // self.block)]


def exact(c, q, lens, news, scale=None, softcap=0.0, window=-1, alibi=None, leftpad=None, causal=True):
    """Packed out (total, Hq, D) and LSE (total, Hq), fp64."""
    hq, d = q.shape[-2:]
    g, outs, lses, at = hq // c.heads, [], [], 0
    for z, (L, n) in enumerate(zip(lens, news)):
        k, v = c.values("k", z, L), c.values("v", z, L)
        x = q[at:at + n].double().view(n, c.heads, g, d)
        at += n
        s = torch.einsum("nhgd,lhd->nhgl", x, k) * (scale or d ** -0.5)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        j, pos = torch.arange(L, device="cuda"), torch.arange(L - n, L, device="cuda")[:, None]
        if alibi is not None:
            s = s + alibi.double().view(1, c.heads, g, 1) * (j - pos)[:, None, None].double()
        seen = torch.ones(n, L, dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= pos
        if window >= 0:
            seen &= j >= pos - window
        if leftpad is not None:
            seen &= j >= leftpad[z]
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        lse = torch.logsumexp(s, -1)
        p = (s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp()
        outs.append(torch.einsum("nhgl,lhd->nhgd", p, v).reshape(n, hq, d))
        lses.append(lse.reshape(n, hq))
    return torch.cat(outs), torch.cat(lses)


def decode(c, q, lens, news, packed=False, scale=None, softcap=0.0, window=-1, alibi=None, leftpad=None, causal=True):
    """The framework's, laid out the same."""
    hq, d = q.shape[-2:]
    qq = q if packed else q.view(len(lens), news[0], hq, d)
    out, lse = fa.flash_attn_with_kvcache_8bit(
        qq, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, softmax_scale=scale, causal=causal, window_size=(window, -1), softcap=softcap,
        alibi_slopes=alibi, cu_seqlens_q=cum(news) if packed else None, max_seqlen_q=max(news) if packed else None,
        cache_leftpad=None if leftpad is None else i32(leftpad), return_softmax_lse=True)
    lse = lse.t() if packed else lse.transpose(1, 2).reshape(-1, hq)
    return out.reshape(-1, hq, d), lse


def check(got, want, dt, bar=None):
    (o, l), (wo, wl) = got, want
    assert torch.isfinite(o).all() and (torch.isneginf(l) == torch.isneginf(wl)).all()
    live = ~torch.isneginf(wl)
    assert rel(o.double(), wo) <= (bar or BAR[dt]), rel(o.double(), wo)
    err = (l.double() - wl)[live].abs().max()
    assert float(err) <= 1e-5 * max(1.0, float(wl[live].square().mean().sqrt())), float(err)


def strips_a_warp(c, lens, news, gqa, packed=False):
    """(strips that a warp takes, stages of its ring) by the kernel's rule for equal ranges."""
    w = 64 if c.dim <= 64 else 128 if c.dim <= 128 else 256
    rt = 16 if w <= 128 and (gqa > 8 or (not packed and gqa * news[0] > 8)) else 8
    st = 32 if rt == 8 and w <= 128 else 16
    ctas = 4 if w == 64 and rt == 8 else 2
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = (max(news) * gqa + rt - 1) // rt
    bound = len(lens) * tiles * ((c.bt.shape[1] * c.page + st - 1) // st)
    ranges = max(1, min(sms * ctas * 4 // c.heads, bound))
    line = sum(max(1, (n + st - 1) // st) * ((k * gqa + rt - 1) // rt) for n, k in zip(lens, news))
    return -(-line // ranges), 2 if rt == 8 else 3 if w == 128 else 4


# ---------------------------------------------------------------------------------------- layouts
def seq_first(x):
    """(batch, 1, heads, dim) as a view of (1, batch, heads, dim): dimension 1 has one entry and batch's stride.  The storage goes on
    to where that stride would lead."""
    b, _, h, d = x.shape
    wide = torch.zeros(b * b, h, d, dtype=x.dtype, device=x.device)
    wide[:b] = x[:, 0]
    y = wide[:b][None].transpose(0, 1)
    assert y.stride(1) == b * h * d and y.is_contiguous() and torch.equal(y, x)
    return y


@pytest.mark.parametrize("code", ["int8", "e4m3", "none"])
def test_one_token_with_the_sequence_dimension_first(code):
    """A dimension of one entry has a stride that says nothing, and such a tensor counts as contiguous whatever it is."""
    lens = [3, 40, 17]
    a, b = (Pool(1, [n + 1 for n in lens], 2, 64, 16, 8, "int8" if code == "none" else code) for _ in range(2))
    for c in (a, b):
        if code == "none":
            c.k, c.v, c.ks, c.vs = c.k.bfloat16(), c.v.bfloat16(), None, None
    k, v, q = a.randn(3, 1, 2, 64).bfloat16(), a.randn(3, 1, 2, 64).bfloat16(), a.randn(3, 1, 8, 64).bfloat16()
    for c, lay in ((a, lambda t: t), (b, seq_first)):
        fa.kvcache_append(lay(k), lay(v), c.k, c.v, i32(lens), c.bt, k_scale=c.ks, v_scale=c.vs)
    same = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert same(a.k, b.k) and same(a.v, b.v)
    if code == "none":
        return
    assert torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs)
    out = [fa.flash_attn_with_kvcache_8bit(x, a.k, a.v, a.ks, a.vs, i32([n + 1 for n in lens]), a.bt) for x in (q, seq_first(q))]
    assert torch.equal(*out)


@pytest.mark.parametrize("rows", [1, 3])
def test_rows_of_a_slice_need_no_copy_to_be_right(rows):
    """(batch, 1) rows cut out of longer sequences, and batches of one."""
    c = Pool(2, [30, 30], 2, 64, 16, 8, "int8")
    wide = c.randn(2, 9, 8, 64).half()
    for q in (wide[:, 4:4 + rows], wide[1:, 4:4 + rows]):
        args = (c.k, c.v, c.ks, c.vs, i32([30] * len(q)), c.bt[:len(q)])
        assert torch.equal(fa.flash_attn_with_kvcache_8bit(q, *args), fa.flash_attn_with_kvcache_8bit(q.clone(), *args))


# ---------------------------------------------------------------------------------------- counts
@pytest.mark.parametrize("code,page,block", [("int8", 16, 16), ("e4m3", 64, 64), ("int8", 32, 4), ("e4m3", 256, 256), ("int8", 8, 8)])
def test_append_counts_beyond_the_rows(code, page, block):
    """cu_seqlens_new that ends past the rows given: the rows given are appended, nothing else is written.  (The rows lie in a
    longer buffer, so that what a call must not read is there.)"""
    lens, total = [5, 0], 20
    a, b = (Pool(3, [300, 300], 2, 64, page, block, code) for _ in range(2))
    wide = a.randn(400, 2, 64)
    k, v = wide[:total], wide[200:200 + total]
    kw = lambda c: dict(k_scale=c.ks, v_scale=c.vs)
    fa.kvcache_append(k, v, a.k, a.v, i32(lens), a.bt, cu_seqlens_new=i32([0, 7, 20]), **kw(a))
    fa.kvcache_append(k, v, b.k, b.v, i32(lens), b.bt, cu_seqlens_new=i32([0, 7, 130]), **kw(b))
    for x, y in ((a.k, b.k), (a.v, b.v), (a.ks, b.ks), (a.vs, b.vs)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # a sequence that begins past them, or before them, has none
    before = [t.clone() for t in (b.k, b.v, b.ks, b.vs)]
    fa.kvcache_append(k, v, b.k, b.v, i32(lens), b.bt, cu_seqlens_new=i32([25, 60, 99]), **kw(b))
    fa.kvcache_append(k, v, b.k, b.v, i32(lens), b.bt, cu_seqlens_new=i32([-9, -9, -4]), **kw(b))
    for x, y in zip(before, (b.k, b.v, b.ks, b.vs)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("code,page,block", [("int8", 16, 16), ("e4m3", 64, 64), ("int8", 16, 4), ("e4m3", 16, 1), ("int8", 8, 8)])
def test_append_leaves_sequences_without_new_tokens_alone(code, page, block):
    """Counts of 0 beside others: their blocks keep codes and scales bit by bit (a scale of 0 among them), their table rows are not
    looked at, and a page that such a sequence shares with one that appends gets what the latter writes."""
    lens, news = [3, 5, 6, 2], [2, 0, 0, 0]
    c = Pool(4, [40] * 4, 2, 64, page, block, code)
    c.ks.zero_()
    c.vs[::2] = 1e-35
    c.table[2, 0] = c.table[0, 0]     # shares the first sequence's page
    c.table[3] = -1                   # has no pages at all
    c.bt = c.table.cuda()
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    x = c.randn(2, 2, 64) * 5
    fa.device_error(clear=True)
    fa.kvcache_append(x, x, c.k, c.v, i32(lens), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=cum(news))
    assert fa.device_error(clear=True) == 0
    pg, touched = int(c.table[0, 0]), sorted({3 // block, 4 // block})
    for old, new in zip(before[2:], (c.ks, c.vs)):
        want = old.clone()
        for b in touched:
            rows = x[[i for i in range(2) if (3 + i) // block == b]]
            want[pg, :, b] = torch.maximum(rows.abs().amax((0, 2)) / QMAX[code], old[pg, :, b] if b * block < 3 else torch.zeros(2, device="cuda"))
        torch.testing.assert_close(new, want, rtol=1e-6, atol=0)
        keep = torch.ones_like(old, dtype=torch.bool)
        keep[pg, :, touched] = False
        assert torch.equal(new[keep], old[keep])
    slots = torch.ones(c.k.shape[:2], dtype=torch.bool, device="cuda")
    slots[pg, touched[0] * block:5] = False   # earlier codes of a block may go onto its larger scale
    for old, new in zip(before, (c.k, c.v)):
        assert torch.equal(old.view(torch.int8)[slots], new.view(torch.int8)[slots])
    # as whole batches do: all of them idle
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    fa.kvcache_append(x, x, c.k, c.v, i32(lens), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=i32([0] * 5))
    assert fa.device_error(clear=True) == 0
    for old, new in zip(before, (c.k, c.v, c.ks, c.vs)):
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))


# ---------------------------------------------------------------------------------------- scores
@pytest.mark.parametrize("code,dt,gqa", [("int8", "bf16", 2), ("e4m3", "fp32", 1), ("int8", "fp32", 12), ("e4m3", "fp16", 16)])
@pytest.mark.parametrize("lens", [[300, 41], [3000, 130]])
def test_decode_alibi_over_long_contexts(code, dt, gqa, lens):
    """The usual slopes 2^-1 .. 2^-8: the first keys' scores lie hundreds below the last ones'."""
    c = Pool(5, lens, 8, 64, 16, 16, code)
    q = c.randn(2, 8 * gqa, 64).to(TDT[dt])
    slopes = (2.0 ** -(1.0 + torch.arange(8, device="cuda"))).repeat_interleave(gqa)
    check(decode(c, q, lens, [1, 1], alibi=slopes), exact(c, q, lens, [1, 1], alibi=slopes), dt)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("gqa", [1, 12])
@pytest.mark.parametrize("opt", [dict(), dict(window=0), dict(leftpad=[32, 40]), dict(window=3)])
def test_decode_scores_far_below_zero(code, gqa, opt):
    """Every visible score at about -120 .. -2000, in strips of many and of one visible key."""
    lens = [33, 41]
    c = Pool(6, lens, 2, 64, 16, 1, code)
    q = c.randn(2, 2 * gqa, 64)
    for z, n in enumerate(lens):      # each key the opposite of the first query of its head, at a size of its own
        for pos in range(n):
            x = -q[z, ::gqa].sign() * (100 if code == "int8" else 256)
            at = int(c.table[z, pos // 16]), pos % 16
            c.k[at] = x.to(CDT[code])
            c.ks[at[0], :, at[1]] = (5 + 2 * ((7 * pos + 11 * z) % 40)) / (100 if code == "int8" else 256)
    q[:, :] = q[:, ::gqa].repeat_interleave(gqa, 1)
    want = exact(c, q, lens, [1, 1], scale=1.0, **opt)
    assert float(want[1].max()) < -89
    check(decode(c, q, lens, [1, 1], scale=1.0, **opt), want, "fp32")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("gqa,dim", [(1, 128), (12, 128), (2, 64), (1, 256)])
@pytest.mark.parametrize("fall,rise", [(0, 0), (14, 20), (20, 30), (30, 60), (40, 60), (90, 300)])
def test_decode_value_scales_fall_while_scores_rise(code, gqa, dim, fall, rise):
    """A block whose V scale is 2^fall times the others' and whose scores lie `rise` (base 2) below: what it leaves behind must not
    cost the later weights a bit.  Each row to 1e-5."""
    lens = [1400, 1100]
    c = Pool(7, lens, 64, dim, 32, 16, code)
    per, stages = strips_a_warp(c, lens, [1, 1], gqa)
    assert per > stages
    q = c.randn(2, 64 * gqa, dim)
    slope = torch.zeros(64 * gqa, device="cuda")
    for z in range(2):
        every = c.blocks_of(z, lens[z])
        # the large block begins a stretch of a third of the sequence: whichever strips a warp takes, some hold it and smaller ones
        for i in range(0, len(every), 6):
            p, j = every[i]
            c.vs[p, :, j] *= 2.0 ** fall
    # scores rise with the position: rise over the 96 positions from one large block to the next
    slope += rise * math.log(2.0) / 96
    got, want = decode(c, q, lens, [1, 1], alibi=slope), exact(c, q, lens, [1, 1], alibi=slope)
    check(got, want, "fp32")
    err = (got[0].double() - want[0]).norm(dim=-1) / want[0].norm(dim=-1)
    assert float(err.max()) <= 1e-5, float(err.max())


@pytest.mark.parametrize("code,gqa,dim", [("int8", 1, 128), ("e4m3", 2, 64), ("int8", 12, 64), ("e4m3", 12, 128)])
@pytest.mark.parametrize("cap", [20.0, 30.0, 50.0])
@pytest.mark.parametrize("size", [3.0, 10.0])
def test_decode_softcap_in_fp32(code, gqa, dim, cap, size):
    """fp32 outputs under a softcap, several strips a warp.  The tanh is good to about 2^-24 of 1 (rms), which cap makes a relative
    error of a weight: 3e-6 at cap 50, with signs that differ from key to key; 1e-6 for the rest.  The bar is 5e-6."""
    lens = [1500, 1130]
    c = Pool(8, lens, 64, dim, 64, 16, code)
    per, stages = strips_a_warp(c, lens, [1, 1], gqa)
    assert per > stages
    q = c.randn(2, 64 * gqa, dim)
    k = c.values("k", 0, 1500)
    scale = size / float(torch.einsum("hgd,lhd->hgl", q[0].double().view(64, gqa, dim), k).square().mean().sqrt())
    check(decode(c, q, lens, [1, 1], softcap=cap, scale=scale), exact(c, q, lens, [1, 1], softcap=cap, scale=scale), "fp32", 5e-6)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("gqa", [2, 12])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_decode_nan_shows_with_and_without_softcap(code, gqa, softcap):
    """A NaN scale of K or of V, or a NaN in q, makes every row that sees it NaN, and no other."""
    lens = [70, 90]
    c = Pool(9, lens, 2, 128, 16, 16, code)
    q = c.randn(2, 1, 2 * gqa, 128)
    run = lambda: fa.flash_attn_with_kvcache_8bit(q, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, softcap=softcap)
    clean = run()
    p = int(c.table[1, 2])
    for t in (c.ks, c.vs):
        was = t[p, 1, 0].clone()
        t[p, 1, 0] = float("nan")
        got = run()
        assert torch.isnan(got[1, :, gqa:]).all()
        got[1, :, gqa:] = clean[1, :, gqa:]
        assert torch.equal(got, clean)
        t[p, 1, 0] = was
    q[0, 0, 1, 5] = float("nan")
    got = run()
    assert torch.isnan(got[0, 0, 1]).all()
    got[0, 0, 1] = clean[0, 0, 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
@pytest.mark.parametrize("news,cu", [([1, 1], [0, 1, 2]), ([3, 2], [2, 5, 7]), ([0, 0], [0, 0, 0]), ([0, 4], [1, 1, 5])])
def test_decode_rows_of_no_sequence_are_empty(dt, news, cu):
    """A padded batch: rows before cu_seqlens_q[0] and from cu_seqlens_q[-1] on give 0 and an LSE of -infinity."""
    lens, total = [40, 33], 12
    c = Pool(10, lens, 2, 80, 16, 8, "int8")
    q = c.randn(total, 6, 80).to(TDT[dt])
    for _ in range(2):   # what the allocator hands out holds something
        junk = [torch.full((total, 6, 80), 7.0, dtype=TDT[dt], device="cuda"), torch.full((6, total), 7.0, device="cuda")]
        del junk
        out, lse = fa.flash_attn_with_kvcache_8bit(q, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, cu_seqlens_q=i32(cu), max_seqlen_q=4,
                                                   return_softmax_lse=True)
    own = slice(cu[0], cu[-1])
    free = torch.ones(total, dtype=torch.bool, device="cuda")
    free[own] = False
    assert (out[free] == 0).all() and torch.isneginf(lse[:, free]).all()
    if cu[-1] > cu[0]:
        want = exact(c, q[own], lens, news)
        check((out[own], lse.t()[own]), want, dt)


def test_window_sizes_beyond_32_bits():
    c = Pool(11, [60], 2, 64, 16, 8, "int8")
    q = c.randn(1, 2, 4, 64)
    args = (q, c.k, c.v, c.ks, c.vs, i32([60]), c.bt)
    for big in (2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 40):
        assert torch.equal(fa.flash_attn_with_kvcache_8bit(*args, window_size=(big, 0)), fa.flash_attn_with_kvcache_8bit(*args))
        assert torch.equal(fa.flash_attn_with_kvcache_8bit(*args, causal=False, window_size=(-1, big)),
                           fa.flash_attn_with_kvcache_8bit(*args, causal=False))


# ---------------------------------------------------------------------------------------- warps with many strips
STRIPS = [
    # code, dtype, page, block, heads, gqa, dim, lens, news, options
    ("int8", "bf16", 256, 64, 64, 4, 128, [2500, 1], [1, 1], {}),
    ("e4m3", "bf16", 256, 64, 64, 4, 128, [2500, 1700], [1, 1], {}),
    ("int8", "fp32", 16, 16, 64, 1, 128, [1999, 2100], [1, 1], {}),
    ("e4m3", "fp32", 16, 1, 64, 2, 128, [1999, 2100], [1, 1], dict(window=900)),
    ("int8", "fp16", 4, 4, 64, 2, 128, [1301, 900], [1, 1], {}),
    ("e4m3", "fp16", 4, 1, 64, 2, 64, [2300, 1900], [1, 1], dict(leftpad=[70, 3])),
    ("int8", "fp32", 64, 16, 64, 12, 128, [1003, 700], [1, 1], {}),
    ("e4m3", "fp32", 64, 64, 64, 16, 128, [1003, 700], [1, 1], dict(softcap=30.0)),
    ("int8", "fp16", 16, 8, 64, 9, 64, [1003, 900], [1, 1], dict(window=333)),
    ("e4m3", "bf16", 256, 256, 64, 16, 64, [1600, 31], [1, 1], {}),
    ("int8", "fp32", 64, 8, 64, 1, 64, [3000, 2600], [1, 1], dict(alibi=True)),
    ("e4m3", "fp32", 256, 32, 64, 8, 64, [3000, 2600], [1, 1], {}),
    ("int8", "fp16", 16, 16, 64, 4, 256, [700, 650], [1, 1], {}),
    ("e4m3", "fp32", 64, 2, 64, 2, 192, [700, 650], [1, 1], dict(softcap=20.0)),
    ("int8", "fp32", 4, 2, 64, 2, 256, [500, 444], [1, 1], dict(alibi=True)),
    ("int8", "bf16", 64, 16, 64, 4, 128, [900, 1000], [3, 3], {}),
    ("e4m3", "fp16", 32, 16, 64, 4, 128, [1300, 0, 1], [4, 0, 1], dict(packed=True)),
    ("int8", "fp32", 32, 16, 64, 2, 96, [1300, 40, 700], [7, 1, 5], dict(packed=True, window=500, softcap=30.0)),
    ("e4m3", "fp32", 16, 8, 64, 2, 128, [900, 800], [2, 2], dict(causal=False)),
    ("int8", "fp16", 16, 16, 64, 1, 128, [33 + 11 * i for i in range(40)], [1] * 40, {}),
    ("e4m3", "fp16", 64, 16, 64, 12, 64, [33 + 11 * i for i in range(30)], [1] * 30, {}),
    ("int8", "fp32", 128, 32, 128, 1, 128, [3 * i for i in range(60)], [1] * 60, dict(alibi=True)),
]


@pytest.mark.parametrize("case", STRIPS, ids=lambda c: "-".join(map(str, (*c[:7], max(c[7]), max(c[8])))))
def test_decode_many_strips_a_warp(case):
    """So many heads and positions that every warp fills its ring again and again: the steady loop, the ring's later rounds,
    pages ahead, sequences written whole, warps that go on from one sequence to the next."""
    code, dt, page, block, heads, gqa, dim, lens, news, opt = case
    opt = dict(opt)
    c = Pool(12, lens, heads, dim, page, block, code)
    packed = opt.pop("packed", False)
    per, stages = strips_a_warp(c, lens, news, gqa, packed)
    assert per > stages, (per, stages)
    q = c.randn(sum(news), heads * gqa, dim).to(TDT[dt])
    if opt.pop("alibi", False):
        opt["alibi"] = torch.rand(heads * gqa, generator=c.gen, device="cuda") * 0.2
    check(decode(c, q, lens, news, packed, **opt), exact(c, q, lens, news, **opt), dt)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("gqa", [1, 12])
@pytest.mark.parametrize("way", [1, -1])
def test_decode_maxima_that_grow_or_shrink_along_a_warp(code, gqa, way):
    """K scales from 2^-6 to 2^6 along the positions, either way: the running maximum moves again and again within a warp."""
    lens = [1500, 1234]
    c = Pool(13, lens, 64, 128, 32, 32, code)
    per, stages = strips_a_warp(c, lens, [1, 1], gqa)
    assert per > stages
    for z in range(2):
        every = c.blocks_of(z, lens[z])
        for i, (p, j) in enumerate(every):
            c.ks[p, :, j] = 2.0 ** (way * (12.0 * i / len(every) - 6)) / QMAX[code]
    q = c.randn(2, 64 * gqa, 128)
    check(decode(c, q, lens, [1, 1]), exact(c, q, lens, [1, 1]), "fp32")


@pytest.mark.parametrize("code,gqa,dim", [("int8", 1, 128), ("e4m3", 2, 64), ("int8", 12, 64), ("e4m3", 4, 256)])
@pytest.mark.parametrize("cap", [30.0, 50.0, 1000.0])
@pytest.mark.parametrize("size", [1.0, 3.0])
def test_decode_softcap_far_above_the_scores(code, gqa, dim, cap, size):
    """Scores far below the cap are the tanh's near 0: a relative error of some 1.5e-7 (rms) of the tanh is as much of a score, 4.5e-7
    at scores of rms 3, beside 3e-7 of what a decode without softcap is off.  The bar is 1e-6, whatever the cap."""
    lens = [700, 530]
    c = Pool(14, lens, 64, dim, 64, 16, code)
    q = c.randn(2, 64 * gqa, dim)
    k = c.values("k", 0, 700)
    scale = size / float(torch.einsum("hgd,lhd->hgl", q[0].double().view(64, gqa, dim), k).square().mean().sqrt())
    check(decode(c, q, lens, [1, 1], softcap=cap, scale=scale), exact(c, q, lens, [1, 1], softcap=cap, scale=scale), "fp32", 1e-6)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("gqa", [1, 12])
@pytest.mark.parametrize("power", [-100, 100])
def test_decode_values_at_the_ends_of_their_range(code, gqa, power):
    """V up to 2^100 in size, and as small, in long sums whose maximum grows: finite, and each row to 1e-5."""
    lens = [1500, 1234]
    c = Pool(15, lens, 64, 128, 32, 32, code)
    c.vs.copy_(torch.full_like(c.vs, 2.0 ** power / QMAX[code]))
    for z in range(2):
        every = c.blocks_of(z, lens[z])
        for i, (p, j) in enumerate(every):
            c.ks[p, :, j] = 2.0 ** (6.0 * i / len(every) - 4) / QMAX[code]
    q = c.randn(2, 64 * gqa, 128)
    got, want = decode(c, q, lens, [1, 1]), exact(c, q, lens, [1, 1])
    assert torch.isfinite(got[0]).all()
    f = 2.0 ** -power                 # norms of such values are beyond fp32, and 2^-100 squared is
    err = (got[0].double() * f - want[0] * f).norm(dim=-1) / (want[0] * f).norm(dim=-1)
    assert float(err.max()) <= 1e-5, float(err.max())
