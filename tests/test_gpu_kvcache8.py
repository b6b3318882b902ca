"""Paged 8-bit caches on the GPU: kvcache_append, kvcache_gather, flash_attn_with_kvcache_8bit against a
64-bit restatement (tests/kv8_ref.py).

Tolerances.  Append, int8: a stored value is within half a scale of the rotated input, e4m3 within 2^-4 of it or half the
least step (2^-10 of a scale); fp32 rotation and division add a few 2^-24 of the block's largest value, i.e. of
Q scales: 1e-4 of a scale covers it.  Scales: amax / Q, relative 1e-6.  Gather: one rounding to the output type, plus
2^-23 for the fp32 product.  Attention: the framework's bars, rel_rms 3e-4 (fp16), 2.5e-3 (bf16), 1e-5 (fp32); LSE is fp32
whatever the type: 1e-5 relative to its rms, or 1e-5 absolute."""
import numpy as np
import pytest
import torch

import fable_attn as fa
import kv8_ref as R

pytestmark = pytest.mark.gpu
BAR = {"fp16": 3e-4, "bf16": 2.5e-3, "fp32": 1e-5}


def rel(a, b):
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


def tables(rows, half):
    ang = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(half) / half)
    c, s = torch.from_numpy(np.cos(ang)).float(), torch.from_numpy(np.sin(ang)).float()
    return c.cuda(), s.cuda(), R.f64(c), R.f64(s)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cum(v):
    return i32([0] + list(np.cumsum(v)))


# ---------------------------------------------------------------------------------------- append
def check_append(c, before, lens, news, k, v, args, half=0, inter=False, rot0=None, dt="bf16"):
    """What the cache holds after the call against the definition: new tokens, kept tokens, untouched slots."""
    cos, sin = args
    for which, rows in (("k", k), ("v", v)):
        held = c.values(which)
        old_codes, old_scale = before[which]
        new_codes = (c.k if which == "k" else c.v).view(torch.int8 if c.code in R.CDT else (c.k.dtype)).cpu()
        touched = np.zeros(c.n * c.page, bool)
        at = 0
        for z, (L, n) in enumerate(zip(lens, news)):
            x = np.stack([R.f64(rows[at + i]) for i in range(n)]) if n else np.zeros((0, c.heads, c.dim))
            at += n
            if which == "k" and half:
                x = np.stack([R.rotate(x[i], (L if rot0 is None else rot0[z]) + i, cos, sin, inter) for i in range(n)]) if n else x
            if c.code not in R.CDT:
                for i in range(n):
                    s = c.slot(z, L + i)
                    touched[s] = True
                    # one rounding; the rotation's own error is below 2^-22 of the row
                    lim = R.ULP[dt] * np.abs(x[i]) + 2.0 ** -22 * np.abs(x[i]).max() + 2.0 ** -25
                    assert (np.abs(held[s] - x[i]) <= lim).all()
                continue
            sc = c.ks if which == "k" else c.vs
            for b0 in range(L // c.block * c.block, L + n, c.block):
                a, e = max(L, b0), min(L + n, b0 + c.block)
                if a >= e:
                    continue
                s0 = c.slot(z, b0)
                pg, j = s0 // c.page, s0 % c.page // c.block
                got = R.f64(sc[pg, :, j])
                amax = np.abs(x[a - L:e - L]).max(axis=(0, 2))
                was = old_scale[pg, :, j] if a > b0 else np.zeros(c.heads)
                want = np.maximum(np.maximum(was, amax / R.QMAX[c.code]), R.MIN_SCALE)
                np.testing.assert_allclose(got, want, rtol=1e-6)
                for pos in range(b0, e):
                    s = c.slot(z, pos)
                    touched[s] = True
                    y = x[pos - L] if pos >= a else old_codes[s] * was[:, None]
                    step = got[:, None] / 2 if c.code == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, got[:, None] * 2.0 ** -10)
                    err = np.abs(held[s] - y)
                    assert (err <= step + 1e-4 * got[:, None]).all(), (which, z, pos, (err / got[:, None]).max())
                    if pos < a:   # kept as it was wherever the scale stayed
                        stay = got == was
                        np.testing.assert_array_equal(held[s][stay], (old_codes[s] * was[:, None])[stay])
        flat_new = R.f64(new_codes.view(c.k.dtype) if c.code in R.CDT else new_codes).reshape(-1, c.heads, c.dim)
        np.testing.assert_array_equal(flat_new[~touched], old_codes[~touched])


def snapshot(c):
    flat = lambda t: R.f64(t).reshape(-1, c.heads, c.dim)
    sc = lambda t: None if t is None else R.f64(t)
    return {"k": (flat(c.k), sc(c.ks)), "v": (flat(c.v), sc(c.vs))}


APPEND = [
    # code, dtype, page, block, heads, dim, lens, news, rotary half, interleaved
    ("int8", "bf16", 16, 16, 2, 128, [0, 5, 16, 31], [1, 1, 1, 1], 64, False),
    ("int8", "fp16", 32, 8, 3, 64, [0, 7, 33], [40, 1, 0], 32, True),
    ("e4m3", "bf16", 64, 64, 2, 128, [63, 64, 1, 130], [70, 2, 3, 129], 64, False),
    ("e4m3", "fp32", 16, 1, 1, 80, [3, 0], [18, 5], 20, False),
    ("int8", "fp32", 8, 4, 1, 16, [2, 9, 0], [1, 30, 3], 8, True),
    ("int8", "bf16", 256, 256, 1, 256, [200, 0], [300, 255], 128, False),
    ("e4m3", "fp16", 4, 2, 5, 96, [1, 2, 3], [9, 1, 6], 9, False),
    ("int8", "bf16", 1, 1, 2, 48, [0, 4], [3, 2], 24, True),
    ("e4m3", "bf16", 128, 32, 1, 192, [31, 95], [66, 2], 48, True),
    ("int8", "fp16", 16, 2, 4, 112, [0, 1, 6], [5, 2, 11], 0, False),
    ("bf16", "bf16", 16, 1, 2, 128, [0, 5, 40], [3, 1, 20], 64, False),
    ("fp16", "fp16", 8, 1, 3, 80, [7, 0], [2, 17], 10, True),
    ("fp32", "fp32", 32, 1, 1, 64, [30], [5], 32, False),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:6])))
def test_append(case):
    code, dt, page, block, heads, dim, lens, news, half, inter = case
    rng = np.random.default_rng(1)
    c = R.Cache(rng, len(lens), heads, dim, page, block, code, max(a + b for a, b in zip(lens, news)))
    tot = sum(news)
    k, v = (torch.from_numpy(rng.standard_normal((tot, heads, dim)) * 3).to("cuda", R.TDT[dt]) for _ in range(2))
    cos, sin, c64, s64 = tables(600, half) if half else (None,) * 4
    before = snapshot(c)
    fa.kvcache_append(k, v, c.k, c.v, i32(lens), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=cum(news), rotary_cos=cos,
                      rotary_sin=sin, rotary_interleaved=inter)
    check_append(c, before, lens, news, k, v, (c64, s64), half, inter, None, dt)


@pytest.mark.parametrize("code", ["int8", "e4m3", "bf16"])
def test_append_dense_strided_and_rotary_seqlens(code):
    """(batch, tokens) rows out of a packed projection (strided heads and rows), own rotary positions."""
    rng = np.random.default_rng(2)
    lens, n, heads, dim = [9, 0, 17], 5, 2, 64
    c = R.Cache(rng, 3, heads, dim, 16, 4 if code != "bf16" else 1, code, 30)
    qkv = torch.from_numpy(rng.standard_normal((3, n, 8, dim))).to("cuda", torch.bfloat16)
    k, v = qkv[:, :, 4:6], qkv[:, :, 6:8]
    cos, sin, c64, s64 = tables(64, 16)
    rot0 = [30, 2, 11]
    before = snapshot(c)
    fa.kvcache_append(k, v, c.k, c.v, i32(lens), c.bt, k_scale=c.ks, v_scale=c.vs, rotary_cos=cos, rotary_sin=sin,
                      rotary_interleaved=False, rotary_seqlens=i32(rot0))
    check_append(c, before, lens, [n] * 3, k.reshape(-1, heads, dim), v.reshape(-1, heads, dim), (c64, s64), 16, False, rot0)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("offset", [1, 3])
def test_append_unaligned_rows(code, offset):
    """Rows that start at odd elements and step by odd counts."""
    rng = np.random.default_rng(3)
    c = R.Cache(rng, 2, 2, 64, 16, 8, code, 40)
    wide = torch.from_numpy(rng.standard_normal((20, 2, 64 * 2 + 7))).to("cuda", torch.float16)
    k, v = wide[..., offset:offset + 64], wide[..., offset + 65:offset + 129]
    cos, sin, c64, s64 = tables(64, 32)
    before = snapshot(c)
    fa.kvcache_append(k, v, c.k, c.v, i32([3, 8]), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=i32([0, 9, 20]),
                      rotary_cos=cos, rotary_sin=sin, rotary_interleaved=False)
    check_append(c, before, [3, 8], [9, 11], k, v, (c64, s64), 32, False)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token_keeps_earlier_values(code):
    """One token at a time with growing values: each step puts the block on a larger scale.  A kept value has been
    rounded once per step, each time by at most half a step of the scale it then got."""
    rng = np.random.default_rng(4)
    c = R.Cache(rng, 1, 1, 32, 16, 16, code, 40)
    rows = [torch.from_numpy(rng.standard_normal((1, 1, 1, 32)) * 1.2 ** i).float().cuda() for i in range(20)]
    for i, x in enumerate(rows):
        fa.kvcache_append(x, -x, c.k, c.v, i32([i]), c.bt, k_scale=c.ks, v_scale=c.vs)
    held = c.values("k")
    for i, x in enumerate(rows):
        last = 15 if i < 16 else 19
        s = max(float(r.abs().max()) for r in rows[(0 if i < 16 else 16):last + 1]) / R.QMAX[code]
        y = R.f64(x)[0, 0, 0]
        lim = (last - i + 1) * (0.5 * s if code == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10)) * 1.1
        assert (np.abs(held[c.slot(0, i), 0] - y) <= lim).all()
    np.testing.assert_array_equal(c.values("v")[[c.slot(0, i) for i in range(20)]], -held[[c.slot(0, i) for i in range(20)]])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_nonfinite_is_carried_by_the_scale(code, bad):
    rng = np.random.default_rng(5)
    c = R.Cache(rng, 1, 2, 64, 16, 4, code, 40)
    k = torch.randn(8, 2, 64, device="cuda", dtype=torch.float16)
    k[5, 1, 7] = bad
    fa.kvcache_append(k, k.clone(), c.k, c.v, i32([0]), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=i32([0, 8]))
    got, _ = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 8]), 8, k_scale=c.ks, v_scale=c.vs, dtype=torch.float32)
    nan = torch.isnan(got)
    assert nan[4:8, 1].all() and not nan[:4].any() and not nan[4:8, 0].any()
    codes = c.k[c.table[0, 0]].float()
    assert torch.isfinite(codes[:8]).all()
    # the block is NaN until it is begun anew
    one = torch.randn(1, 1, 2, 64, device="cuda", dtype=torch.float16)
    fa.kvcache_append(one, one, c.k, c.v, i32([6]), c.bt, k_scale=c.ks, v_scale=c.vs)
    got, _ = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 8]), 8, k_scale=c.ks, v_scale=c.vs, dtype=torch.float32)
    assert torch.isnan(got[4:8, 1]).all()
    fa.kvcache_append(one, one, c.k, c.v, i32([4]), c.bt, k_scale=c.ks, v_scale=c.vs)
    got, _ = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 5]), 5, k_scale=c.ks, v_scale=c.vs, dtype=torch.float32)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_zeros_and_extremes(code):
    rng = np.random.default_rng(6)
    c = R.Cache(rng, 1, 1, 16, 16, 1, code, 10)
    k = torch.zeros(4, 1, 16, device="cuda")
    k[1] = 3.0e38
    k[2, 0, 3] = 1e-38
    k[3, 0, 5] = -2.0 ** -149
    fa.kvcache_append(k, k, c.k, c.v, i32([0]), c.bt, k_scale=c.ks, v_scale=c.vs, cu_seqlens_new=i32([0, 4]))
    got, _ = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 4]), 4, k_scale=c.ks, v_scale=c.vs, dtype=torch.float32)
    assert torch.isfinite(got).all() and (got[0] == 0).all()
    assert ((got[1] - 3.0e38).abs() <= 3.0e38 * 1e-6).all()


def test_append_outside_the_table_is_skipped_and_flagged():
    rng = np.random.default_rng(7)
    c = R.Cache(rng, 2, 1, 32, 16, 8, "int8", 40)
    bt = c.bt.clone()
    bt[0, 1] = c.n            # past the pool
    bt[1, 0] = -1
    cap = c.per * 16
    before = snapshot(c)
    k = torch.randn(2, 20, 1, 32, device="cuda")
    fa.device_error(clear=True)
    fa.kvcache_append(k, k, c.k, c.v, i32([cap - 4, 0]), bt, k_scale=c.ks, v_scale=c.vs)
    assert fa.device_error(clear=True) == 8192
    after = snapshot(c)
    ok = {c.slot(0, p) for p in range(cap - 4, cap)} | {c.slot(1, p) for p in range(16, 20)}
    keep = np.array([s not in ok for s in range(c.n * 16)])
    np.testing.assert_array_equal(after["k"][0][keep], before["k"][0][keep])
    cos, sin, _, _ = tables(8, 16)
    fa.kvcache_append(k[:, :1], k[:, :1], c.k, c.v, i32([8, 20]), c.bt, k_scale=c.ks, v_scale=c.vs, rotary_cos=cos, rotary_sin=sin)
    assert fa.device_error(clear=True) == 16384


# ---------------------------------------------------------------------------------------- gather
GATHER = [
    ("int8", "bf16", 16, 16, 2, 128, [5, 40, 1], [0, 3, 16]),
    ("e4m3", "fp16", 64, 64, 1, 64, [100, 0, 33], [0, 0, 31]),
    ("int8", "fp32", 32, 1, 3, 80, [50], [7]),
    ("e4m3", "bf16", 8, 2, 2, 256, [9, 20], [1, 2]),
    ("int8", "fp16", 1, 1, 1, 16, [3, 4], [2, 0]),
    ("bf16", "bf16", 16, 1, 2, 96, [20, 3], [1, 0]),
    ("fp16", "fp32", 4, 1, 1, 48, [11], [0]),
]


@pytest.mark.parametrize("case", GATHER, ids=lambda c: "-".join(map(str, c[:6])))
def test_gather(case):
    code, dt, page, block, heads, dim, counts, starts = case
    rng = np.random.default_rng(8)
    c = R.Cache(rng, len(counts), heads, dim, page, block, code, max(a + b for a, b in zip(counts, starts)))
    tot = sum(counts)
    got = fa.kvcache_gather(c.k, c.v, c.bt, cum(counts), tot, k_scale=c.ks, v_scale=c.vs, seq_starts=i32(starts), dtype=R.TDT[dt])
    for x, which in zip(got, "kv"):
        want = c.values(which)[[c.slot(z, starts[z] + i) for z, n in enumerate(counts) for i in range(n)]]
        assert x.shape == (tot, heads, dim) and x.dtype == R.TDT[dt]
        lim = (R.ULP[dt] + 2.0 ** -23) * np.abs(want) + 2.0 ** -24
        assert (np.abs(R.f64(x) - want) <= lim).all()


def test_gather_defaults_and_bad_pages():
    rng = np.random.default_rng(9)
    c = R.Cache(rng, 1, 1, 32, 16, 4, "e4m3", 40)
    k, v = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 20]), 20, k_scale=c.ks, v_scale=c.vs)
    assert k.dtype == torch.bfloat16
    want = c.values("v")[[c.slot(0, i) for i in range(20)]]
    assert (np.abs(R.f64(v) - want) <= 2.0 ** -8 * np.abs(want)).all()
    bt = c.bt.clone()
    bt[0, 0] = -7
    fa.device_error(clear=True)
    k, _ = fa.kvcache_gather(c.k, c.v, bt, i32([0, 20]), 20, k_scale=c.ks, v_scale=c.vs)
    assert fa.device_error(clear=True) == 8192
    assert (k[:16] == 0).all() and (k[16:] != 0).any()
    k, v = fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 0]), 0, k_scale=c.ks, v_scale=c.vs)
    assert k.shape == (0, 1, 32)


# ---------------------------------------------------------------------------------------- attention
def run_decode(c, q, lens, news, dt, packed, softcap=0.0, window=(-1, -1), causal=True, alibi=None, leftpad=None, half=0, inter=False,
               rot0=None, scale=None):
    cos, sin, c64, s64 = tables(max(max(lens), max(rot0 or [0]) + max(news)) + 8, half) if half else (None,) * 4
    hq, dim = q.shape[-2:]
    qq = q if packed else q.view(len(lens), news[0], hq, dim)
    out, lse = fa.flash_attn_with_kvcache_8bit(
        qq, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, softmax_scale=scale, causal=causal, window_size=window, softcap=softcap,
        alibi_slopes=None if alibi is None else alibi.cuda(), cu_seqlens_q=cum(news) if packed else None,
        max_seqlen_q=max(news) if packed else None, cache_leftpad=None if leftpad is None else i32(leftpad), rotary_cos=cos,
        rotary_sin=sin, rotary_interleaved=inter, rotary_seqlens=None if rot0 is None else i32(rot0), return_softmax_lse=True)
    assert out.shape == qq.shape and out.dtype == q.dtype
    lse = lse.cpu().double().numpy()
    lse = lse.T if packed else lse.transpose(0, 2, 1).reshape(-1, hq)
    kv, vv = c.values("k"), c.values("v")
    want, wl, at = [], [], 0
    for z, (L, n) in enumerate(zip(lens, news)):
        slots = [c.slot(z, j) if 0 <= int(c.table[z, j // c.page]) < c.n else -1 for j in range(L)]
        o, l = R.decode(R.f64(q[at:at + n]), kv, vv, slots, L, scale or dim ** -0.5, window[0], 0 if causal else window[1], softcap,
                        None if alibi is None else alibi.double().numpy(), 0 if leftpad is None else leftpad[z], c64, s64, inter,
                        None if rot0 is None else rot0[z])
        at += n
        want.append(o)
        wl.append(l)
    got = R.f64(out).reshape(-1, hq, dim)
    return got, np.concatenate(want), lse, np.concatenate(wl)


def check_decode(got, want, lse, wl, dt):
    dead = np.isneginf(wl)
    assert (np.isneginf(lse) == dead).all()
    assert (got[dead] == 0).all()
    if (~dead).any():
        assert rel(got[~dead], want[~dead]) <= BAR[dt], rel(got[~dead], want[~dead])
        err = np.abs(lse[~dead] - wl[~dead])
        assert err.max() <= 1e-5 * max(1.0, np.sqrt(np.mean(wl[~dead] ** 2))), err.max()


DECODE = [
    # code, dtype, page, block, hq, hk, dim, lens, news, options
    ("int8", "fp16", 16, 16, 8, 8, 64, [1], [1], {}),
    ("int8", "bf16", 16, 16, 8, 2, 128, [300, 1, 17, 128], [1] * 4, dict(half=64)),
    ("e4m3", "bf16", 256, 64, 8, 2, 128, [700, 33, 256], [1] * 3, dict(half=32, inter=True)),
    ("e4m3", "fp16", 32, 1, 4, 4, 96, [70, 31, 2], [1] * 3, {}),
    ("int8", "fp32", 16, 4, 6, 2, 80, [90, 15], [1, 1], dict(half=20)),
    ("e4m3", "fp32", 64, 32, 16, 1, 64, [200, 64], [1, 1], dict(softcap=20.0)),
    ("int8", "fp16", 8, 8, 7, 1, 48, [61, 7, 8], [1] * 3, dict(alibi=True)),
    ("int8", "bf16", 1, 1, 4, 2, 32, [20, 5], [1, 1], {}),
    ("e4m3", "bf16", 4, 2, 32, 2, 192, [50, 3], [1, 1], dict(half=96)),
    ("int8", "fp16", 128, 32, 16, 2, 256, [400, 129], [1, 1], dict(half=64)),
    ("int8", "fp16", 16, 16, 16, 1, 128, [130, 64], [1, 1], dict(half=64)),
    ("e4m3", "fp16", 16, 2, 40, 2, 128, [130, 16], [1, 1], {}),
    ("int8", "bf16", 32, 32, 8, 2, 128, [200, 50, 9], [3] * 3, dict(half=64)),
    ("e4m3", "fp16", 32, 16, 8, 1, 64, [200, 50, 9, 64], [1, 4, 0, 7], dict(packed=True, half=32)),
    ("int8", "fp32", 16, 8, 4, 4, 112, [70, 20, 33], [5, 2, 9], dict(packed=True, window=(10, -1))),
    ("int8", "fp16", 64, 16, 8, 4, 128, [300, 90, 64], [2] * 3, dict(window=(64, 0), softcap=30.0)),
    ("e4m3", "bf16", 16, 16, 4, 2, 128, [100, 40], [4, 4], dict(causal=False)),
    ("int8", "bf16", 16, 16, 4, 2, 64, [100, 40], [4, 4], dict(causal=False, window=(20, 1))),
    ("int8", "fp16", 16, 16, 4, 2, 128, [100, 40, 30], [1, 1, 1], dict(leftpad=[20, 40, 29])),
    ("int8", "bf16", 16, 16, 4, 2, 128, [0, 2, 0], [1, 4, 2], dict(packed=True)),
    ("e4m3", "fp16", 16, 8, 4, 1, 128, [40, 25], [2, 1], dict(packed=True, half=64, rot0=[3, 50], inter=True, alibi=True)),
    ("int8", "fp16", 256, 128, 12, 4, 128, [1500], [1], dict(half=64, scale=0.5)),
    ("int8", "bf16", 128, 256 // 2, 64, 8, 128, [3000, 10], [1, 1], {}),
    ("e4m3", "fp16", 16, 16, 2, 2, 16, [33, 100], [33, 40], dict(packed=True)),
    ("int8", "fp16", 32, 16, 24, 2, 64, [64, 200], [10, 2], dict(packed=True, softcap=10.0, half=16)),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c[:9])).replace(" ", ""))
def test_decode(case):
    code, dt, page, block, hq, hk, dim, lens, news, opt = case
    opt = dict(opt)
    rng = np.random.default_rng(10)
    c = R.Cache(rng, len(lens), hk, dim, page, block, code, max(lens) + 1)
    q = torch.from_numpy(rng.standard_normal((sum(news), hq, dim))).to("cuda", R.TDT[dt])
    if opt.pop("alibi", False):
        opt["alibi"] = torch.from_numpy(rng.random(hq) * 0.3).float()
    packed = opt.pop("packed", False)
    check_decode(*run_decode(c, q, lens, news, dt, packed, **opt), dt)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("hq", [4, 16])
def test_decode_scales_of_every_size(code, hq):
    """Block scales over 2^-60 .. 2^60, so that the weights' range is far outside any 16-bit type's."""
    rng = np.random.default_rng(11)
    c = R.Cache(rng, 2, 1, 128, 16, 4, code, 100)
    c.vs.copy_(torch.from_numpy(2.0 ** rng.integers(-60, 61, tuple(c.vs.shape))).float())
    q = torch.from_numpy(rng.standard_normal((2, hq, 128))).to("cuda", torch.float32)
    got, want, lse, wl = run_decode(c, q, [100, 37], [1, 1], "fp32", False)
    # per row: a dominating block must come out to fp32 grade whatever the others are
    for r in range(2):
        for h in range(hq):
            assert rel(got[r, h], want[r, h]) <= 1e-5
    check_decode(got, want, lse, wl, "fp32")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_decode_large_and_small_scores(code):
    """K scales that make the scores run from hundreds to nothing: growing maxima along the keys."""
    rng = np.random.default_rng(12)
    c = R.Cache(rng, 2, 2, 64, 16, 16, code, 320)
    for z in range(2):
        for b in range(20):
            c.ks[int(c.table[z, b])] = (2.0 ** (b - 12) if z == 0 else 2.0 ** (6 - b)) / R.QMAX[code]
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).to("cuda", torch.float32)
    got, want, lse, wl = run_decode(c, q, [320, 309], [1, 1], "fp32", False)
    check_decode(got, want, lse, wl, "fp32")


@pytest.mark.parametrize("hq,dim", [(4, 256), (8, 128), (16, 128), (16, 64)])
def test_decode_sums_of_the_largest_codes(hq, dim):
    """Every code at an end of int8 and every |q| just below a power of two: the largest sums that a score can need.
    Scores stay within 4, each good to a few units of 2^-23 of that: far below the fp32 bar of 1e-5."""
    rng = np.random.default_rng(31)
    c = R.Cache(rng, 1, 1, dim, 16, 16, "int8", 200)
    ends = torch.from_numpy(rng.choice(np.array([-128, 127]), (c.n, 16, 1, 1))).to(torch.int8)
    c.k.copy_(ends.expand(-1, -1, 1, dim))
    c.ks.copy_(torch.from_numpy(rng.uniform(1, 4, tuple(c.ks.shape))).float())
    q = np.full((1, hq, dim), np.nextafter(np.float32(2), np.float32(0)))
    q[0, 1] *= -1
    q[0, 2:] *= rng.choice([-1, 1], (hq - 2, dim))
    got, want, lse, wl = run_decode(c, torch.from_numpy(q).to("cuda", torch.float32), [200], [1], "fp32", False, scale=1 / (256 * dim))
    check_decode(got, want, lse, wl, "fp32")


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("hq", [4, 16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_decode_nonfinite_q_stays_in_its_row(code, hq, bad):
    rng = np.random.default_rng(32)
    c = R.Cache(rng, 2, 1, 128, 16, 16, code, 100)
    q = torch.from_numpy(rng.standard_normal((2, 1, hq, 128))).to("cuda", torch.float32)
    args = (c.k, c.v, c.ks, c.vs, i32([100, 37]), c.bt)
    clean = fa.flash_attn_with_kvcache_8bit(q, *args)
    q[1, 0, 2, 77] = bad
    got = fa.flash_attn_with_kvcache_8bit(q, *args)
    assert torch.isnan(got[1, 0, 2]).all()
    got[1, 0, 2] = clean[1, 0, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("hq", [2, 12])
def test_decode_hidden_places_may_hold_anything(code, hq):
    """Slots past the lengths, before the pad, outside the window and in unused pages: NaN scales, NaN codes; among the
    new tokens a NaN block that only later rows see."""
    rng = np.random.default_rng(13)
    lens, news = [37, 70], [3, 2]
    c = R.Cache(rng, 2, 1, 64, 16, 1, code, 80)
    used = np.zeros(c.n * 16, bool)
    for z, (L, n) in enumerate(zip(lens, news)):
        for p in range(max(5, L - n - 20), L):
            used[c.slot(z, p)] = True
    hidden = torch.from_numpy(~used).cuda().view(c.n, 16)
    want_args = (c, torch.from_numpy(rng.standard_normal((5, hq, 64))).to("cuda", torch.float16), lens, news, "fp16", True)
    got0 = run_decode(*want_args, window=(20, 0), leftpad=[5, 5])
    check_decode(*got0, "fp16")
    for s in (c.ks, c.vs):
        s.masked_fill_(hidden[:, None], float("nan"))
    if code == "e4m3":
        for t in (c.k, c.v):
            t.view(torch.uint8).masked_fill_(hidden[:, :, None, None], 0x7f)
    qq = want_args[1]
    out = fa.flash_attn_with_kvcache_8bit(qq, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, cu_seqlens_q=cum(news), max_seqlen_q=3,
                                          window_size=(20, 0), cache_leftpad=i32([5, 5]))
    np.testing.assert_array_equal(R.f64(out), got0[0])
    # the last token of sequence 0 is NaN: only its own row sees it
    s = c.slot(0, 36)
    c.vs[s // 16, :, s % 16] = float("nan")
    c.ks[s // 16, :, s % 16] = float("nan")
    out = fa.flash_attn_with_kvcache_8bit(qq, c.k, c.v, c.ks, c.vs, i32(lens), c.bt, cu_seqlens_q=cum(news), max_seqlen_q=3,
                                          window_size=(20, 0), cache_leftpad=i32([5, 5]))
    assert torch.isnan(out[2]).all()
    keep = [0, 1, 3, 4]
    np.testing.assert_array_equal(R.f64(out)[keep], got0[0][keep])


def test_decode_bad_pages_read_as_empty():
    rng = np.random.default_rng(14)
    c = R.Cache(rng, 2, 2, 128, 16, 16, "int8", 100)
    c.table[0, 2], c.table[1, 0] = -1, c.n + 5
    c.bt = c.table.cuda()
    q = torch.from_numpy(rng.standard_normal((2, 4, 128))).to("cuda", torch.float16)
    fa.device_error(clear=True)
    r = run_decode(c, q, [90, 70], [1, 1], "fp16", False)
    assert fa.device_error(clear=True) == 8192
    check_decode(*r, "fp16")
    cos, sin, _, _ = tables(8, 32)
    fa.flash_attn_with_kvcache_8bit(q.view(2, 1, 4, 128), c.k, c.v, c.ks, c.vs, i32([17, 4]), c.bt, rotary_cos=cos, rotary_sin=sin)
    assert fa.device_error(clear=True) & 16384


def test_decode_strided_q_and_empty_calls():
    rng = np.random.default_rng(15)
    c = R.Cache(rng, 2, 2, 64, 16, 8, "int8", 60)
    wide = torch.from_numpy(rng.standard_normal((2, 12, 3 * 64 + 5))).to("cuda", torch.bfloat16)
    for q in (wide[:, :8, 64:128], wide[:, 1:9, 3:67]):
        r = run_decode(c, q.contiguous(), [55, 20], [1, 1], "bf16", True)
        check_decode(*r, "bf16")
        out = fa.flash_attn_with_kvcache_8bit(q, c.k, c.v, c.ks, c.vs, i32([55, 20]), c.bt, cu_seqlens_q=i32([0, 1, 2]), max_seqlen_q=1)
        np.testing.assert_array_equal(R.f64(out), r[0])
    none = fa.flash_attn_with_kvcache_8bit(wide[:0, :8, :64], c.k, c.v, c.ks, c.vs, i32([55, 20]), c.bt, cu_seqlens_q=i32([0, 0, 0]),
                                           max_seqlen_q=1)
    assert none.shape == (0, 8, 64)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_decode_many_sequences_of_unlike_lengths(code):
    """More groups than workers, and one sequence far longer than the rest: whole and split contexts side by side."""
    rng = np.random.default_rng(16)
    lens = [int(x) for x in rng.integers(1, 60, 180)]
    lens[77], lens[3] = 9001, 0
    c = R.Cache(rng, 1, 1, 16, 16, 16, code, 9001 + 180 * 64)
    # one pool, each sequence its own run of pages
    flat, per, at, rows = c.table.view(-1), (9001 + 15) // 16, 0, []
    for L in lens:
        n = (L + 15) // 16
        rows.append(torch.cat([flat[at:at + n], torch.zeros(per - n, dtype=torch.int32)]))
        at += n
    c.table = torch.stack(rows)
    c.bt, c.per = c.table.cuda(), per
    q = torch.from_numpy(rng.standard_normal((180, 8, 16))).to("cuda", torch.float16)
    check_decode(*run_decode(c, q, lens, [1] * 180, "fp16", False), "fp16")


def test_repeatable_on_another_stream_and_captured():
    """Same bits on every call, on a side stream, and from a replayed graph whose lengths change on the device; no
    host synchronisation in any of the three calls."""
    rng = np.random.default_rng(17)
    c = R.Cache(rng, 3, 2, 128, 16, 16, "int8", 900)
    q = torch.from_numpy(rng.standard_normal((3, 1, 8, 128))).to("cuda", torch.bfloat16)
    k = torch.from_numpy(rng.standard_normal((3, 1, 2, 128))).to("cuda", torch.bfloat16)
    lens = i32([850, 33, 400])
    torch.cuda.set_sync_debug_mode("error")
    try:
        def step():
            fa.kvcache_append(k, k, c.k, c.v, lens, c.bt, k_scale=c.ks, v_scale=c.vs)
            return fa.flash_attn_with_kvcache_8bit(q, c.k, c.v, c.ks, c.vs, lens + 1, c.bt, return_softmax_lse=True)
        step()
        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step()
            g = torch.cuda.CUDAGraph()
        torch.cuda.current_stream().wait_stream(side)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    with torch.cuda.graph(g):
        third = step()
    for new in ([850, 33, 400], [100, 700, 0]):
        lens.copy_(i32(new))
        g.replay()
        torch.cuda.synchronize()
        again = step()
        for a, b in zip(third, again):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------- refusals
def test_refusals():
    c = R.Cache(np.random.default_rng(18), 2, 2, 64, 16, 8, "int8", 40)
    q = torch.zeros(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = q[:, :, :2]
    lens = i32([3, 4])
    attend = lambda q=q, kc=c.k, vc=c.v, ks=c.ks, vs=c.vs, lens=lens, bt=c.bt, **kw: fa.flash_attn_with_kvcache_8bit(
        q, kc, vc, ks, vs, lens, bt, **kw)
    append = lambda k=k, v=k, kc=c.k, vc=c.v, lens=lens, bt=c.bt, ks=c.ks, vs=c.vs, **kw: fa.kvcache_append(
        k, v, kc, vc, lens, bt, k_scale=ks, v_scale=vs, **kw)
    for call in (
            lambda: attend(q=q[..., :48]), lambda: attend(q=q[:1]), lambda: attend(q=torch.cat([q, q[:, :, :1]], 2)),
            lambda: attend(q=q[:, 0]), lambda: attend(q=q[:, 0], cu_seqlens_q=i32([0, 2])), lambda: attend(lens=lens.float()),
            lambda: attend(lens=i32([1])), lambda: attend(bt=c.bt[0]), lambda: attend(ks=c.ks.double()), lambda: attend(ks=c.ks[:, :, :1]),
            lambda: attend(ks=c.ks.transpose(1, 2)), lambda: attend(kc=c.k[:, ::2]), lambda: attend(vc=c.v[:-1]), lambda: attend(q=q.cpu()),
            lambda: attend(q=q.double()), lambda: attend(alibi_slopes=torch.ones(3, device="cuda")),
            lambda: attend(cache_leftpad=i32([1])), lambda: attend(rotary_seqlens=i32([1])),
            lambda: attend(rotary_cos=torch.ones(8, 16, device="cuda")),
            lambda: attend(rotary_cos=torch.ones(8, 64, device="cuda"), rotary_sin=torch.ones(8, 64, device="cuda")),
            lambda: append(k=k[..., :32]), lambda: append(v=k.float()), lambda: append(k=k[:1], v=k[:1]), lambda: append(ks=None),
            lambda: append(ks=None, vs=None), lambda: append(cu_seqlens_new=i32([0, 1, 2])), lambda: append(lens=i32([1, 2, 3])),
            lambda: append(kc=c.k.bfloat16(), vc=c.v.bfloat16()), lambda: append(kc=c.k.half(), vc=c.v.half(), ks=None, vs=None),
            lambda: fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 1]), 1, k_scale=c.ks, v_scale=c.vs),
            lambda: fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 1, 2]), -2, k_scale=c.ks, v_scale=c.vs),
            lambda: fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 1, 2]), 2, k_scale=c.ks, v_scale=c.vs, seq_starts=i32([0])),
            lambda: fa.kvcache_gather(c.k, c.v, c.bt, i32([0, 1, 2]), 2, k_scale=c.ks, v_scale=c.vs, dtype=torch.float64)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):   # headdim not a multiple of 16
        z = torch.zeros(4, 16, 2, 72, device="cuda", dtype=torch.int8)
        attend(q=torch.zeros(2, 1, 4, 72, device="cuda"), kc=z, vc=z, ks=c.ks[:4], vs=c.vs[:4])
