"""Rotary of q and k at their tokens' own positions, against 64-bit arithmetic.

Bounds: x' = factor (x cos - y sin).  cos and sin in fp32 are off by at most 4 units of 2^-24 (the angle within an eighth of a
turn is rounded once, sincospi is good to 1.5 units, the factor's product rounds once more), the frequency is rounded in fp64 (2^-52 of the angle in turns,
times the position), the two products and the sum round in 2^-24 each; then half a step of the type."""
import math

import pytest
import torch

import fable_attn as fa
from fable_attn.layers.rotary import apply_rotary_emb_qk, rotary_tables, scaled_inv_freq

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def turned(x, pos, freq, interleaved, factor, back=False):
    """(value, size of its terms), fp64."""
    x = x.detach().double().cpu()
    r = 2 * len(freq)
    ang = pos.cpu().double()[..., None, None] * freq.cpu().double()
    c, s = ang.cos() * factor, ang.sin() * factor * (-1 if back else 1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    put = lambda p, q: torch.cat((torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1), x[..., r:]), -1)
    size = factor * (a.abs() + b.abs())
    return put(a * c - b * s, b * c + a * s), put(size, size) - 0


def close(got, ref, freq, far):
    want, amp = ref
    r = 2 * len(freq)
    amp = amp.clone()
    amp[..., r:] = 0
    u = U[got.dtype]
    rel = 8 * 2.0 ** -24 + far * float(freq.max()) * 2.0 ** -51
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -130
    off = (got.detach().double().cpu() - want).abs()
    assert (off <= u * want.abs() + rel * amp + tiny).all(), float((off / (u * want.abs() + rel * amp + tiny)).max())
    assert torch.equal(got.detach()[..., r:].double().cpu(), want[..., r:])


CASES = [(2, 7, 4, 2, 128, 128, False), (2, 7, 4, 2, 128, 128, True), (1, 1, 8, 8, 64, 32, False), (3, 33, 3, 1, 80, 80, True),
         (2, 5, 2, 2, 72, 10, False), (2, 5, 2, 2, 72, 10, True), (1, 9, 1, 1, 256, 256, False), (1, 700, 4, 1, 64, 64, True),
         (5, 300, 6, 2, 64, 64, False), (1, 3, 2, 1, 7, 6, False), (1, 3, 2, 1, 7, 6, True), (40, 40, 2, 2, 32, 2, True)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("b,n,hq,hk,d,r,inter", CASES)
def test_values_and_gradients(dt, b, n, hq, hk, d, r, inter):
    dt, far = DT[dt], 1 << 20
    freq, factor = scaled_inv_freq(r, scaling="yarn", factor=8.0, original_max_position=2048, device="cuda")
    pos = torch.randint(0, far, (b, n), generator=torch.Generator().manual_seed(1)).cuda()
    q, k = rand(1, b, n, hq, d, dtype=dt).requires_grad_(), rand(2, b, n, hk, d, dtype=dt).requires_grad_()
    dq, dk = rand(3, b, n, hq, d, dtype=dt), rand(4, b, n, hk, d, dtype=dt)
    out = apply_rotary_emb_qk(q, k, freq, pos.int(), interleaved=inter, factor=factor)
    grads = torch.autograd.grad(out, (q, k), (dq, dk))
    for x, y in zip(out, (q, k)):
        close(x, turned(y, pos, freq, inter, factor), freq, far)
    for x, y in zip(grads, (dq, dk)):
        close(x, turned(y, pos, freq, inter, factor, True), freq, far)
    wide = apply_rotary_emb_qk(q.detach(), k.detach(), freq, pos, interleaved=inter, factor=factor)
    assert all(torch.equal(x, y) for x, y in zip(out, wide))


@pytest.mark.parametrize("inter", [False, True])
def test_far_and_negative_positions(inter):
    freq, _ = scaled_inv_freq(64, base=500000.0, device="cuda")
    pos = torch.tensor([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789, 2 ** 40 + 12345, -2 ** 33]]).cuda()
    q, k = rand(1, 1, 8, 2, 64), rand(2, 1, 8, 1, 64)
    got = apply_rotary_emb_qk(q, k, freq, pos, interleaved=inter)
    for i in range(8):
        p = pos[:, i:i + 1]
        # fp64's own product is off by 2^-53 of the angle: counted in `far`
        for x, y in zip(got, (q, k)):
            close(x[:, i:i + 1], turned(y[:, i:i + 1], p, freq, inter, 1.0), freq, float(p.abs().max()))
    narrow = apply_rotary_emb_qk(q[:, :6], k[:, :6], freq, pos[:, :6].int(), interleaved=inter)
    assert all(torch.equal(x, y[:, :6]) for x, y in zip(narrow, got))


@pytest.mark.parametrize("n", [1, 40])
def test_offsets_packed_and_in_place(n):
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k = rand(1, 3, n, 4, 64, dtype=torch.bfloat16), rand(2, 3, n, 2, 64, dtype=torch.bfloat16)
    offs = torch.tensor([5, 0, 70000], dtype=torch.int32).cuda()
    pos = offs[:, None] + torch.arange(n, device="cuda", dtype=torch.int32)
    want = apply_rotary_emb_qk(q, k, freq, pos)
    same = lambda a, b: all(torch.equal(x.reshape(y.shape), y) for x, y in zip(a, b))
    assert same(apply_rotary_emb_qk(q, k, freq, seqlen_offsets=offs), want)
    assert same(apply_rotary_emb_qk(q[2:], k[2:], freq, seqlen_offsets=70000), [x[2:] for x in want])
    assert same(apply_rotary_emb_qk(q.flatten(0, 1), k.flatten(0, 1), freq, pos.flatten()), want)
    leaf = q.clone().requires_grad_()
    got = torch.autograd.grad(apply_rotary_emb_qk(leaf, k, freq, seqlen_offsets=offs)[0], leaf, q)[0]
    assert torch.equal(got, apply_rotary_emb_qk(q, k, freq, -pos)[0])
    qkv = torch.cat((q, k, k), 2)                     # slices of one projection, written in place
    a, b = qkv[:, :, :4], qkv[:, :, 4:6]
    ret = apply_rotary_emb_qk(a, b, freq, pos, inplace=True)
    assert ret[0] is a and same((a, b), want) and torch.equal(qkv[:, :, 6:], k)


def test_strides_and_shared_heads():
    freq, _ = scaled_inv_freq(32, device="cuda")
    q, k = rand(1, 4, 6, 4, 64, dtype=torch.float16), rand(2, 4, 6, 1, 64, dtype=torch.float16)
    pos = torch.arange(24, device="cuda").view(4, 6)
    want = apply_rotary_emb_qk(q, k, freq, pos)
    for f in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
              lambda x: torch.cat((x, x), -1)[..., :64], lambda x: torch.cat((x[..., :1], x), -1)[..., 1:],
              lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)):
        for got, w in zip(apply_rotary_emb_qk(f(q), f(k), freq, pos), want):
            assert torch.equal(got, w)
    wide = apply_rotary_emb_qk(q, k.expand(4, 6, 4, 64), freq, pos)[1]
    assert torch.equal(wide, want[1].expand_as(wide))
    flip = pos.t().contiguous().t()
    assert torch.equal(apply_rotary_emb_qk(q, k, freq, flip)[0], want[0])
    assert apply_rotary_emb_qk(q[:, :0], k[:, :0], freq, pos[:, :0])[0].shape == (4, 0, 4, 64)


def test_tables_serve_the_cache_alike():
    """kvcache_append over rotary_tables writes what apply_rotary_emb_qk gives, within half a step and the tables' roundings."""
    freq, factor = scaled_inv_freq(64, scaling="yarn", factor=4.0, original_max_position=64, device="cuda")
    cos, sin = rotary_tables(freq, 300, factor)
    q, k = rand(1, 2, 3, 2, 64), rand(2, 2, 3, 2, 64)
    lens = torch.tensor([250, 3], dtype=torch.int32).cuda()
    kc, vc = (torch.zeros(20, 16, 2, 64, device="cuda") for _ in range(2))
    # two sequences of up to 10 pages... each needs ceil(253 / 16) = 16 and 1
    table = torch.cat((torch.arange(16), torch.arange(16, 20), torch.zeros(12))).int().view(2, 16).cuda()
    fa.kvcache_append(k, k, kc, vc, lens, table, rotary_cos=cos, rotary_sin=sin, rotary_interleaved=False)
    want = apply_rotary_emb_qk(q, k, freq, seqlen_offsets=lens, factor=factor)[1]
    for z, start in enumerate((250, 3)):
        for i in range(3):
            p = start + i
            got = kc[int(table[z, p // 16]), p % 16]
            assert float((got - want[z, i]).abs().max()) <= 16 * 2.0 ** -24 * factor * 2 * float(k.abs().max())


def test_captured_and_on_another_stream():
    freq, _ = scaled_inv_freq(128, device="cuda")
    q, k = rand(1, 4, 1, 8, 128, dtype=torch.bfloat16), rand(2, 4, 1, 2, 128, dtype=torch.bfloat16)
    pos = torch.arange(4, device="cuda")[:, None].int()
    apply_rotary_emb_qk(q, k, freq, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary_emb_qk(q, k, freq, pos)
    pos.add_(1000)
    graph.replay()
    want = apply_rotary_emb_qk(q, k, freq, pos)
    assert all(torch.equal(x, y) for x, y in zip(out, want))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.zeros(64 << 20, device="cuda")
        pos.add_(1)
        got = apply_rotary_emb_qk(q, k, freq, pos)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, apply_rotary_emb_qk(q, k, freq, pos)))


def test_non_finite_values_stay_in_their_pair():
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k = rand(1, 1, 2, 2, 64, dtype=torch.bfloat16), rand(2, 1, 2, 1, 64, dtype=torch.bfloat16)
    pos = torch.tensor([[3, 4]]).cuda()
    want = apply_rotary_emb_qk(q, k, freq, pos)[0]
    q[0, 1, 0, 5] = float("inf")
    got = apply_rotary_emb_qk(q, k, freq, pos)[0]
    fine = torch.ones_like(got, dtype=torch.bool)
    fine[0, 1, 0, [5, 37]] = False
    assert torch.equal(got[fine], want[fine]) and not got[~fine].isfinite().any()


def test_saved_for_a_gradient_and_then_turned_in_place():
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k, w = rand(1, 2, 3, 4, 64), rand(2, 2, 3, 2, 64), torch.ones(64, device="cuda", requires_grad=True)
    for x in (q, k):
        y = (x * w).sum()
        apply_rotary_emb_qk(q, k, freq, inplace=True)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():
        q, k = q.clone(), k.clone()
        before = q.clone()
        apply_rotary_emb_qk(q, k, freq, seqlen_offsets=1, inplace=True)
        assert not torch.equal(before, q)


@pytest.mark.parametrize("bad", ["cpu", "types", "heads", "freq", "freq_grad", "pos", "pos_float", "both", "inplace_grad", "overlap", "same", "rank", "dims"])
def test_refusals(bad):
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k, pos, kw = rand(1, 2, 3, 4, 64), rand(2, 2, 3, 2, 64), torch.zeros(2, 3, dtype=torch.int32).cuda(), {}
    err = (ValueError, RuntimeError, NotImplementedError)
    if bad == "cpu": k = k.cpu()
    if bad == "types": k = k.half()
    if bad == "heads": k = k[:1]
    if bad == "freq": freq = torch.ones(33, device="cuda")
    if bad == "freq_grad": freq = freq.requires_grad_()
    if bad == "pos": pos = pos[0]
    if bad == "pos_float": pos = pos.float()
    if bad == "both": kw["seqlen_offsets"] = 3
    if bad == "inplace_grad": q, kw["inplace"] = q.requires_grad_(), True
    if bad == "overlap": k, kw["inplace"] = k[:, :, :1].expand(2, 3, 4, 64), True
    if bad == "same": q, kw["inplace"] = k, True
    if bad == "rank": q, k = q[0, 0], k[0, 0]
    if bad == "dims": k = k[..., :32]
    with pytest.raises(err):
        apply_rotary_emb_qk(q, k, freq, pos, **kw)
