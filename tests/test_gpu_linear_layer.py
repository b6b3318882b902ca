"""Rotary positions and linear attention together, as a layer trains and serves, against the 64-bit formulas; and the example."""
import importlib.util
import os

import pytest
import torch

import fable_attn as fa
import lin_ref as R
from fable_attn.layers.rotary import apply_rotary_emb_qk, rotary_tables, scaled_inv_freq

pytestmark = pytest.mark.gpu


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def turned64(x, pos, freq, factor, back=False):
    x, ang = x.detach().double().cpu(), pos.cpu().double()[:, None, None] * freq.cpu()
    c, s = ang.cos() * factor, ang.sin() * factor * (-1 if back else 1)
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 2)])
def test_training_step_in_fp32(hq, hk):
    """In fp32 nothing is rounded between the two operators but to 2^-24, so the chain's bound is the sum of its parts': turned values of size up to
    |x| + |y| per pair carry 8 roundings each way, which the terms' sizes below (every factor replaced by the pair's largest) cover."""
    n, d = 200, 64
    freq, factor = scaled_inv_freq(d, scaling="yarn", factor=4.0, original_max_position=1024, device="cuda")
    pos = torch.arange(5000, 5000 + n, device="cuda")
    q, k, v = rand(0, n, hq, d).requires_grad_(), rand(1, n, hk, d).requires_grad_(), rand(2, n, hk, d).requires_grad_()
    do, g = rand(3, n, hq, d), torch.linspace(-0.3, -0.001, hk).cuda()
    qr, kr = apply_rotary_emb_qk(q, k, freq, pos, factor=factor)
    out = fa.linear_attn_varlen_func(qr, kr, v, g, torch.tensor([0, n], dtype=torch.int32).cuda(), n)
    grads = torch.autograd.grad(out, (q, k, v), do)
    q64, k64 = turned64(q, pos, freq, factor), turned64(k, pos, freq, factor)
    o, _, dq, dk, dv, _ = R.one(q64, k64, v.detach().double().cpu(), g.double().cpu(), d ** -0.5, None, do.double().cpu())
    want = (o, turned64(dq, pos, freq, factor, True), turned64(dk, pos, freq, factor, True), dv)
    wide = lambda x: factor * torch.cat([sum(p.abs() for p in x.detach().double().cpu().chunk(2, -1))] * 2, -1)
    amp = R.one(wide(q), wide(k), v.detach().double().cpu().abs(), g.double().cpu(), d ** -0.5, None, do.double().cpu().abs())
    sizes = (amp[0], wide(amp[2]), wide(amp[3]), amp[4])
    rel = (n * hq // hk + 3 * d + 64 + 32) * 2.0 ** -24
    for got, w, a in zip((out,) + grads, want, sizes):
        assert ((got.detach().double().cpu() - w).abs() <= rel * a).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_beside_softmax_attention_of_the_same_rows(dt):
    """A hybrid stack's two kinds of layer take the same turned q and k: the cache's append by rotary_tables, and the fp32 turn."""
    n, h, d = 70, 2, 64
    freq, factor = scaled_inv_freq(d, scaling="ntk", factor=4.0, device="cuda")
    q, k, v = (rand(i, 1, n, h, d, dtype=dt) for i in range(3))
    qr, kr = apply_rotary_emb_qk(q, k, freq, factor=factor)
    cos, sin = rotary_tables(freq, n, factor)
    kc, vc = (torch.zeros(5, 16, h, d, device="cuda", dtype=dt) for _ in range(2))
    table = torch.arange(5, dtype=torch.int32, device="cuda")[None]
    fa.kvcache_append(k, v, kc, vc, torch.zeros(1, dtype=torch.int32, device="cuda"), table, rotary_cos=cos, rotary_sin=sin, rotary_interleaved=False)
    step = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dt]       # a step of the type: each side rounds by half of one
    kept = kc.flatten(0, 1)[:n].float()
    assert ((kept - kr[0].float()).abs() <= step * kept.abs() + 2.0 ** -20).all()
    soft = fa.flash_attn_func(qr, kr, v, causal=True)
    lin = fa.linear_attn_func(qr, kr, v, torch.zeros(h, device="cuda"))
    assert soft.shape == lin.shape and soft.isfinite().all()
    R.close(lin[0], *R.both(qr[0], kr[0], v[0], torch.zeros(h), d ** -0.5)[0], n, (d, d), torch.zeros(h), dt)


def test_example_runs():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-rdna2_b200", "examples", "linear_layer.py")
    spec = importlib.util.spec_from_file_location("linear_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    # outputs differ by two roundings to bf16 (2^-8 each) and the pair products' rounding, states by fp32 sums in another order
    assert mod.main([]) < 2 * 2.0 ** -8 + 2.0 ** -8
