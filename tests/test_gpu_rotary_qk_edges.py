"""The rotary of q and k at the edges of what it is given, against exact fractions of a turn."""
import math
from fractions import Fraction

import pytest
import torch

from fable_attn.layers.rotary import apply_rotary_emb_qk, scaled_inv_freq
from test_gpu_rotary_qk import rand

pytestmark = pytest.mark.gpu
TWO_PI = 2 * Fraction(31415926535897932384626433832795028841971693993751058209749445923, 10 ** 64)


def turned(x, pos, freq, factor=1.0):
    """One token x (heads, dim) at `pos`, pairs (i, i + len(freq)): the angle by rational arithmetic, the rest in fp64."""
    part = [Fraction(f) * pos / TWO_PI for f in freq.cpu().tolist()]
    ang = torch.tensor([2 * math.pi * float(t - round(t)) for t in part], dtype=torch.float64)
    a, b = x.double().cpu().chunk(2, -1)
    c, s = ang.cos() * factor, ang.sin() * factor
    return torch.cat((a * c - b * s, b * c + a * s), -1), factor * (a.abs() + b.abs()).repeat(1, 2)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_angles_of_far_positions(base, sign):
    """2^-64 of a turn for each position, and the roundings of fp32: 8 units of 2^-24 of a value's two terms, as near a position as far."""
    freq, _ = scaled_inv_freq(64, base=base, device="cuda")
    freq = freq * sign
    far = [0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31, 2 ** 35 + 3, 2 ** 40 + 12345, -2 ** 40 + 1]
    pos = torch.tensor([far]).cuda()
    q, k = rand(1, 1, len(far), 2, 64), rand(2, 1, len(far), 1, 64)
    for got, x in zip(apply_rotary_emb_qk(q, k, freq, pos), (q, k)):
        for i, p in enumerate(far):
            want, amp = turned(x[0, i], p, freq)
            off = (got[0, i].double().cpu() - want).abs()
            bound = amp * (8 * 2.0 ** -24 + abs(p) * 2 * math.pi * 2.0 ** -64) + 2.0 ** -24 * want.abs()
            assert (off <= bound).all(), (p, float((off / bound).max()))


def test_frequencies_of_many_turns_and_of_almost_none():
    """Whole turns for each position, fractions below fp64's smallest step of 1, and their negatives."""
    freq = torch.tensor([2 * math.pi, 1000.0, 1e-18, 7.0, -3.0, -1e-12, 2.0 ** -60, 0.0], dtype=torch.float64, device="cuda")
    far = [1, 3, 10 ** 6, -10 ** 6, 2 ** 31]
    q, k = rand(1, len(far), 1, 16), rand(2, len(far), 1, 16)
    for got, x in zip(apply_rotary_emb_qk(q, k, freq, torch.tensor(far).cuda()), (q, k)):
        for i, p in enumerate(far):
            want, amp = turned(x[i], p, freq)
            bound = amp * (8 * 2.0 ** -24 + abs(p) * 2 * math.pi * 2.0 ** -64) + 2.0 ** -24 * want.abs()
            assert ((got[i].double().cpu() - want).abs() <= bound).all(), p


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n", [1, 3000])
def test_frequencies_that_are_no_numbers_show(inter, n):
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k = rand(1, 1, n, 2, 80), rand(2, 1, n, 1, 80)
    want = apply_rotary_emb_qk(q, k, freq, interleaved=inter)
    for i, bad in ((3, math.nan), (17, math.inf), (31, -math.inf)):
        f = freq.clone()
        f[i] = bad
        pair = [2 * i, 2 * i + 1] if inter else [i, i + 32]
        rest = [d for d in range(80) if d not in pair]
        for a, b in zip(apply_rotary_emb_qk(q, k, f, interleaved=inter), want):
            assert a[..., pair].isnan().all() and torch.equal(a[..., rest], b[..., rest])
