"""Linear attention with a decay per head in 64 bits, all pairs of tokens at once, and how far the kernels may be from it.

Every term of every sum is a product, so the same formulas over absolute values give `amp`, the sum of the terms' sizes.
Bounds count roundings (half a step u each, relative to a term):
  fp32 sums          a term passes at most n + dk + dv + 64 additions and products, u = 2^-24;
  powers of lam      exp2(n log2 lam): the exponent is rounded twice, which moves lam^n by n |log_decay| 2 u, and exp2f by 2 u;
  16-bit operands    pair products, states and decayed rows enter matrix products as two 16-bit numbers hi + lo: what is left is
                     u16^2 of a term (2^-16 for bf16, 2^-22 for fp16), three times at most; below fp16's normal numbers a step is 2^-24;
  the result         half a step of its type.
"""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def one(q, k, v, g, scale, s0=None, do=None, ds=None):
    """One sequence: q (n, hq, dk), k (n, hk, dk), v (n, hk, dv), fp64.  (o, final) and, with do, (dq, dk, dv, ds0)."""
    n, hq, dk = q.shape
    hk, dv = v.shape[1:]
    grp = hq // hk
    s0 = q.new_zeros(hk, dk, dv) if s0 is None else s0
    g = g.clamp(max=0)
    t = torch.arange(n, dtype=torch.float64)

    def power(steps):          # (hk, *steps.shape), 0 where steps < 0; lam^0 = 1 for lam = 0 too
        x = torch.where(steps == 0, torch.zeros(()).double(), g.view(-1, *[1] * steps.dim()) * steps.clamp(min=0))
        return torch.where(steps >= 0, x.exp(), torch.zeros(()).double())

    w = power(t[:, None] - t)                                   # hk i j
    rise, fall, whole = power(t + 1), power(n - 1 - t), power(torch.tensor(float(n)))
    qg = q.view(n, hk, grp, dk)
    a = torch.einsum("ihgd,jhd->hgij", qg, k) * w[:, None]
    o = torch.einsum("hgij,jhe->ihge", a, v) + torch.einsum("ihgd,hde,hi->ihge", qg, s0, rise)
    final = whole[:, None, None] * s0 + torch.einsum("hj,jhd,jhe->hde", fall, k, v)
    out = [scale * o.reshape(n, hq, dv), final]
    if do is not None:
        dog = do.view(n, hk, grp, dv)
        b = torch.einsum("ihge,jhe->hgij", dog, v) * w[:, None]
        dq = torch.einsum("hgij,jhd->ihgd", b, k) + torch.einsum("ihge,hde,hi->ihgd", dog, s0, rise)
        gk = scale * torch.einsum("hgij,ihgd->jhd", b, qg)
        gv = scale * torch.einsum("hgij,ihge->jhe", a, dog)
        g0 = scale * torch.einsum("ihgd,ihge,hi->hde", qg, dog, rise)
        if ds is not None:
            gk = gk + torch.einsum("jhe,hde,hj->jhd", v, ds, fall)
            gv = gv + torch.einsum("jhd,hde,hj->jhe", k, ds, fall)
            g0 = g0 + whole[:, None, None] * ds
        out += [scale * dq.reshape(n, hq, dk), gk, gv, g0]
    return out


def both(q, k, v, g, scale, s0=None, do=None, ds=None):
    """[(value, amp)] of one()."""
    f = lambda x: None if x is None else x.detach().double().cpu()
    a = lambda x: None if x is None else f(x).abs()
    return list(zip(one(f(q), f(k), f(v), f(g), scale, f(s0), f(do), f(ds)), one(a(q), a(k), a(v), f(g), scale, a(s0), a(do), a(ds))))


def close(got, want, amp, n, dims, g, operands, what=""):
    """Every element within the bound above.  operands: the type of q, k, v."""
    u = U[got.dtype]
    size = g.double().abs()
    gmax = float(torch.where(size > 100, torch.zeros_like(size), size).max())     # lam below e^-100: what is left is below `tiny`
    rel = (n * (1 + 2 * gmax) + sum(dims) + 64) * 2.0 ** -24
    tiny = 2.0 ** -120
    if operands != torch.float32:
        rel += 3 * U[operands] ** 2
    if operands == torch.float16:
        tiny = 2.0 ** -24
    x = got.detach().double().cpu()
    off = (x - want).abs()
    bound = u * want.abs() + rel * amp + tiny
    assert torch.isfinite(x).all(), f"{what}: not finite"
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} times the bound"
