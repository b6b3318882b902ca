"""What fp16 operands of the tensor-core kernels of linear attention may lose below fp16's smallest step, beside the relative bounds of lin_ref.

Three things enter a matrix product as two fp16 numbers hi + lo.  Where hi is below fp16's normal numbers the two together are off by up to half of its
smallest step, 2^-25:
  pair products   a power of 2 brings a row's largest one to 2^10 or more, so that 2^-35 of that one is lost;
  the state       likewise, with the largest element of a state;
  decayed rows    b lam^m (dk: c lam^m) as they are: 2^-25 each, carried from their chunk's end on with the other operand.
Last states are summed from rows whose second number is held 2^11 times as large: 2^-36 each.  A chunk is 128 tokens from the sequence's start.
(What the tensor cores cut from a sum of operands that small, about 2^-37 of the other operand's largest value for each sixteen tokens, is of
the same size and not counted.)"""
import torch

CHUNK = 128


def _role(a, b, c, x, w_intra, w_inter, w_up, g, rev, swap):
    """(n, heads of a, dims of c) for one kv head: a (n, ga, da), b (n, gb, da), c (n, gb, dc), absolute values; x: bound on the state's elements."""
    n = len(a)
    i, j = torch.arange(n)[:, None], torch.arange(n)
    seen = ((j >= i) if rev else (j <= i)).double()
    steps = CHUNK * (j // CHUNK) - 1 - i if rev else i + 1 - CHUNK * (j // CHUNK + 1)
    far = torch.where((j // CHUNK > i // CHUNK) if rev else (j // CHUNK < i // CHUNK), (g.clamp(min=-1e30) * steps.clamp(min=0)).exp(), torch.zeros(()).double())
    p = torch.einsum("iad,jbd->abij", a, b)
    total = w_intra * 2.0 ** -35 * torch.einsum("abi,ij,jbc->iac", (p * seen).amax(-1), seen, c)
    of_a = a.sum(-1)[..., None]
    if swap:
        total = total + w_inter * w_up * 2.0 ** -25 * torch.einsum("abij,ij->ia", p, far)[..., None]
    else:
        total = total + w_inter * w_up * 2.0 ** -25 * of_a * torch.einsum("ij,jbc->ic", far, c)[:, None]
    return total + w_inter * 2.0 ** -35 * of_a * x


def floors(q, k, v, g, scale, s0=None, do=None, ds=None):
    """For the results of lin_ref.one, in its order."""
    f = lambda t: t.detach().double().cpu().abs()
    q, k, v, g, scale = f(q), f(k), f(v), g.detach().double().cpu().clamp(max=0), abs(scale)
    n, hk, grp = len(q), k.shape[1], q.shape[1] // k.shape[1]
    outs = [[] for _ in range(6 if do is not None else 2)]
    for h in range(hk):
        qh, kh, vh = q[:, h * grp:h * grp + grp], k[:, h:h + 1], v[:, h:h + 1]
        x = torch.einsum("jbd,jbc->dc", kh, vh).max() + (0 if s0 is None else f(s0)[h].max())
        outs[0].append(_role(qh, kh, vh, x, scale, scale, 1.0, g[h], False, False))
        outs[1].append(2.0 ** -36 * vh.sum(0).expand(k.shape[2], -1)[None])
        if do is None:
            continue
        dh = f(do)[:, h * grp:h * grp + grp]
        r = scale * torch.einsum("jbd,jbc->dc", qh, dh).max() + (0 if ds is None else f(ds)[h].max())
        outs[2].append(_role(dh, vh, kh, x, scale, scale, 1.0, g[h], False, False))
        outs[3].append(_role(vh, dh, qh, r, scale, 1.0, scale, g[h], True, True))
        outs[4].append(_role(kh, qh, dh, r, scale, 1.0, scale, g[h], True, False))
        outs[5].append(scale * 2.0 ** -36 * dh.sum((0, 1)).expand(k.shape[2], -1)[None])
    return [torch.cat(o, 0 if i in (1, 5) else 1) for i, o in enumerate(outs)]


def close(got, want, amp, floor, n, dims, g, operands, what=""):
    """lin_ref.close with `floor` in the place of one allowance for every size."""
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
    size = g.double().abs()
    gmax = float(torch.where(size > 100, torch.zeros_like(size), size).max())
    rel = (n * (1 + 2 * gmax) + sum(dims) + 64) * 2.0 ** -24 + (3 * u[operands] ** 2 if operands != torch.float32 else 0.0)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -120       # half of the result's smallest step
    x = got.detach().double().cpu()
    assert torch.isfinite(x).all(), f"{what}: not finite"
    bound = u[got.dtype] * want.abs() + rel * amp + (floor if operands == torch.float16 else 0.0) + tiny
    off = (x - want).abs()
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} times the bound"
