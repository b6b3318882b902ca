"""64-bit restatement of the paged 8-bit cache operators for their tests, on the host: one token, head
and sequence at a time, from the definitions in include/fable_attn.h."""
import math

import numpy as np
import torch

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CDT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -100
# half a unit in the last place of a rounding to the type, relative
ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}


def f64(t):
    return t.detach().cpu().float().double().numpy() if t.dtype != torch.int8 else t.cpu().double().numpy()


def rotate(x, pos, cos, sin, interleaved):
    """x (heads, dim) float64 at table row pos."""
    if cos is None:
        return x
    half = cos.shape[1]
    y = x.copy()
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c, s = cos[pos, j], sin[pos, j]
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


class Cache:
    """A random paged cache on the GPU: permuted pages, unused slots full of codes."""

    def __init__(self, rng, batch, heads, dim, page, block, code, max_tokens, spare=2):
        self.page, self.block, self.code, self.heads, self.dim = page, block, code, heads, dim
        self.per = (max_tokens + page - 1) // page + 1
        self.n = batch * self.per + spare
        self.table = torch.from_numpy(rng.permutation(self.n)[:batch * self.per].astype(np.int32).reshape(batch, self.per))
        shape = (self.n, page, heads, dim)
        if code in CDT:
            x = rng.standard_normal(shape) * QMAX[code] / 3
            x = torch.from_numpy(np.clip(x, -QMAX[code], QMAX[code]))
            y = torch.from_numpy(np.clip(rng.standard_normal(shape) * QMAX[code] / 3, -QMAX[code], QMAX[code]))
            conv = (lambda t: t.round().to(torch.int8)) if code == "int8" else (lambda t: t.float().to(CDT[code]))
            self.k, self.v = conv(x).cuda(), conv(y).cuda()
            sc = lambda: torch.from_numpy(np.exp(rng.standard_normal((self.n, heads, page // block))) * 3 / QMAX[code]).float().cuda()
            self.ks, self.vs = sc(), sc()
        else:
            self.k, self.v = (torch.from_numpy(rng.standard_normal(shape)).to("cuda", TDT[code]) for _ in range(2))
            self.ks = self.vs = None
        self.bt = self.table.cuda()

    def values(self, which):
        """float64 (slots of the pool, heads, dim) of what the codes stand for."""
        c = f64(self.k if which == "k" else self.v)
        s = self.ks if which == "k" else self.vs
        if s is not None:
            c = c * np.repeat(f64(s).transpose(0, 2, 1), self.block, axis=1)[..., None]
        return c.reshape(-1, self.heads, self.dim)

    def slot(self, z, pos):
        return int(self.table[z, pos // self.page]) * self.page + pos % self.page


def decode(q, kv, vv, slots, n_ctx, scale, win_left=-1, win_right=0, softcap=0.0, alibi=None, leftpad=0, cos=None, sin=None,
           interleaved=False, rot0=None):
    """One sequence: q (n, Hq, D) float64, kv / vv (slots, Hk, D) values, slots[pos].  Returns out, lse."""
    n, hq, d = q.shape
    hk = kv.shape[1]
    out, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    for t in range(n):
        pos = n_ctx - n + t
        lo = max(leftpad, 0 if win_left < 0 else pos - win_left, 0)
        hi = n_ctx if win_right < 0 else min(n_ctx, pos + win_right + 1)
        if hi <= lo:
            continue
        x = rotate(q[t], pos if rot0 is None else rot0 + t, cos, sin, interleaved)
        keys = np.arange(lo, hi)
        rows = np.array([slots[j] for j in keys])
        keep = rows >= 0
        keys, rows = keys[keep], rows[keep]
        if not len(keys):
            continue
        for h in range(hq):
            s = kv[rows, h // (hq // hk)] @ x[h] * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if alibi is not None:
                s = s + alibi[h] * (keys - pos)
            m = s.max()
            w = np.exp(s - m)
            lse[t, h] = m + math.log(w.sum()) if np.isfinite(m) else m
            out[t, h] = w @ vv[rows, h // (hq // hk)] / w.sum()
    return out, lse
