"""Serving with an 8-bit paged K/V cache: chunked prefill, then decode steps.

One attention layer of a small batch, with random projections' worth of q / k / v:
  prefill  each chunk is rotated and appended (kvcache_append), the whole context so far comes back as packed bf16
           (kvcache_gather), and flash_attn_varlen_func attends with the causal mask aligned to the chunk's end;
  decode   each step appends one token a sequence and attends over the cache (flash_attn_with_kvcache_8bit).
Every output is compared with the same layer over an unquantised cache, and the relative distance is printed: about
1 % for int8 and 3 % for e4m3, which is what the 8 bits cost.

    python flash-attention-rdna2_b200/examples/serve_8bit_cache.py [--dtype int8|e4m3] [--steps N]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fable_attn as fa  # noqa: E402
from fable_attn.layers.rotary import apply_rotary_emb  # noqa: E402


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--dtype", choices=("int8", "e4m3"), default="int8")
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--chunk", type=int, default=256)
    a = ap.parse_args(argv)
    dev = torch.device("cuda")
    torch.manual_seed(0)
    hq, hk, d, page, block = 16, 4, 128, 64, 16
    prompts = [700, 33, 1025, 256]
    batch, longest = len(prompts), max(prompts) + a.steps
    per = (longest + page - 1) // page
    codes = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[a.dtype]
    k_cache, v_cache, k_scale, v_scale = fa.new_cache_8bit(batch * per, page, hk, d, codes, block, dev)
    table = torch.randperm(batch * per, device=dev).to(torch.int32).view(batch, per)
    ang = torch.arange(longest, device=dev)[:, None] * 10000.0 ** (-torch.arange(d // 2, device=dev) / (d // 2))
    cos, sin = ang.cos(), ang.sin()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    cum = lambda v: i32([0] + [sum(v[:i + 1]) for i in range(len(v))])

    def tokens(counts):   # new q, k, v of a step, packed
        n = sum(counts)
        return (torch.randn(n, h, d, device=dev, dtype=torch.bfloat16) for h in (hq, hk, hk))

    kept = [([], []) for _ in prompts]     # the unquantised cache: rotated keys, values
    scales = dict(k_scale=k_scale, v_scale=v_scale)

    def keep(k, v, counts, done):
        at = 0
        for b, n in enumerate(counts):
            if n:
                kept[b][0].append(apply_rotary_emb(k[None, at:at + n], cos[done[b]:], sin[done[b]:])[0])
                kept[b][1].append(v[at:at + n])
            at += n

    def exact(q, counts, done):            # the same attention over it
        outs, at = [], 0
        for b, n in enumerate(counts):
            if n:
                qr = apply_rotary_emb(q[None, at:at + n], cos[done[b]:], sin[done[b]:])
                outs.append(fa.flash_attn_func(qr, torch.cat(kept[b][0])[None], torch.cat(kept[b][1])[None], causal=True)[0])
            at += n
        return torch.cat(outs)

    done, worst = [0] * batch, 0.0
    while any(n < p for n, p in zip(done, prompts)):
        counts = [min(a.chunk, p - n) for n, p in zip(done, prompts)]
        q, k, v = tokens(counts)
        fa.kvcache_append(k, v, k_cache, v_cache, i32(done), table, cu_seqlens_new=cum(counts), rotary_cos=cos, rotary_sin=sin,
                          rotary_interleaved=False, **scales)
        now = [x + n for x, n in zip(done, counts)]
        ks, vs = fa.kvcache_gather(k_cache, v_cache, table, cum(now), sum(now), dtype=q.dtype, **scales)
        qr = apply_rotary_emb(q, cos, sin, seqlen_offsets=i32(done), cu_seqlens=cum(counts), max_seqlen=max(counts))
        out = fa.flash_attn_varlen_func(qr, ks, vs, cum(counts), cum(now), max(counts), max(now), causal=True)
        keep(k, v, counts, done)
        worst = max(worst, rel(out, exact(q, counts, done)))
        done = now
    print(f"prefill of {prompts} tokens in chunks of {a.chunk}: {worst:.4f} from the unquantised cache")

    prefill, worst = worst, 0.0
    for _ in range(a.steps):
        q, k, v = tokens([1] * batch)
        fa.kvcache_append(k[:, None], v[:, None], k_cache, v_cache, i32(done), table, rotary_cos=cos, rotary_sin=sin,
                          rotary_interleaved=False, **scales)
        now = [x + 1 for x in done]
        out = fa.flash_attn_with_kvcache_8bit(q[:, None], k_cache, v_cache, k_scale, v_scale, i32(now), table, rotary_cos=cos,
                                              rotary_sin=sin, rotary_interleaved=False)
        keep(k, v, [1] * batch, done)
        worst = max(worst, rel(out[:, 0], exact(q, [1] * batch, done)))
        done = now
    print(f"{a.steps} decode steps: {worst:.4f} from the unquantised cache")
    return max(prefill, worst)


if __name__ == "__main__":
    main()
