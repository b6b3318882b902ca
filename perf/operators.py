"""Workloads of the paged-cache operators: kvcache_append, kvcache_gather and flash_attn_with_kvcache_8bit.

A cache is paged, (num_blocks, page, nheads_k, headdim), and holds 16-bit elements or 8-bit codes
(int8 or e4m3) with one fp32 scale for each `block` consecutive slots of a page and each head,
(num_blocks, nheads_k, page / block): an element's value is code * scale.

    append  new K/V rows (one per sequence, or ragged counts) are rotated and written behind each
            sequence's cached tokens.  In 8 bits, the values that the touched blocks now stand for are
            read back with kvcache_gather.
    gather  a range of each sequence's cache comes back as packed 16-bit K/V, as the prefill of a
            further chunk takes it.
    decode  attention of one or several new tokens per sequence over the 8-bit cache.

`run` computes them with elementary fp32 torch operations, or, with `own` set, through fable_attn.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -100
CACHED = dict(op="", batch=1, heads_q=8, heads_k=8, dim=128, page=16, block=16, code="int8", dtype="bf16",
              ctx_lo=0, ctx_hi=0, new_lo=1, new_hi=1, rotary=0, interleaved=False, window=-1, softcap=0.0, alibi=False)


def _case(name, **kw):
    c = dict(CACHED, **kw)
    assert not set(kw) - set(CACHED)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of 64 chats into a bf16 cache: a launch-bound call
        _case("append_bf16_step", op="append", code="none", batch=64, ctx_lo=100, ctx_hi=4000, rotary=128),
        # ragged prefill of 16 prompts (256 to 8192 tokens) into an empty fp16 cache, half of the head rotated
        _case("append_fp16_prompts", op="append", code="none", dtype="fp16", batch=16, page=256, ctx_lo=0, ctx_hi=0,
              new_lo=256, new_hi=8192, rotary=64),
        # one decode step of 32 sequences into an int8 cache: blocks that are partly filled
        _case("append_int8_step", op="append", batch=32, ctx_lo=37, ctx_hi=2111, rotary=128, interleaved=True),
        # the same ragged prompts appended behind earlier chunks, e4m3 with a scale for 64 tokens
        _case("append_e4m3_prompts", op="append", code="e4m3", batch=16, page=256, block=64, ctx_lo=0, ctx_hi=1000,
              new_lo=256, new_hi=8192, rotary=128),
        # one 4k context brought back for its next prefill chunk
        _case("gather_int8_one", op="gather", ctx_lo=4099, ctx_hi=4099),
        # 16 contexts of 16k to 32k, the paged decode workload's cache
        _case("gather_e4m3_many", op="gather", code="e4m3", batch=16, page=256, block=64, ctx_lo=16384, ctx_hi=32768),
        # the smallest decode: one short chat, no grouping, headdim 64
        _case("decode_int8_short", op="decode", dtype="fp16", dim=64, page=16, ctx_lo=611, ctx_hi=611),
        # a serving batch of medium contexts, a scale for each token
        _case("decode_e4m3_batch", op="decode", code="e4m3", batch=48, heads_q=32, page=64, block=1, ctx_lo=700,
              ctx_hi=9000, rotary=128),
        # the paged decode workload (16 sequences of 16k to 32k, 32 / 8 heads, pages of 256) in both codes
        _case("decode_int8_paged", op="decode", batch=16, heads_q=32, page=256, block=64, ctx_lo=16384, ctx_hi=32768),
        _case("decode_e4m3_paged", op="decode", code="e4m3", batch=16, heads_q=32, page=256, block=64, ctx_lo=16384,
              ctx_hi=32768),
        # speculative verification of 1 to 4 tokens, sliding window, softcap
        _case("decode_int8_verify", op="decode", dtype="fp16", batch=24, heads_q=32, page=32, ctx_lo=1000, ctx_hi=20000,
              new_lo=1, new_hi=4, rotary=64, window=4096, softcap=30.0),
        # one long document, groups of 8 query heads
        _case("decode_int8_long", op="decode", batch=1, heads_q=64, page=128, block=32, ctx_lo=131001, ctx_hi=131001,
              rotary=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "gather", "decode", "decode", "decode"])
    c = _case(None, op=op)
    c["code"] = rng.choice(["int8", "e4m3", "none"] if op == "append" else ["int8", "e4m3"])
    c["dtype"] = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"] if op == "decode" else ["bf16", "fp16"])
    c["dim"] = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    c["heads_k"] = rng.choice([1, 2, 3, 4, 8, 8])
    c["heads_q"] = c["heads_k"] * rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    c["page"] = rng.choice([16, 32, 64, 128, 256])
    c["block"] = min(c["page"], rng.choice([1, 2, 8, 16, 16, 32, 64, 256]))
    c["batch"] = _log(rng, 1, 128)
    room = 16 * 24000 * 8 * 128 // (c["heads_k"] * c["dim"])     # cached tokens of the largest listed case
    if op == "append":
        c["new_hi"] = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(8192, room // 8 // c["batch"])))
        c["new_lo"] = 1 if c["new_hi"] == 1 else _log(rng, 1, c["new_hi"])
        c["ctx_hi"] = 0 if rng.random() < 0.3 else _log(rng, 1, max(1, min(20000, room // 8 // c["batch"])))
    else:
        # several query rows a head read the cache as often: they come with smaller caches
        if op == "decode" and rng.random() < 0.35:
            c["new_hi"] = rng.choice([2, 3, 4, 8])
            c["new_lo"] = rng.randint(1, c["new_hi"])
        rows = c["new_hi"] * c["heads_q"] // c["heads_k"] if op == "decode" else 1
        c["ctx_hi"] = max(8, _log(rng, 8, max(9, min(131072, room // c["batch"] // max(1, (rows + 7) // 8)))))
    c["ctx_lo"] = _log(rng, 1, c["ctx_hi"]) if c["ctx_hi"] else 0
    if op != "gather" and rng.random() < 0.7:
        c["rotary"] = rng.choice([c["dim"], c["dim"] // 2])
        c["interleaved"] = rng.random() < 0.5
    if op == "decode":
        c["window"] = rng.choice([-1, -1, -1, 128, 1000, 4096])
        c["softcap"] = rng.choice([0.0, 0.0, 30.0])
        c["alibi"] = rng.random() < 0.2
    return c


def _spread(lo, hi, n, turn):
    """n whole numbers of [lo, hi], both ends among them where n > 1, in an order that is no order."""
    if n == 1:
        return [hi]
    got = [lo + round((hi - lo) * i / (n - 1)) for i in range(n)]
    return [got[(i * turn + 3) % n] for i in range(n)] if math.gcd(turn, n) == 1 else got


def _lengths(case):
    """(cached tokens, new tokens) of each sequence.  A decode's cached tokens include the new ones."""
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], 7)
    new = _spread(case["new_lo"], case["new_hi"], case["batch"], 5)
    if case["op"] == "decode":
        ctx = [max(c, n) for c, n in zip(ctx, new)]
    return ctx, new


def _visible(case):
    """[(first position that any query sees, one past the last)] of a decode's sequences, and its query-key pairs."""
    ctx, new = _lengths(case)
    w, spans, pairs = case["window"], [], 0
    for c, n in zip(ctx, new):
        rows = [(max(0, c - n + t - w) if w >= 0 else 0, c - n + t + 1) for t in range(n)]
        spans.append((rows[0][0], c))
        pairs += sum(b - a for a, b in rows)
    return spans, pairs


def work(case):
    hk, d, sb = case["heads_k"], case["dim"], case["block"]
    e = {"fp32": 4}.get(case["dtype"], 2)
    ctx, new = _lengths(case)
    if case["op"] == "decode":
        spans, pairs = _visible(case)
        keys = sum(b - a for a, b in spans)
        blocks = sum((b - 1) // sb + 1 - a // sb for a, b in spans)
        byt = 2 * hk * (keys * d + blocks * 4) + sum(new) * case["heads_q"] * (2 * d * e + 4) + sum(new) * case["rotary"] * 4
        return {"bytes": byt, "flops": 4 * d * case["heads_q"] * pairs}
    if case["op"] == "gather":
        blocks = sum((c - 1) // sb + 1 for c in ctx)
        return {"bytes": 2 * hk * (sum(ctx) * d * (1 + e) + blocks * 4), "flops": 2 * hk * d * sum(ctx)}
    n = sum(new)
    byt = 2 * hk * n * d * e + n * case["rotary"] * 4
    if case["code"] == "none":
        return {"bytes": byt + 2 * hk * n * d * e, "flops": 3 * hk * case["rotary"] * n}
    held = sum(c + k - c // sb * sb for c, k in zip(ctx, new))       # tokens of the touched blocks
    blocks = sum((c + k - 1) // sb + 1 - c // sb for c, k in zip(ctx, new))
    # written as codes, scales written, and the touched blocks read as codes and written as values
    byt += 2 * hk * (n * d + blocks * 8 + held * d * (1 + e))
    return {"bytes": byt, "flops": 2 * hk * d * (3 * n + held)}


# ------------------------------------------------------------------ inputs
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=_device())


def _cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _rows(n, hk, d, gen):
    """n rows of K- or V-like values: channels of unlike size, a few of them several times the others'."""
    ch = torch.randn(hk, d, generator=gen, device=_device()).mul_(0.4).exp_()
    ch *= 1 + 4 * (torch.rand(hk, d, generator=gen, device=_device()) < 0.03)
    x = torch.randn(n, hk, d, generator=gen, device=_device())
    return x * (ch / ch.square().mean().sqrt())


def _quantised(blocks, page, sb, hk, d, code, gen):
    """A pool of pages full of codes and their scales, as earlier appends left them."""
    codes = torch.empty(blocks, page, hk, d, dtype=CODES[code], device=_device())
    scale = torch.empty(blocks, hk, page // sb, device=_device())
    step = max(1, (1 << 27) // (page * hk * d))
    for a in range(0, blocks, step):
        b = min(blocks, a + step)
        x = _rows((b - a) * page, hk, d, gen).view(b - a, page // sb, sb, hk, d)
        s = (x.abs().amax(dim=(2, 4)) / QMAX[code]).clamp_min(MIN_SCALE)
        x = x * (1.0 / s)[:, :, None, :, None]
        codes[a:b] = (x.round() if code == "int8" else x).clamp(-QMAX[code], QMAX[code]).to(CODES[code]).view(
            b - a, page, hk, d)
        scale[a:b] = s.transpose(1, 2)
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(seed)
    op, b, hk, d, page, sb = (case[k] for k in ("op", "batch", "heads_k", "dim", "page", "block"))
    dt = DTYPES[case["dtype"]]
    ctx, new = _lengths(case)
    end = [c + n for c, n in zip(ctx, new)] if op == "append" else ctx
    pages = [(e + page - 1) // page for e in end]
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=gen, device=_device()).to(torch.int32).cpu()
    table = torch.zeros(b, max(max(pages), 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"case": case, "table": table.to(_device()), "ctx": _i32(ctx), "total_new": sum(new), "total_ctx": sum(ctx),
         "cu_new": _i32(_cum(new)), "cu_ctx": _i32(_cum(ctx)), "new_hi": max(new), "ctx_hi": max(ctx), "k_scale": None,
         "v_scale": None, "cos": None, "sin": None, "slopes": None}
    if case["code"] == "none":
        s["k_cache"] = _rows(pool * page, hk, d, gen).to(dt).view(pool, page, hk, d)
        s["v_cache"] = _rows(pool * page, hk, d, gen).to(dt).view(pool, page, hk, d)
    else:
        s["k_cache"], s["k_scale"] = _quantised(pool, page, sb, hk, d, case["code"], gen)
        s["v_cache"], s["v_scale"] = _quantised(pool, page, sb, hk, d, case["code"], gen)
    if op == "append":
        s["k"] = _rows(s["total_new"], hk, d, gen).to(dt)
        s["v"] = _rows(s["total_new"], hk, d, gen).to(dt)
        s["even"] = case["new_lo"] == case["new_hi"]
        # the blocks that the append touches, whole: from the first one's first slot to the last new token
        first = [c // sb * sb for c in ctx]
        s["starts"] = _i32(first)
        s["cu_held"] = _i32(_cum([e - f for e, f in zip(end, first)]))
        s["total_held"] = sum(e - f for e, f in zip(end, first))
    if op == "decode":
        s["q"] = torch.randn(s["total_new"], case["heads_q"], d, generator=gen, device=_device()).to(dt)
        s["even"] = case["new_lo"] == case["new_hi"]
        if case["alibi"]:
            s["slopes"] = torch.rand(case["heads_q"], generator=gen, device=_device()) * 0.05
    if case["rotary"]:
        half = case["rotary"] // 2
        inv = 10000.0 ** (-torch.arange(half, device=_device(), dtype=torch.float64) / half)
        ang = torch.arange(max(end) + 1, device=_device(), dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


# ------------------------------------------------------------------ the framework's operators
_module = None


def _fa():
    global _module
    if _module is None:
        here = os.path.dirname(os.path.abspath(__file__))
        sys.path.insert(0, os.path.join(os.path.dirname(here), "flash-attention-rdna2_b200"))
        import fable_attn
        _module = fable_attn
    return _module


def _batched(x, s):
    """(batch, tokens, heads, dim) where every sequence has as many new tokens, else packed rows."""
    return x.view(s["case"]["batch"], -1, *x.shape[1:]) if s["even"] else x


def _run_own(s):
    fa, case = _fa(), s["case"]
    if case["op"] == "append":
        fa.kvcache_append(_batched(s["k"], s), _batched(s["v"], s), s["k_cache"], s["v_cache"], s["ctx"], s["table"],
                          k_scale=s["k_scale"], v_scale=s["v_scale"], cu_seqlens_new=None if s["even"] else s["cu_new"],
                          rotary_cos=s["cos"], rotary_sin=s["sin"], rotary_interleaved=case["interleaved"])
        if case["code"] == "none":
            return s["k_cache"], s["v_cache"]
        k, v = fa.kvcache_gather(s["k_cache"], s["v_cache"], s["table"], s["cu_held"], s["total_held"],
                                 k_scale=s["k_scale"], v_scale=s["v_scale"], seq_starts=s["starts"], dtype=s["k"].dtype)
        return k, v, s["k_scale"], s["v_scale"]
    if case["op"] == "gather":
        return fa.kvcache_gather(s["k_cache"], s["v_cache"], s["table"], s["cu_ctx"], s["total_ctx"],
                                 k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=DTYPES[case["dtype"]])
    out, lse = fa.flash_attn_with_kvcache_8bit(
        _batched(s["q"], s), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["ctx"], s["table"], causal=True,
        window_size=(case["window"], 0), softcap=case["softcap"], alibi_slopes=s["slopes"], rotary_cos=s["cos"],
        rotary_sin=s["sin"], rotary_interleaved=case["interleaved"],
        cu_seqlens_q=None if s["even"] else s["cu_new"], max_seqlen_q=None if s["even"] else s["new_hi"],
        return_softmax_lse=True)
    if s["even"]:   # (batch, heads, tokens) -> (heads, batch * tokens), as the packed form has it
        lse = lse.transpose(0, 1).reshape(lse.shape[1], -1)
    return out.reshape(-1, *out.shape[-2:]), lse


# ------------------------------------------------------------------ their plain form
def _rotated(x, pos, s):
    """x (rows, heads, dim) in fp32, rotated by the table rows of pos."""
    rd = s["case"]["rotary"]
    if not rd:
        return x
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    y = x.clone()
    if s["case"]["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        y[..., 0:rd:2], y[..., 1:rd:2] = a * c - b * n, b * c + a * n
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        y[..., :rd // 2], y[..., rd // 2:rd] = a * c - b * n, b * c + a * n
    return y


def _packed(cu, total, first):
    """Sequence and position of each of the packed rows; sequence b's rows begin at position first[b]."""
    row = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), row, right=True)
    return seq, row - cu.long()[seq] + first.long()[seq]


def _slots(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos // page].long() * page + pos % page


def _scales_of(scale, slot, case):
    """The scale (rows, heads) of each slot."""
    page = case["page"]
    return scale[slot // page, :, slot % page // case["block"]]


def _to_codes(x, case):
    q = QMAX[case["code"]]
    return (x.round() if case["code"] == "int8" else x).clamp(-q, q).to(CODES[case["code"]])


def _append_8bit(x, cache, scale, slot, s):
    case = s["case"]
    page, sb = case["page"], case["block"]
    bits = cache.view(-1, *cache.shape[2:]).view(torch.uint8)
    by_block = scale.transpose(1, 2)                                  # (num_blocks, page / block, heads)
    blk = slot // sb
    most = torch.zeros(by_block.shape[0] * by_block.shape[1], x.shape[1], device=x.device)
    most.scatter_reduce_(0, blk[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    # the block that a sequence's new tokens continue: its earlier tokens hold on to their scale
    ctx = s["ctx"].long()
    part = torch.nonzero(ctx % sb).view(-1)
    last = _slots(s, part, ctx[part] - 1) // sb
    old = by_block[last // (page // sb), last % (page // sb)]         # (sequences, heads)
    base = torch.zeros_like(most)
    base[last] = old
    fresh = torch.maximum(base, (most / QMAX[case["code"]]).clamp_min(MIN_SCALE))
    bits[slot] = _to_codes(x * (1.0 / fresh[blk])[..., None], case).view(torch.uint8)
    # earlier tokens of those blocks, by the scale that the block has now
    now = fresh[last]
    inner = torch.arange(sb, device=x.device)
    where = last[:, None] * sb + inner
    stale = (inner < (ctx[part] % sb)[:, None])[..., None] & (now > old)[:, None]
    held = bits[where]                                                # (sequences, block, heads, dim)
    again = _to_codes(held.view(cache.dtype).float() * (old / now)[:, None, :, None], case).view(torch.uint8)
    bits[where] = torch.where(stale[..., None], again, held)
    by_block[blk // (page // sb), blk % (page // sb)] = fresh[blk]


def _run_append(s):
    case = s["case"]
    seq, pos = _packed(s["cu_new"], s["total_new"], s["ctx"])
    slot = _slots(s, seq, pos)
    k, v = _rotated(s["k"].float(), pos, s), s["v"].float()
    if case["code"] == "none":
        s["k_cache"].view(-1, *k.shape[1:])[slot] = k.to(s["k"].dtype)
        s["v_cache"].view(-1, *v.shape[1:])[slot] = v.to(s["v"].dtype)
        return s["k_cache"], s["v_cache"]
    _append_8bit(k, s["k_cache"], s["k_scale"], slot, s)
    _append_8bit(v, s["v_cache"], s["v_scale"], slot, s)
    seq, pos = _packed(s["cu_held"], s["total_held"], s["starts"])
    return (*_values(s, _slots(s, seq, pos), s["k"].dtype), s["k_scale"], s["v_scale"])


def _values(s, slot, dtype):
    """K and V (rows, heads, dim) that the slots stand for."""
    got = []
    for which in ("k", "v"):
        cache = s[which + "_cache"]
        codes = cache.view(-1, *cache.shape[2:]).view(torch.uint8)[slot].view(cache.dtype)
        got.append((codes.float() * _scales_of(s[which + "_scale"], slot, s["case"])[..., None]).to(dtype))
    return got


def _run_gather(s):
    seq, pos = _packed(s["cu_ctx"], s["total_ctx"], torch.zeros_like(s["ctx"]))
    return _values(s, _slots(s, seq, pos), DTYPES[s["case"]["dtype"]])


def _run_decode(s):
    case = s["case"]
    b, hk, hq, d = case["batch"], case["heads_k"], case["heads_q"], case["dim"]
    dev, n, g = s["q"].device, s["new_hi"], hq // hk
    ctx = s["ctx"].long()
    count = (s["cu_new"][1:] - s["cu_new"][:-1]).long()
    seq, pos = _packed(s["cu_new"], s["total_new"], ctx - count)
    row = pos - (ctx - count)[seq]
    q = torch.zeros(b, n, hq, d, device=dev)
    q[seq, row] = _rotated(s["q"].float(), pos, s)
    q = q.view(b, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, d)
    keys = torch.arange(s["ctx_hi"], device=dev)
    at = torch.minimum(keys, ctx[:, None] - 1)                        # rows past a sequence's end are masked below
    k, v = _values(s, _slots(s, torch.arange(b, device=dev)[:, None], at).view(-1), torch.float32)
    k, v = (x.view(b, -1, hk, d).transpose(1, 2) for x in (k, v))
    score = (q @ k.transpose(-1, -2) * d ** -0.5).view(b, hk, n, g, -1)
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    q_pos = (ctx - count)[:, None] + torch.arange(n, device=dev)      # (batch, tokens)
    away = keys - q_pos[..., None]                                    # (batch, tokens, keys)
    if s["slopes"] is not None:
        score = score + s["slopes"].view(1, hk, 1, g, 1) * away[:, None, :, None].float()
    seen = (away <= 0) & (keys < ctx[:, None, None])
    if case["window"] >= 0:
        seen &= away >= -case["window"]
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p / total.clamp_min(1e-30)).view(b, hk, n * g, -1) @ v
    out = out.view(b, hk, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    lse = (top + total.log()).view(b, hk, n, g).permute(1, 3, 0, 2).reshape(hq, b, n)
    return out[seq, row].to(s["q"].dtype), lse[:, seq, row]


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "gather": _run_gather, "decode": _run_decode}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _turned(x, first, s):
    """One sequence's rows x (n, heads, dim), fp64, from position `first` on: pairs as complex numbers."""
    rd, half = s["case"]["rotary"], s["case"]["rotary"] // 2
    if not rd:
        return x
    e = torch.complex(s["cos"][first:first + len(x)].double(), s["sin"][first:first + len(x)].double())[:, None]
    if s["case"]["interleaved"]:
        z = torch.complex(x[..., :rd].unflatten(-1, (half, 2))[..., 0], x[..., :rd].unflatten(-1, (half, 2))[..., 1]) * e
        turned = torch.stack((z.real, z.imag), -1).flatten(-2)
    else:
        z = torch.complex(x[..., :half], x[..., half:rd]) * e
        turned = torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _line(s, i, a, b, which):
    """What positions [a, b) of sequence i stand for, fp64 (b - a, heads, dim)."""
    case, page = s["case"], s["case"]["page"]
    got = []
    for p in range(a // page, (max(a, b - 1)) // page + 1):
        blk = int(s["table"][i, p])
        x = s[which + "_cache"][blk].double()
        if s[which + "_scale"] is not None:
            x = x * s[which + "_scale"][blk].double().repeat_interleave(case["block"], 1).t()[..., None]
        got.append(x)
    return torch.cat(got)[a - a // page * page:][:b - a]


def _rounded(x, code):
    """x in units of a scale, as the nearest code: whole numbers, or 4 significant bits and a least step of 2^-9."""
    if code == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.frexp(x.abs().clamp_min(2.0 ** -20)).exponent.double().sub(4).clamp_min(-9))
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(s):
    case, page, sb = s["case"], s["case"]["page"], s["case"]["block"]
    ctx, new = _lengths(case)
    out = {}
    for which in ("k", "v"):
        cache = s[which + "_cache"].double() if case["code"] == "none" else None
        scale = None if cache is not None else s[which + "_scale"].double()
        held, at = [], 0
        for i, (c, n) in enumerate(zip(ctx, new)):
            x = s[which][at:at + n].double()
            at += n
            x = _turned(x, c, s) if which == "k" else x
            if cache is not None:
                for p in range(c // page, (c + n - 1) // page + 1):
                    a, b = max(c, p * page), min(c + n, (p + 1) * page)
                    cache[int(s["table"][i, p]), a - p * page:b - p * page] = x[a - c:b - c]
                continue
            lead, f = c % sb, c - c % sb
            tail = -(c + n) % sb
            z = torch.cat((_line(s, i, f, c, which) if lead else x[:0], x, x.new_zeros(tail, *x.shape[1:])))
            z = z.view(-1, sb, *x.shape[1:])                          # (blocks, block, heads, dim)
            mine = z.clone()
            mine[0, :lead] = 0
            unit = (mine.abs().amax((1, 3)) / QMAX[case["code"]]).clamp_min(MIN_SCALE)
            blocks = torch.arange(f // sb, f // sb + len(z), device=z.device)
            pages, inner = s["table"][i].long()[blocks * sb // page], blocks * sb % page // sb
            if lead:
                was = scale[pages[0], :, inner[0]]
                unit[0] = torch.maximum(unit[0], was)
            y = _rounded(z / unit[:, None, :, None], case["code"]) * unit[:, None, :, None]
            if lead:                                                  # kept as they are where the scale stayed
                y[0, :lead] = torch.where((unit[0] > was)[:, None], y[0, :lead], z[0, :lead])
            scale[pages, :, inner] = unit
            held.append(y.flatten(0, 1)[:lead + n])
        out[which] = (cache, None) if cache is not None else (torch.cat(held), scale)
    if case["code"] == "none":
        return out["k"][0], out["v"][0]
    return out["k"][0], out["v"][0], out["k"][1], out["v"][1]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    ctx, new = _lengths(case)
    if case["op"] == "gather":
        return tuple(torch.cat([_line(s, i, 0, c, w) for i, c in enumerate(ctx)]) for w in ("k", "v"))
    hk, g, d = case["heads_k"], case["heads_q"] // case["heads_k"], case["dim"]
    outs, lses, at = [], [], 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        first = max(0, c - n - case["window"]) if case["window"] >= 0 else 0
        k, v = _line(s, i, first, c, "k"), _line(s, i, first, c, "v")
        q = _turned(s["q"][at:at + n].double(), c - n, s)
        at += n
        j = torch.arange(first, c, device=q.device)
        for t in range(n):
            a = torch.einsum("hgd,jhd->hgj", q[t].view(hk, g, d), k) / math.sqrt(d)
            if case["softcap"]:
                a = torch.tanh(a / case["softcap"]) * case["softcap"]
            if s["slopes"] is not None:
                a = a + s["slopes"].double().view(hk, g, 1) * (j - (c - n + t)).double()
            ok = j <= c - n + t
            if case["window"] >= 0:
                ok &= j >= c - n + t - case["window"]
            a = a[..., ok]
            lse = torch.logsumexp(a, -1)
            outs.append(torch.einsum("hgj,jhd->hgd", (a - lse[..., None]).exp(), v[ok]).reshape(hk * g, d))
            lses.append(lse.reshape(-1))
    return torch.stack(outs), torch.stack(lses, 1)
