"""Workloads of linear attention with a decay per head, and of rotary positions scaled for long contexts.

    train   linear_attn_func, forward and backward: per kv head lam = exp(log_decay), S_t = lam S_{t-1} + k_t v_t^T and
            o_t = scale S_t^T q_t; with `carried`, S starts from a given state and the last one is returned, both with gradients.
    serve   linear_attn_with_state: packed tokens of a batch continue states that live in a pool, found by state_indices;
            prompts of thousands of tokens, or one or a few tokens of a decode step.  The new states go to a second
            pool, as where drafted tokens may be taken back.
    rotary  apply_rotary_emb_qk: q and k turned by their tokens' own positions, with frequencies scaled as YaRN does;
            with `backward` the gradients are turned back too.

`run` computes them with elementary torch operations (linear attention in chunks, as matrix products), or, with `own` set,
through fable_attn.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CASE = dict(op="", dtype="bf16", batch=1, heads_q=8, heads_k=8, dim=128, dim_v=128, lo=1, hi=1, fresh=False, carried=False,
            rotary=128, interleaved=False, far=4096, backward=False)


def _case(name, **kw):
    c = dict(CASE, **kw)
    assert not set(kw) - set(CASE)
    if "dim" in kw and "dim_v" not in kw:
        c["dim_v"] = c["dim"]
    return dict(c, name=name) if name else c


def listed():
    return [
        # a training step of one layer, the training benchmark's shape
        _case("train_fp16_step", op="train", dtype="fp16", batch=2, heads_q=32, heads_k=32, lo=4096, hi=4096),
        # heads that share keys, values and state; headdim 64, a length that ends inside a chunk
        _case("train_bf16_shared", op="train", batch=4, heads_q=16, heads_k=4, dim=64, lo=1000, hi=1000),
        # fp32, the smallest benchmark configuration
        _case("train_fp32_small", op="train", dtype="fp32", heads_q=8, heads_k=8, dim=64, lo=512, hi=512),
        # one piece of a long document: the state comes in and goes out, with its gradient
        _case("train_bf16_carried", op="train", heads_q=16, heads_k=16, lo=8192, hi=8192, carried=True),
        # the prompt of the dense forward benchmark, from an empty state
        _case("serve_bf16_prompt", op="serve", heads_q=32, heads_k=32, lo=16384, hi=16384, fresh=True),
        # 16 ragged chunks of prompts, 8 query heads for each state
        _case("serve_bf16_ragged", op="serve", batch=16, heads_q=64, heads_k=8, lo=500, hi=4096),
        # the smallest call: the next token of one chat
        _case("serve_bf16_one", op="serve", heads_q=8, heads_k=8, dim=64),
        # a decode step of a large batch
        _case("serve_bf16_step", op="serve", batch=256, heads_q=32, heads_k=32),
        # 1 to 4 drafted tokens of 24 sequences
        _case("serve_fp16_drafts", op="serve", dtype="fp16", batch=24, heads_q=32, heads_k=8, lo=1, hi=4),
        # rotary of a decode step, far into long contexts
        _case("rotary_bf16_step", op="rotary", batch=64, heads_q=32, heads_k=8, far=1000000),
        # rotary of the paged decode benchmark's heads over one long prompt
        _case("rotary_bf16_prompt", op="rotary", heads_q=32, heads_k=8, lo=16384, hi=16384, far=131072, interleaved=True),
        # rotary and its gradients in the training step, half of the head turned
        _case("rotary_fp16_train", op="rotary", dtype="fp16", batch=2, heads_q=32, heads_k=32, lo=4096, hi=4096, rotary=64,
              backward=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["train", "train", "serve", "serve", "serve", "rotary"])
    c = _case(None, op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"]))
    c["dim"] = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    c["dim_v"] = c["dim"] if rng.random() < 0.7 else rng.choice([32, 64, 80, 128])
    c["heads_k"] = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    c["heads_q"] = c["heads_k"] * (rng.choice([1, 1, 2, 3, 4, 8]) if c["heads_k"] <= 8 else 1)
    # elements of q: the largest listed prompt's, a quarter of it for a training step, and less where fp32 or steps over states cost more
    room = 16384 * 32 * 128 // (8 if c["dtype"] == "fp32" else 4 if op == "train" else 1)
    rows = max(1, room // (c["heads_q"] * max(c["dim"], c["dim_v"])))
    if op == "serve" and rng.random() < 0.5:
        c["hi"] = rng.choice([1, 1, 1, 2, 4, 8])
        c["batch"] = _log(rng, 1, max(1, min(512, 256 * 32 // c["heads_k"])))
    else:
        c["hi"] = _log(rng, 1 if op == "rotary" else 16, min(16384, rows))
        c["batch"] = _log(rng, 1, max(1, min(64, rows // c["hi"])))
    c["lo"] = c["hi"] if op == "train" else _log(rng, 1, c["hi"])
    c["fresh"] = op == "serve" and rng.random() < 0.3
    c["carried"] = op == "train" and rng.random() < 0.4
    if op == "rotary":
        c["lo"] = c["hi"]
        c["rotary"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2])
        c["interleaved"] = rng.random() < 0.5
        c["far"] = _log(rng, c["hi"], 4000000)
        c["backward"] = rng.random() < 0.4
    return c


def _lengths(case):
    """Tokens of each sequence: whole numbers of [lo, hi], both ends among them, in an order that is no order."""
    lo, hi, n = case["lo"], case["hi"], case["batch"]
    if n == 1:
        return [hi]
    got = [lo + round((hi - lo) * i / (n - 1)) for i in range(n)]
    return [got[(i * 7 + 3) % n] for i in range(n)] if n % 7 else got[::-1]


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    hq, hk, d, dv = case["heads_q"], case["heads_k"], case["dim"], case["dim_v"]
    tokens = sum(_lengths(case))
    if case["op"] == "rotary":
        turns = 2 if case["backward"] else 1
        return {"bytes": turns * 2 * tokens * (hq + hk) * d * e, "flops": turns * 3 * tokens * (hq + hk) * case["rotary"]}
    read, out = (hq + hk) * d + hk * dv, hq * dv
    step = 2 * tokens * (hq + hk) * d * dv         # a rank-one update for each state, a product for each query
    states = case["batch"] * hk * d * dv * 4
    if case["op"] == "serve":
        return {"bytes": tokens * (read + out) * e + states * (1 if case["fresh"] else 2), "flops": step}
    return {"bytes": tokens * (3 * read + 2 * out) * e + (4 * states if case["carried"] else 0), "flops": 3 * step + step // 2}


def _yarn(rotary, base, factor, original):
    """Radians for each position, fp64, and the factor that YaRN multiplies cos and sin with: frequencies that turn
    less than once over the original length are slowed by `factor`, those that turn over 32 times stay."""
    f = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    turns = original * f / (2 * math.pi)
    keep = ((turns.log() - 0.0) / math.log(32.0)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 1 + 0.1 * math.log(factor)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, hq, hk, d, dv = case["batch"], case["heads_q"], case["heads_k"], case["dim"], case["dim_v"]
    lens = _lengths(case)
    total = sum(lens)
    s = {"case": case}
    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)
    if case["op"] == "rotary":
        inv, s["factor"] = _yarn(case["rotary"], 10000.0, 16.0, 4096)
        s["inv_freq"] = inv.to(dev)
        s["q"], s["k"] = (normal(b, case["hi"], h, d).to(dt) for h in (hq, hk))
        if case["far"] > case["hi"]:                  # each sequence starts at a place of its own
            start = torch.randint(0, case["far"] - case["hi"], (b, 1), generator=gen, device=dev)
        else:
            start = torch.zeros(b, 1, dtype=torch.long, device=dev)
        s["positions"] = (start + torch.arange(case["hi"], device=dev)).to(torch.int32)
        if case["backward"]:
            s["dq"], s["dk"] = (normal(b, case["hi"], h, d).to(dt) for h in (hq, hk))
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    # factors from about exp(-1) to exp(-1/1000), as slopes of a geometric row; every draw has others
    at = (torch.arange(hk, device=dev) + torch.rand(hk, generator=gen, device=dev)) / hk
    s["log_decay"] = -torch.exp(-math.log(1000.0) * at)
    lead = (b, case["hi"]) if case["op"] == "train" else (total,)
    s["q"], s["k"] = (normal(*lead, h, d).to(dt) for h in (hq, hk))
    s["v"] = normal(*lead, hk, dv).to(dt)
    s["scale"] = d ** -0.5
    if case["op"] == "train":
        s["do"] = normal(*lead, hq, dv).to(dt)
        wanted = ["q", "k", "v"]
        if case["carried"]:
            s["initial"], s["dfinal"] = (normal(b, hk, d, dv) for _ in range(2))
            wanted.append("initial")
        for w in wanted:
            s[w].requires_grad_()
        return s
    slots = b + b // 4 + 1
    s["state"] = normal(slots, hk, d, dv)
    s["state_out"] = torch.zeros_like(s["state"])
    s["indices"] = torch.randperm(slots, generator=gen, device=dev)[:b].to(torch.int32)
    s["seen"] = torch.zeros(b, dtype=torch.int32, device=dev) if case["fresh"] else None
    s["cu"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
    return s


@functools.cache
def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-rdna2_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fable_attn
    from fable_attn.layers import rotary
    return fable_attn, rotary


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return _rotary(state)
    if case["op"] == "train":
        return _train(state)
    return _serve(state)


def _rotary(s):
    if own:
        q, k = _package()[1].apply_rotary_emb_qk(s["q"], s["k"], s["inv_freq"], s["positions"], interleaved=s["case"]["interleaved"],
                                                 factor=s["factor"])
    else:
        angle = s["positions"].double()[..., None, None] * s["inv_freq"]
        cos, sin = ((f(angle) * s["factor"]).float() for f in (torch.cos, torch.sin))
        q, k = (_turn(s[w], cos, sin, s["case"]["interleaved"]) for w in ("q", "k"))
    if not s["case"]["backward"]:
        return q, k
    return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x[..., :r].float()
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :r // 2], y[..., r // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((y.to(x.dtype), x[..., r:]), -1)


def _train(s):
    carried = s["case"]["carried"]
    leaves = (s["q"], s["k"], s["v"]) + ((s["initial"],) if carried else ())
    if own:
        got = _package()[0].linear_attn_func(s["q"], s["k"], s["v"], s["log_decay"], s["scale"],
                                             initial_state=s["initial"] if carried else None, return_final_state=carried)
        out = got[:2] if carried else (got,)
    else:
        o, final = _linear(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["initial"] if carried else None, None)
        out = (o.to(s["q"].dtype), final)[:1 + carried]
    return out + torch.autograd.grad(out, leaves, (s["do"], s["dfinal"]) if carried else (s["do"],))


def _serve(s):
    if own:
        o = _package()[0].linear_attn_with_state(s["q"], s["k"], s["v"], s["state"], s["log_decay"], s["scale"],
                                                 state_indices=s["indices"], cache_seqlens=s["seen"], cu_seqlens=s["cu"],
                                                 max_seqlen=s["case"]["hi"], state_out=s["state_out"])
        return o, s["state_out"]
    total, b, longest = s["q"].shape[0], s["case"]["batch"], s["case"]["hi"]
    cu, at = s["cu"].long(), s["indices"].long()
    lens = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(b, device=cu.device), lens, output_size=total)
    pos = torch.arange(total, device=cu.device) - cu[seq]
    token = torch.arange(longest, device=cu.device)
    rows = (cu[:-1, None] + token).clamp(max=total - 1)
    q, k, v = (s[w][rows] for w in ("q", "k", "v"))
    first = s["state"][at]
    if s["seen"] is not None:
        first = torch.where((s["seen"] > 0)[:, None, None, None], first, torch.zeros_like(first))
    o, final = _linear(q, k, v, s["log_decay"], s["scale"], first, lens)
    s["state_out"][at] = final
    return o[seq, pos].to(s["q"].dtype), s["state_out"]


def _linear(q, k, v, log_decay, scale, first, lens):
    """(o, last state) of padded sequences (batch, tokens, heads, dim) with lens tokens each (None: all), fp32, in chunks of
    up to 128 tokens: products within each chunk, and each chunk's start from the sums of those before it."""
    (b, n, hq, d), (hk, dv) = q.shape, v.shape[2:]
    c = min(128, n)
    chunks = -(-n // c)
    t = torch.arange(chunks * c, device=q.device)
    own_tokens = torch.full((b,), n, device=q.device) if lens is None else lens
    real = (t < own_tokens[:, None])[..., None, None]
    q, k, v = (torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, chunks * c - n)) for x in (q, k, v))
    k, v = (torch.where(real, x, torch.zeros_like(x)) for x in (k, v))
    q = q.view(b, chunks, c, hk, hq // hk, d).permute(0, 3, 4, 1, 2, 5)                     # b hk g chunk c d
    k, v = (x.view(b, chunks, c, hk, -1).permute(0, 3, 1, 2, 4) for x in (k, v))            # b hk chunk c d
    g = log_decay.double()
    i = torch.arange(c, device=q.device)
    def power(steps):                                                                      # lam^steps, 0 where steps < 0
        p = torch.exp(g.view(-1, *[1] * steps.dim()) * steps.clamp(min=0).double())
        return (p * (steps >= 0)).float()
    # within the chunk
    scores = (q @ k.transpose(-1, -2)[:, :, None]) * power(i[:, None] - i)[:, None, None]
    o = scores @ v[:, :, None]
    # what the chunks leave behind, and the state at each chunk's start
    left = (k * power(c - 1 - i)[:, None, :, None]).transpose(-1, -2) @ v                     # b hk chunk d dv
    m = torch.arange(chunks, device=q.device)
    start = torch.einsum("hnm,bhmx->bhnx", power((m[:, None] - 1 - m) * c), left.flatten(-2)).view(b, hk, chunks, d, dv)
    if first is not None:
        start = start + power(m * c)[:, :, None, None] * first[:, :, None].float()
    o = o + (q * power(i + 1)[:, None, None, :, None]) @ start[:, :, None]
    o = (o * scale).permute(0, 3, 4, 1, 2, 5).reshape(b, chunks * c, hq, dv)[:, :n]
    # the state after each sequence's own last token
    since = power(own_tokens[:, None] - 1 - t).view(hk, b, chunks, c).transpose(0, 1)
    final = (k * since[..., None]).flatten(2, 3).transpose(-1, -2) @ v.flatten(2, 3)
    if first is not None:
        final = final + power(own_tokens).t()[:, :, None, None] * first.float()
    return o, final


def exact(case, seed):
    """In 64 bits, one head of one sequence after the other, all pairs of tokens at once."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    lens = _lengths(case)
    if sum(n * n for n in lens) * case["heads_q"] > 16384 ** 2 * 40:
        return None
    group = case["heads_q"] // case["heads_k"]
    train = case["op"] == "train"
    with torch.no_grad():
        out = torch.zeros(s["q"].shape[:-1] + (case["dim_v"],), dtype=torch.float64, device="cuda")
        dq, dk, dv = (torch.zeros_like(s[w], dtype=torch.float64) for w in ("q", "k", "v"))
        pool = None if train else s["state_out"].double()
        finals = torch.zeros(case["batch"], case["heads_k"], case["dim"], case["dim_v"], dtype=torch.float64, device="cuda")
        dfirst = torch.zeros_like(finals)
        begin = 0
        for z, n in enumerate(lens):
            at = (z, slice(None)) if train else (slice(begin, begin + n),)
            begin += n
            steps = torch.arange(n, dtype=torch.float64, device="cuda")
            gap = steps[:, None] - steps[None, :]
            for h in range(case["heads_k"]):
                lam = torch.exp(s["log_decay"][h].double())
                decay = torch.where(gap >= 0, lam ** gap.clamp(min=0), torch.zeros_like(gap))
                k, v = s["k"][at + (h,)].double(), s["v"][at + (h,)].double()
                if train:
                    first = s["initial"][z, h].double() if case["carried"] else torch.zeros_like(finals[0, 0])
                    dlast = s["dfinal"][z, h].double() if case["carried"] else torch.zeros_like(finals[0, 0])
                else:
                    first = s["state"][int(s["indices"][z]), h].double() * (0 if case["fresh"] else 1)
                rise, fall = lam ** (steps + 1), lam ** (n - 1 - steps)
                finals[z, h] = lam ** n * first + (k * fall[:, None]).t() @ v
                for j in range(h * group, (h + 1) * group):
                    q = s["q"][at + (j,)].double() * s["scale"]
                    out[at + (j,)] = (q @ k.t() * decay) @ v + rise[:, None] * (q @ first)
                    if train:
                        do = s["do"][at + (j,)].double()
                        pairs = do @ v.t() * decay
                        dq[at + (j,)] = (pairs @ k + rise[:, None] * (do @ first.t())) * s["scale"]
                        dk[at + (h,)] += pairs.t() @ q
                        dv[at + (h,)] += (q @ k.t() * decay).t() @ do
                        dfirst[z, h] += (q * rise[:, None]).t() @ do
                if train:
                    dk[at + (h,)] += fall[:, None] * (v @ dlast.t())
                    dv[at + (h,)] += fall[:, None] * (k @ dlast)
                    dfirst[z, h] += lam ** n * dlast
                else:
                    pool[int(s["indices"][z]), h] = finals[z, h]
    if not train:
        return out, pool
    return (out, finals, dq, dk, dv, dfirst) if case["carried"] else (out, dq, dk, dv)


def _exact_rotary(s):
    case, r = s["case"], s["case"]["rotary"]
    angle = (s["positions"].double()[..., None] * s["inv_freq"])[:, :, None]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)

    def turned(x, e):
        x = x.detach().double()
        y = x[..., :r].unflatten(-1, (r // 2, 2) if case["interleaved"] else (2, r // 2))
        y = y if case["interleaved"] else y.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * e)
        y = (y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2)
        return torch.cat((y, x[..., r:]), -1)

    out = turned(s["q"], turn), turned(s["k"], turn)
    if case["backward"]:
        out += turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())
    return out
