"""Linear attention with a decay per head on the GPU, against the 64-bit formulas of lin_ref."""
import pytest
import torch

import fable_attn as fa
import lin_ref as R

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ALL = ["bf16", "fp16", "fp32"]
SLOT = 131072          # device error bit of a state slot outside the pool or named twice


def rand(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def decays(hk, kind="mixed"):
    if kind == "mixed":      # none, slow, fast, only the token itself
        return torch.tensor([0.0, -0.003, -0.9, float("-inf"), -0.05][:hk] + [-0.01] * max(0, hk - 5)).cuda()
    return torch.full((hk,), float(kind)).cuda()


def inputs(dt, lens, hq, hk, dk, dv, seed=0):
    n = sum(lens)
    return rand(seed, n, hq, dk, dtype=dt), rand(seed + 1, n, hk, dk, dtype=dt), rand(seed + 2, n, hk, dv, dtype=dt)


def cum(lens, first=0):
    c = [first]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device="cuda")


def check_run(dt, lens, hq, hk, dk, dv, g, carried, varlen, seed=0, grads=True, strided=False):
    q, k, v = inputs(dt, lens, hq, hk, dk, dv, seed)
    if strided:              # slices of one packed projection
        rows = torch.cat([x.flatten(1) for x in (q, k, v)], 1)
        q, k, v = (x.view(len(rows), h, d) for x, h, d in zip(rows.split([hq * dk, hk * dk, hk * dv], 1), (hq, hk, hk), (dk, dk, dv)))
    b = len(lens)
    s0, ds = (rand(seed + 3, b, hk, dk, dv), rand(seed + 4, b, hk, dk, dv)) if carried else (None, None)
    do = rand(seed + 5, sum(lens), hq, dv, dtype=dt)
    leaves = [x.detach().requires_grad_(grads) for x in (q, k, v)] + ([s0.requires_grad_(grads)] if carried else [])
    scale = dk ** -0.5
    if varlen:
        res = fa.linear_attn_varlen_func(*leaves[:3], g, cum(lens), max(lens), initial_state=s0, return_final_state=True)
    else:
        shaped = [x.view(b, lens[0], *x.shape[1:]) for x in leaves[:3]]
        res = fa.linear_attn_func(*shaped, g, initial_state=s0, return_final_state=True)
    out, final = res[0].reshape(sum(lens), hq, dv), res[1]
    got = [out, final]
    if grads:
        got += list(torch.autograd.grad(res, leaves, (do.view(res[0].shape), ds if carried else None),
                                        allow_unused=True)) if carried else list(
            torch.autograd.grad(res[0], leaves, do.view(res[0].shape)))
    at = 0
    for z, n in enumerate(lens):
        s = slice(at, at + n)
        at += n
        ref = R.both(q[s], k[s], v[s], g, scale, s0[z] if carried else None, do[s] if grads else None, ds[z] if carried else None)
        parts = [out[s], final[z]]
        if grads:
            parts += [x[s] for x in got[2:5]] + ([got[5][z]] if carried else [])
        for name, x, (want, amp) in zip(("out", "final", "dq", "dk", "dv", "dinitial"), parts, ref):
            R.close(x, want, amp, n * max(1, hq // hk), (dk, dv), g, dt, f"{name} of sequence {z}")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n", [1, 2, 31, 33, 127, 128, 129, 257, 700])
def test_lengths(dt, n):
    check_run(DT[dt], [n] * 2, 4, 4, 64, 64, decays(4), True, False, seed=n)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (80, 96), (32, 32), (8, 8), (96, 40), (256, 256), (160, 16)])
def test_head_dims(dt, dk, dv):
    check_run(DT[dt], [150], 2, 2, dk, dv, decays(2), True, False)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("hq,hk", [(4, 1), (6, 2), (8, 8), (9, 3)])
@pytest.mark.parametrize("d", [64, 128])
def test_shared_heads(dt, hq, hk, d):
    check_run(DT[dt], [140, 140], hq, hk, d, d, decays(hk), True, False)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("carried", [False, True])
def test_ragged(dt, carried):
    check_run(DT[dt], [5, 0, 300, 1, 128, 129, 64], 4, 2, 64, 64, decays(2), carried, True)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("g", ["0", "-0.0001", "-0.3", "-4", "-60", "-inf"])
def test_decays(dt, g):
    check_run(DT[dt], [260], 2, 2, 128, 128, decays(2, g), True, False)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("g", ["-7", "-9", "-12", "-16"])
def test_states_of_fast_decays(dt, g):
    """Rows whose decay takes them below fp16's smallest step, next to elements of the state that are as small."""
    check_run(DT[dt], list(range(1, 41)), 8, 8, 72, 64, decays(8, g), True, True)
    check_run(DT[dt], [130], 4, 4, 128, 128, decays(4, g), True, False)


@pytest.mark.parametrize("dt", ALL)
def test_many_segments(dt):
    check_run(DT[dt], [2500], 2, 1, 64, 64, decays(1, "-0.01"), True, False)
    check_run(DT[dt], [2500, 40, 1300], 2, 2, 128, 128, decays(2), True, True)


@pytest.mark.parametrize("dt", ALL)
def test_one_state_many_sequences(dt):
    check_run(DT[dt], [40] * 200, 4, 4, 32, 32, decays(4), True, False)


@pytest.mark.parametrize("dt", ALL)
def test_strided_inputs(dt):
    check_run(DT[dt], [3, 200, 77], 4, 2, 64, 64, decays(2), False, True, strided=True)


@pytest.mark.parametrize("dt,dk,dv", [("fp32", 64, 64), ("fp32", 128, 72), ("fp32", 200, 136), ("bf16", 160, 160), ("fp16", 256, 8)])
@pytest.mark.parametrize("hq,hk", [(4, 4), (6, 2), (2, 2)])
def test_cuda_core_chunks_of_64(dt, dk, dv, hq, hk):
    """More heads than the SMs hold blocks of (chunks of 64 tokens), and one long sequence (segments of several chunks)."""
    cols = (dv + 63) // 64
    check_run(DT[dt], [70] * (300 // (hk * cols) + 1), hq, hk, dk, dv, decays(hk), True, False)
    lens = [0, 1, 63, 64, 65, 130, 31]
    check_run(DT[dt], lens * (600 // (hk * cols * len(lens)) + 1), hq, hk, dk, dv, decays(hk), True, True)
    if hq == hk == 2:
        check_run(DT[dt], [12000 // cols], hq, hk, dk, dv, decays(hk), True, False, grads=dt == "fp32")


@pytest.mark.parametrize("dt,d", [("fp32", 64), ("fp32", 136), ("bf16", 136)])
@pytest.mark.parametrize("n", [150, 5000])
def test_cuda_core_rows_at_odd_places(dt, d, n):
    """Elements one at a time where four are not on their boundary: the same bits."""
    dt, h = DT[dt], 4
    wide = rand(0, 2, n, 3 * h * d + 3, dtype=dt)
    q, k, v = (wide[..., 1 + i * h * d:1 + (i + 1) * h * d].unflatten(-1, (h, d)).requires_grad_() for i in range(3))
    near = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for x in (q, k, v)]
    do = rand(1, 2, n, h, d + 1, dtype=dt)[..., 1:]
    a, b = fa.linear_attn_func(q, k, v, decays(h)), fa.linear_attn_func(*near, decays(h))
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, (q, k, v), do), torch.autograd.grad(b, near, do.contiguous())):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_rows_off_sixteen_bytes_and_repeated_heads(dt):
    """Slices at odd places, a head that serves all, a gradient that is one row for all tokens: the same bits as of whole copies."""
    dt, n, h, d = DT[dt], 150, 4, 64
    wide = rand(0, n, 3 * h * d + 5, dtype=dt)
    q, k, v = (wide[:, 3 + i * h * d:3 + (i + 1) * h * d].view(n, h, d)[None].requires_grad_() for i in range(3))
    g, do = decays(h), rand(1, 1, 1, h, d, dtype=dt).expand(1, n, h, d)
    near = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for x in (q, k, v)]
    a, b = fa.linear_attn_func(q, k, v, g), fa.linear_attn_func(*near, g)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, (q, k, v), do), torch.autograd.grad(b, near, do.contiguous())):
        assert torch.equal(x, y)
    one = near[1].detach()[:, :, :1].expand(1, n, h, d)
    assert torch.equal(fa.linear_attn_func(near[0], one, near[2], g), fa.linear_attn_func(near[0], one.contiguous(), near[2], g))


def test_positive_decay_counts_as_none_and_nan_shows():
    q, k, v = inputs(torch.bfloat16, [130], 2, 2, 64, 64)
    g = torch.tensor([0.5, 0.0]).cuda()
    a, b = (fa.linear_attn_func(q[None], k[None], v[None], x) for x in (g, torch.zeros(2).cuda()))
    assert torch.equal(a, b)
    c = fa.linear_attn_func(q[None], k[None], v[None], torch.tensor([float("nan"), 0.0]).cuda())
    assert c[:, :, 0].isnan().all() and torch.equal(c[:, :, 1], b[:, :, 1])


def test_layouts_agree():
    """Batch-major, sequence-major and transposed-head tensors give the same bits, and so does a one-entry dimension of any stride."""
    b, n, h, d = 3, 140, 4, 64
    x = [rand(i, b, n, h, d, dtype=torch.bfloat16) for i in range(3)]
    g = decays(h)
    want = fa.linear_attn_func(*x, g)
    seq = [y.transpose(0, 1).contiguous().transpose(0, 1) for y in x]
    heads = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in x]
    odd = [torch.empty(b, n, h, d + 3, dtype=torch.bfloat16, device="cuda")[..., :d].copy_(y) for y in x]
    for y in (seq, heads, odd):
        assert torch.equal(fa.linear_attn_func(*y, g), want) or torch.allclose(fa.linear_attn_func(*y, g).float(), want.float(), rtol=2 ** -7, atol=2 ** -9 * d ** 0.5)
    one = [y[:1].as_strided((1, n, h, d), (7, h * d, d, 1)) for y in x]
    assert torch.equal(fa.linear_attn_func(*one, g), fa.linear_attn_func(*[y[:1] for y in x], g))


def test_gradients_against_differences():
    """out and final are linear in each of q, k, v and the initial state by itself, so a difference over any step is exact but for
    the forward's own error; fp32, so that it is small."""
    b, n, hq, hk, d = 2, 150, 4, 2, 64
    x = [rand(0, b, n, hq, d), rand(1, b, n, hk, d), rand(2, b, n, hk, d), rand(3, b, hk, d, d)]
    do, ds, g = rand(4, b, n, hq, d), rand(5, b, hk, d, d), torch.tensor([-0.02, -0.4]).cuda()
    run = lambda y: fa.linear_attn_func(*y[:3], g, initial_state=y[3], return_final_state=True)
    loss = lambda y: sum((p.double() * w.double()).sum() for p, w in zip(run(y), (do, ds)))
    size = lambda y: sum((p.double().abs() * w.double().abs()).sum() for p, w in zip(run(y), (do, ds)))
    leaves = [y.clone().requires_grad_() for y in x]
    grads = torch.autograd.grad(run(leaves), leaves, (do, ds))
    for i in range(4):
        step = rand(10 + i, *x[i].shape)
        up, down = ([y + s * step if j == i else y for j, y in enumerate(x)] for s in (1.0, -1.0))
        diff = float(loss(up) - loss(down)) / 2
        # each element of the four results carries at most (n + 3 d + 64) roundings of 2^-24 of its terms' sizes, here taken as 8 times the result's
        # own size (64 terms of random sign sum to an eighth of their sizes)
        bound = 8 * (n + 3 * d + 64) * 2.0 ** -24 * float(size(up) + size(down) + (grads[i].double().abs() * step.double().abs()).sum())
        assert abs(diff - float((grads[i].double() * step.double()).sum())) <= bound


def test_gradient_of_each_output_alone():
    q, k, v = (x[None].requires_grad_() for x in inputs(torch.bfloat16, [140], 2, 2, 64, 64))
    s0 = rand(9, 1, 2, 64, 64).requires_grad_()
    g = decays(2)
    out, final = fa.linear_attn_func(q, k, v, g, initial_state=s0, return_final_state=True)
    do, ds = rand(4, 1, 140, 2, 64, dtype=torch.bfloat16), rand(5, 1, 2, 64, 64)
    a = torch.autograd.grad(out, (q, k, v, s0), do, retain_graph=True)
    b = torch.autograd.grad(final, (q, k, v, s0), ds)
    r1 = R.both(q[0], k[0], v[0], g, 0.125, s0[0], do[0])
    r2 = R.both(q[0], k[0], v[0], g, 0.125, s0[0], torch.zeros_like(do[0]), ds[0])
    for got, ref in ((a, r1), (b, r2)):
        for x, (want, amp) in zip(got, ref[2:]):
            R.close(x[0], want, amp, 140, (64, 64), g, torch.bfloat16)
    assert torch.equal(b[0], torch.zeros_like(b[0]))


def test_broadcast_gradient_and_shared_leaf():
    """The gradient of a sum is one element seen everywhere; k and v that are one tensor get both shares."""
    q, k, _ = inputs(torch.float32, [70], 2, 2, 64, 64)
    q, k, g = q[None], k[None].requires_grad_(), torch.tensor([-0.1, 0.0]).cuda()
    got, = torch.autograd.grad(fa.linear_attn_func(q, k, k, g).sum(), k)
    r = R.both(q[0], k[0], k[0], g, 0.125, None, torch.ones(70, 2, 64))
    R.close(got[0], r[3][0] + r[4][0], r[3][1] + r[4][1], 70, (64, 64), g, torch.float32)


def test_runs_repeat():
    q, k, v = (x[None].requires_grad_() for x in inputs(torch.bfloat16, [1500], 8, 2, 64, 64))
    do, g = rand(4, 1, 1500, 8, 64, dtype=torch.bfloat16), decays(2)
    runs = []
    for _ in range(3):
        out = fa.linear_attn_func(q, k, v, g)
        runs.append((out,) + torch.autograd.grad(out, (q, k, v), do))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [64, 256])
def test_rows_of_no_sequence(dt, d):
    """Rows before the first and behind the last sequence give 0, and what stands there, NaN and infinities, reaches nobody."""
    lens, pad = [130, 40], 9
    q, k, v = inputs(DT[dt], [pad] + lens + [pad], 2, 2, d, d)
    for x in (q, k, v):
        x[:pad], x[-pad:] = float("nan"), float("inf")
    g, do = decays(2, "-0.1"), rand(7, len(q), 2, d, dtype=DT[dt])
    clean = [x[pad:-pad].clone().requires_grad_() for x in (q, k, v)]
    want = fa.linear_attn_varlen_func(*clean, g, cum(lens), 130)
    wg = torch.autograd.grad(want, clean, do[pad:-pad])
    leaves = [x.requires_grad_() for x in (q, k, v)]
    do[:pad], do[-pad:] = float("nan"), float("nan")
    got = fa.linear_attn_varlen_func(*leaves, g, cum(lens, pad), 130)
    gg = torch.autograd.grad(got, leaves, do)
    for a, b in zip((want,) + wg, (got,) + gg):
        assert torch.equal(a, b[pad:-pad]) and not b[:pad].any() and not b[-pad:].any()


@pytest.mark.parametrize("dt", ALL)
def test_nan_stays_in_its_sequence_and_head(dt):
    lens = [60, 90, 61]
    q, k, v = inputs(DT[dt], lens, 2, 2, 64, 64)
    g = decays(2, "-0.1")
    clean = fa.linear_attn_varlen_func(q, k, v, g, cum(lens), 90)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for x in (q, k, v):
            y = x.clone()
            y[75, 1, 3] = bad                       # in the second sequence, head 1
            args = [y if t is x else t for t in (q, k, v)]
            out = fa.linear_attn_varlen_func(*args, g, cum(lens), 90)
            assert torch.equal(out[:, 0], clean[:, 0])
            assert torch.equal(out[:60], clean[:60]) and torch.equal(out[150:], clean[150:])
            assert not out[75, 1].isfinite().all()


def test_too_small_a_bound_and_bad_offsets():
    lens = [300, 20]
    q, k, v = inputs(torch.bfloat16, lens, 2, 2, 64, 64)
    g = decays(2)
    want = fa.linear_attn_varlen_func(q, k, v, g, cum(lens), 300)
    for bound in (17, 128, 1000000):
        got = fa.linear_attn_varlen_func(q, k, v, g, cum(lens), bound)
        assert torch.allclose(got.float(), want.float(), rtol=2 ** -6, atol=2 ** -5)
    wild = torch.tensor([0, 300, 2000000000], dtype=torch.int32, device="cuda")      # offsets past the rows end there
    assert torch.equal(fa.linear_attn_varlen_func(q, k, v, g, wild, 300)[:300], want[:300])
    back = torch.tensor([-5, 300, 100], dtype=torch.int32, device="cuda")            # a length below 0 is 0
    assert torch.equal(fa.linear_attn_varlen_func(q, k, v, g, back, 300)[:300], want[:300])


def test_empty_calls():
    g = decays(2)
    x = torch.empty(2, 0, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    s0 = rand(1, 2, 2, 64, 64).requires_grad_()
    out, final = fa.linear_attn_func(x, x, x, g, initial_state=s0, return_final_state=True)
    assert out.shape == x.shape and torch.equal(final, s0)
    assert torch.equal(torch.autograd.grad(final.sum(), s0)[0], torch.ones_like(s0))
    none = torch.empty(0, 5, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert fa.linear_attn_func(none, none, none, g).shape == none.shape
    packed = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    out, final = fa.linear_attn_varlen_func(packed, packed, packed, g, cum([0, 0]), 0, initial_state=s0.detach(), return_final_state=True)
    assert torch.equal(final, s0)


# ------------------------------------------------------------------ serving
def served(dt, lens, hq, hk, dk, dv, seed, slots=None, **kw):
    q, k, v = inputs(dt, lens, hq, hk, dk, dv, seed)
    b = len(lens)
    slots = slots or b + 3
    state = rand(seed + 3, slots, hk, dk, dv)
    perm = torch.randperm(slots, generator=torch.Generator().manual_seed(seed))[:b].to(torch.int32).cuda()
    return q, k, v, state, perm


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("lens", [[1], [1] * 9, [3, 1, 4, 0, 2], [16, 7], [17, 5], [40, 300, 0, 1, 128]])
@pytest.mark.parametrize("hq,hk,dk,dv", [(4, 4, 64, 64), (12, 2, 128, 128), (3, 3, 80, 96), (2, 1, 256, 256), (6, 1, 8, 40)])
def test_states_in_a_pool(dt, lens, hq, hk, dk, dv):
    q, k, v, state, at = served(DT[dt], lens, hq, hk, dk, dv, len(lens))
    g, before = decays(hk), state.clone()
    other = torch.full_like(state, 7.0)
    out = fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cu_seqlens=cum(lens), max_seqlen=max(lens), state_out=other)
    assert torch.equal(state, before)
    again = fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cu_seqlens=cum(lens), max_seqlen=max(lens))
    assert torch.equal(again, out)
    row = 0
    for z, n in enumerate(lens):
        s, slot = slice(row, row + n), int(at[z])
        row += n
        ref = R.both(q[s], k[s], v[s], g, dk ** -0.5, before[slot])
        for x, (want, amp) in zip((out[s], other[slot]), ref):
            R.close(x, want, amp, n, (dk, dv), g, DT[dt], f"sequence {z}")
        assert torch.equal(state[slot], other[slot])
    rest = [i for i in range(len(state)) if i not in at.tolist()]
    assert torch.equal(state[rest], before[rest]) and bool((other[rest] == 7).all())


@pytest.mark.parametrize("n", [1, 5, 200])
def test_padding_fresh_and_refused_slots(n):
    lens = [n] * 6
    q, k, v, state, _ = served(torch.bfloat16, lens, 4, 2, 64, 64, 3, slots=5)
    g, before = decays(2), state.clone()
    before[0] = state[0] = float("nan")             # what a slot held does not matter where the sequence is new
    at = torch.tensor([2, -1, 0, 2, 5, 4], dtype=torch.int32).cuda()     # padding, a slot named twice, one outside
    seen = torch.tensor([3, 3, 0, 3, 3, 9], dtype=torch.int32).cuda()
    fa.device_error(clear=True)
    out = fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cache_seqlens=seen, cu_seqlens=cum(lens), max_seqlen=n)
    assert fa.device_error(clear=True) == SLOT
    for z, fine in enumerate([True, False, True, False, False, True]):
        s = slice(z * n, z * n + n)
        if not fine:
            assert not out[s].any()
            continue
        ref = R.both(q[s], k[s], v[s], g, 0.125, before[int(at[z])] if int(seen[z]) else None)
        R.close(out[s], *ref[0], n, (64, 64), g, torch.bfloat16)
        R.close(state[int(at[z])], *ref[1], n, (64, 64), g, torch.bfloat16)
    assert torch.equal(state[[1, 3]], before[[1, 3]])
    pad = torch.full((6,), -1, dtype=torch.int32).cuda()
    assert not fa.linear_attn_with_state(q, k, v, state, g, state_indices=pad, cu_seqlens=cum(lens), max_seqlen=n).any()
    assert fa.device_error() == 0


@pytest.mark.parametrize("n", [2, 40])
def test_padded_serving_batch(n):
    """A batch padded for a captured graph: rows behind the last sequence and sequences of no tokens."""
    lens = [n, n - 1, 0, 0]
    q, k, v, state, at = served(torch.bfloat16, lens + [6], 2, 2, 64, 64, 5)
    at, g = at[:4].clone(), decays(2)
    at[2:] = -1
    q[-6:], k[-6:], v[-6:] = float("nan"), float("nan"), float("nan")
    before = state.clone()
    out = fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cu_seqlens=cum(lens), max_seqlen=n)
    assert not out[-6:].any()
    for z, m in ((0, n), (1, n - 1)):
        s = slice(z * n, z * n + m)
        R.close(out[s], *R.both(q[s], k[s], v[s], g, 0.125, before[int(at[z])])[0], n, (64, 64), g, torch.bfloat16)


@pytest.mark.parametrize("dt", ALL)
def test_dense_batch_and_pieces(dt):
    """A prompt in two pieces and then single tokens is the whole sequence."""
    b, n, h, d = 3, 300, 4, 64
    x = [rand(i, b, n, h, d, dtype=DT[dt]) for i in range(3)]
    g, state = decays(h), torch.full((b, h, d, d), float("nan"), device="cuda")
    outs, at = [], 0
    for piece in (170, 126, 1, 2, 1):
        seen = torch.full((b,), at, dtype=torch.int32).cuda()
        outs.append(fa.linear_attn_with_state(*[y[:, at:at + piece] for y in x], state, g, cache_seqlens=seen))
        at += piece
    out = torch.cat(outs, 1)
    for z in range(b):
        ref = R.both(*[y[z] for y in x], g, d ** -0.5)
        R.close(out[z], *ref[0], n, (d, d), g, DT[dt])
        R.close(state[z], *ref[1], n, (d, d), g, DT[dt])


@pytest.mark.parametrize("n", [1, 200])
def test_captured_and_replayed(n):
    """A captured step follows the buffers' new contents, on a stream of its own, beside another graph that shares its memory pool."""
    lens = [n, n]
    q, k, v, state, at = served(torch.bfloat16, lens, 4, 2, 128, 128, 8)
    g, cu, new = decays(2), cum(lens), torch.zeros_like(state)
    call = lambda: fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cu_seqlens=cu, max_seqlen=n, state_out=new)
    call()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(call())
        graphs.append(graph)
    for turn in range(2):
        q.copy_(rand(50 + turn, *q.shape, dtype=q.dtype))
        want, swant = call().clone(), new.clone()
        new.zero_()
        graphs[turn].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn], want) and torch.equal(new, swant)


def test_captured_training_step():
    q, k, v = (x[None].requires_grad_() for x in inputs(torch.bfloat16, [300], 4, 2, 64, 64))
    do, g = rand(4, 1, 300, 4, 64, dtype=torch.bfloat16), decays(2)

    def step():
        out = fa.linear_attn_func(q, k, v, g)
        return (out,) + torch.autograd.grad(out, (q, k, v), do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        q.copy_(rand(77, *q.shape, dtype=q.dtype))
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in got]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_other_stream_and_no_synchronisation():
    q, k, v, state, at = served(torch.bfloat16, [1] * 5, 4, 2, 64, 64, 9)
    lq, lk, lv = (x[None].requires_grad_() for x in inputs(torch.bfloat16, [400], 4, 2, 64, 64))
    g, cu = decays(2), cum([1] * 5)
    fa.linear_attn_with_state(q, k, v, state.clone(), g, state_indices=at, cu_seqlens=cu, max_seqlen=1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with torch.cuda.stream(side):
            big = torch.zeros(64 << 20, device="cuda")
            big.add_(1)
            lq2 = lq.detach().mul(2).requires_grad_()
            out = fa.linear_attn_func(lq2, lk, lv, g)
            grad, = torch.autograd.grad(out, lq2, out)
            fa.linear_attn_with_state(q, k, v, state, g, state_indices=at, cu_seqlens=cu, max_seqlen=1)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    side.synchronize()
    want = fa.linear_attn_func(lq.detach().mul(2), lk, lv, g)
    assert torch.equal(out, want) and grad.isfinite().all()


def test_far_addresses():
    """Rows and slots past 2^31 elements."""
    n, h, d = 130, 2, 64
    step = (1 << 31) + 4096
    buf = torch.empty(step + n * 3 * h * d, dtype=torch.bfloat16, device="cuda")
    x = []
    for i in range(3):
        y = buf[i * h * d:].as_strided((2, n, h, d), (step, 3 * h * d, d, 1))
        y.copy_(rand(i, 2, n, h, d, dtype=torch.bfloat16))
        x.append(y)
    g = decays(h)
    leaves = [y.detach().requires_grad_() for y in x]
    near = [y.contiguous().requires_grad_() for y in x]
    do = rand(5, 2, n, h, d, dtype=torch.bfloat16)
    a, b = fa.linear_attn_func(*leaves, g), fa.linear_attn_func(*near, g)
    assert torch.equal(a, b)
    for s, t in zip(torch.autograd.grad(a, leaves, do), torch.autograd.grad(b, near, do)):
        assert torch.equal(s, t)
    del buf, x, leaves, a
    slots = (1 << 31) // (h * d * d) + 3
    pool = torch.empty(slots, h, d, d, device="cuda")
    at = torch.tensor([slots - 1, 0], dtype=torch.int32).cuda()
    for m in (1, 130):
        pool[[0, slots - 1]] = rand(9, 2, h, d, d)
        small = pool[[slots - 1, 0]].clone()
        y = [rand(20 + i, 2, m, h, d, dtype=torch.bfloat16) for i in range(3)]
        assert torch.equal(fa.linear_attn_with_state(*y, pool, g, state_indices=at), fa.linear_attn_with_state(*y, small, g))
        assert torch.equal(pool[[slots - 1, 0]], small)


@pytest.mark.parametrize("other", [False, True])
def test_state_saved_for_a_gradient_and_then_written(other):
    q, k, v = (rand(i, 2, 40, 2, 64, dtype=torch.bfloat16).requires_grad_() for i in range(3))
    state, g = rand(4, 2, 2, 64, 64), decays(2)
    near = [x.detach() for x in (q, k, v)]
    out = fa.linear_attn_func(q, k, v, g, initial_state=state)
    fa.linear_attn_with_state(*near, state.clone() if other else state, g, state_out=state if other else None)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with torch.inference_mode():
        pool = torch.zeros(2, 2, 64, 64, device="cuda")
        fa.linear_attn_with_state(*near, pool, g)
    assert pool.any()


@pytest.mark.parametrize("bad", ["fp64", "heads", "dims", "batch", "decay", "decay_grad", "state", "state_grad", "slots", "index", "cpu", "dim7", "rank", "device_state", "overlap"])
def test_refusals(bad):
    b, n, h, d = 2, 20, 4, 64
    q, k, v = (rand(i, b, n, h, d, dtype=torch.bfloat16) for i in range(3))
    g, state, kw = decays(h), rand(5, b, h, d, d), {}
    err = ValueError
    if bad == "fp64": q, k, v = q.double(), k.double(), v.double()
    if bad == "heads": k, v = k[:, :, :3], v[:, :, :3]
    if bad == "dims": k = k[..., :32]
    if bad == "batch": v = v[:1]
    if bad == "decay": g = g[:2]
    if bad == "decay_grad": g, err = g.requires_grad_(), NotImplementedError
    if bad == "state": state = state.half()
    if bad == "state_grad": state, err = state.requires_grad_(), NotImplementedError
    if bad == "slots": state = rand(5, b + 1, h, d, d)
    if bad == "index": kw["state_indices"] = torch.zeros(3, dtype=torch.int32).cuda()
    if bad == "cpu": q = q.cpu()
    if bad == "dim7": q, k, v, state = q[..., :7], k[..., :7], v[..., :7], state[..., :7, :7].contiguous()
    if bad == "rank": q, k, v = q[0], k[0], v[0]
    if bad == "device_state": state = state.cpu()
    if bad == "overlap":
        pool = rand(5, b + 1, h, d, d)
        state, kw["state_out"], err = pool[:-1], pool[1:], RuntimeError
    with pytest.raises(err):
        fa.linear_attn_with_state(q, k, v, state, g, **kw)
    if bad not in ("state", "state_grad", "slots", "index", "device_state", "overlap"):
        with pytest.raises(err):
            fa.linear_attn_func(q, k, v, g)


@pytest.mark.parametrize("dt", ALL)
def test_workspace_follows_the_rows_and_not_the_bound(dt):
    """Many short sequences beside a long one, without a bound on the lengths: segments are counted by the rows."""
    lens = [3000] + [1, 0, 20] * 40 + [700]
    q, k, v = inputs(DT[dt], lens, 2, 2, 64, 64)
    state = torch.randn(len(lens), 2, 64, 64, device="cuda")
    g, before = decays(2, "-0.01"), state.clone()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    out = fa.linear_attn_with_state(q, k, v, state, g, cu_seqlens=cum(lens))
    assert torch.cuda.max_memory_allocated() - held < 64 << 20
    at = 0
    for z, n in enumerate(lens):
        s = slice(at, at + n)
        at += n
        if z in (0, 1, 2, 3, 60, len(lens) - 1):
            ref = R.both(q[s], k[s], v[s], g, 0.125, before[z])
            R.close(out[s], *ref[0], n, (64, 64), g, DT[dt], f"sequence {z}")
            R.close(state[z], *ref[1], n, (64, 64), g, DT[dt], f"state {z}")
