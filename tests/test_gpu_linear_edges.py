"""Linear attention on the GPU at the edges of what it is given, against the 64-bit formulas of lin_ref."""
import ctypes as C

import pytest
import torch

import fa_abi as A
import fable_attn as fa
import lin_floor as F
import lin_ref as R
from test_gpu_linear import ALL, DT, SLOT, check_run, cum, decays, inputs, rand
from test_linear_cpu import FaLinearBwdParams, FaLinearParams

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one sequence without tokens, behind the rows
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("cu", [[512, 512], [0, 0], [256, 256], [612, 712], [384, 512]])
def test_one_empty_sequence_leaves_the_workspace_alone(dt, cu):
    """The C entries with a workspace of exactly fa_linear_plan floats: what lies behind it stays as it was, the last state is
    the first one, and so are their gradients."""
    L, dev = A.lib(), "cuda"
    L.fa_linear_plan.restype = C.c_longlong
    n, h, d = 512, 8, 128
    seg, nseg = C.c_int(), C.c_int()
    floats = L.fa_linear_plan(1, n, C.c_longlong(n), h, 1, d, d, A.DT[dt], C.byref(seg), C.byref(nseg))
    assert nseg.value > 1 and floats == -(-n // seg.value) * h * d * d
    guard = 2 * h * d * d
    # room for a slot on each side, so that even a write past the workspace stays in this test's memory
    states, work = (torch.full((floats + 2 * guard,), 7.0, device=dev) for _ in range(2))
    q, k, v, do = (rand(i, n, h, d, dtype=DT[dt]) for i in range(4))
    o, dq, dk, dv = (torch.full_like(q, 3.0) for _ in range(4))
    s0, ds = rand(5, 1, h, d, d), rand(6, 1, h, d, d)
    s1, ds0 = torch.empty_like(s0), torch.empty_like(s0)
    g, cut = decays(h), torch.tensor(cu, dtype=torch.int32, device=dev)
    rows = A.FaStrides(0, d, h * d)
    inside = lambda x: A.ptr(x[guard:])
    p = FaLinearParams(struct_size=C.sizeof(FaLinearParams), q=A.ptr(q), k=A.ptr(k), v=A.ptr(v), o=A.ptr(o), sQ=rows, sK=rows, sV=rows, sO=rows,
                       log_decay=A.ptr(g), state_in=A.ptr(s0), state_out=A.ptr(s1), slots=1, cu=A.ptr(cut), total=n, batch=1, S=n, NH=h, gqa=1,
                       dk=d, dv=d, scale=0.125, seg_len=seg.value, nseg=nseg.value, keep_states=1, states=inside(states))
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    A.check(L.fa_linear_launch(C.byref(p), A.DT[dt], st))
    b = FaLinearBwdParams(struct_size=C.sizeof(FaLinearBwdParams), q=A.ptr(q), k=A.ptr(k), v=A.ptr(v), dO=A.ptr(do), dQ=A.ptr(dq), dK=A.ptr(dk),
                          dV=A.ptr(dv), sQ=rows, sK=rows, sV=rows, sdO=rows, sdQ=rows, sdK=rows, sdV=rows, log_decay=A.ptr(g), initial=A.ptr(s0),
                          dfinal=A.ptr(ds), dinitial=A.ptr(ds0), cu=A.ptr(cut), total=n, batch=1, S=n, NH=h, gqa=1, dk=d, dv=d, scale=0.125,
                          seg_len=seg.value, nseg=nseg.value, states=inside(states), work=inside(work))
    A.check(L.fa_linear_backward_launch(C.byref(b), A.DT[dt], st))
    torch.cuda.synchronize()
    for x in (states, work):
        assert bool((x[:guard] == 7).all()) and bool((x[guard + floats:] == 7).all())
    lo, hi = min(cu[0], n), min(cu[1], n)
    for x in (o, dq, dk, dv):
        assert not x[:lo].any() and not x[hi:].any()
    if hi == lo:
        assert torch.equal(s1, s0) and torch.equal(ds0, ds)
        return
    ref = R.both(q[lo:hi], k[lo:hi], v[lo:hi], g, 0.125, s0[0], do[lo:hi], ds[0])
    for x, (want, amp), name in zip((o[lo:hi], s1[0], dq[lo:hi], dk[lo:hi], dv[lo:hi], ds0[0]), ref, ("o", "final", "dq", "dk", "dv", "dinitial")):
        R.close(x, want, amp, hi - lo, (d, d), g, DT[dt], name)


@pytest.mark.parametrize("dt", ALL)
def test_one_empty_sequence(dt):
    n, h, d = 512, 8, 128
    q, k, v = (x.requires_grad_() for x in inputs(DT[dt], [n], h, h, d, d))
    s0, ds, g = rand(5, 1, h, d, d).requires_grad_(), rand(6, 1, h, d, d), decays(h)
    cu = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    out, final = fa.linear_attn_varlen_func(q, k, v, g, cu, n, initial_state=s0, return_final_state=True)
    assert torch.equal(final, s0) and not out.any()
    grads = torch.autograd.grad((out, final), (q, k, v, s0), (torch.ones_like(out), ds))
    assert not any(x.any() for x in grads[:3]) and torch.equal(grads[3], ds)
    pool = s0.detach().clone()
    with torch.no_grad():
        assert not fa.linear_attn_with_state(q, k, v, pool, g, cu_seqlens=cu).any()
    assert torch.equal(pool, s0)


# ------------------------------------------------------------------ operands of other sizes than 1
def check_sizes(dt, n, hq, hk, d, g, sizes, carried=False, scale=None, seed=0):
    """check_run of test_gpu_linear for one sequence, with q, k, v, dO (and the states) of given sizes and bounds that follow them."""
    q, k, v = inputs(dt, [n], hq, hk, d, d, seed)
    do = rand(seed + 5, n, hq, d, dtype=dt)
    q, k, v, do = ((x.float() * s).to(dt) for x, s in zip((q, k, v, do), sizes))
    s0, ds = (rand(seed + 3, 1, hk, d, d) * sizes[4], rand(seed + 4, 1, hk, d, d) * sizes[5]) if carried else (None, None)
    leaves = [x[None].requires_grad_() for x in (q, k, v)] + ([s0.requires_grad_()] if carried else [])
    scale = d ** -0.5 if scale is None else scale
    out, final = fa.linear_attn_func(*leaves[:3], g, scale=scale, initial_state=s0, return_final_state=True)
    grads = torch.autograd.grad((out, final) if carried else out, leaves, (do[None], ds) if carried else do[None])
    one = (q, k, v, g, scale, s0[0] if carried else None, do, ds[0] if carried else None)
    for x, (want, amp), floor, name in zip((out[0], final[0], *(x[0] for x in grads)), R.both(*one), F.floors(*one),
                                           ("out", "final", "dq", "dk", "dv", "dinitial")):
        F.close(x, want, amp, floor, n * max(1, hq // hk), (d, d), g, dt, name)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("g", ["-0.2", "-10", "-10.5", "-11", "-11.5", "-11.7", "-11.75", "-11.78", "-11.8"])
@pytest.mark.parametrize("size", [1.0, 0.1, 0.01, 0.003])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (4, 2, 128)])
def test_fast_decays_of_small_operands(dt, g, size, hq, hk, d):
    """Around the decay where the factors of a diagonal piece are formed in another way, with rows whose largest product is small."""
    check_sizes(DT[dt], 150, hq, hk, d, decays(hk, g), (size, size, 1.0, 1.0))
    check_sizes(DT[dt], 40, hq, hk, d, decays(hk, g), (1.0, 1.0, 1.0, size * 2.0 ** -8))
    check_sizes(DT[dt], 40, hq, hk, d, decays(hk, g), (1.0, 1.0, size, 1.0))


# ------------------------------------------------------------------ what stands next to a sequence
def packed_grads(x, do, g, lens, first=0):
    leaves = [y.detach().clone().requires_grad_() for y in x]
    out = fa.linear_attn_varlen_func(*leaves, g, cum(lens, first), max(lens))
    return (out,) + torch.autograd.grad(out, leaves, do)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (2, 2, 128), (4, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0, 1.0), (1.0, 1.0, 1.0, 2.0 ** -18), (2.0 ** -9, 2.0 ** -9, 1.0, 1.0), (64.0, 64.0, 2.0 ** -8, 2.0 ** -12)])
@pytest.mark.parametrize("bad", [float("inf"), 6e4, float("nan")])
def test_neighbours_change_no_bit(dt, hq, hk, d, sizes, bad):
    """A sequence's values and gradients are the same bits whatever the rows of other sequences, and of none, hold: small gradients,
    small and large products next to infinities and to fp16's largest numbers."""
    lens, pad = [70, 61, 130], 5
    x = inputs(DT[dt], [pad] + lens + [pad], hq, hk, d, d)
    do, g = rand(7, len(x[0]), hq, d, dtype=DT[dt]), decays(hk, "-0.1")
    x, do = [(y.float() * s).to(DT[dt]) for y, s in zip(x, sizes)], (do.float() * sizes[3]).to(DT[dt])
    want = packed_grads(x, do, g, lens, pad)
    mine = slice(pad + 70, pad + 131)
    for y in x + [do]:
        keep = y[mine].clone()
        y.fill_(bad)
        y[mine] = keep
    got = packed_grads(x, do, g, lens, pad)
    for a, b, name in zip(want, got, ("out", "dq", "dk", "dv")):
        assert torch.equal(a[mine], b[mine]) and a[mine].isfinite().all(), name
        assert not b[:pad].any() and not b[-pad:].any()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (4, 4, 128), (6, 2, 128)])
def test_packed_runs_repeat(dt, hq, hk, d):
    """Bit for bit, next to rows of very different sizes that meet in a chunk."""
    lens = [60, 700, 1, 33, 129, 400] * 4
    x = inputs(DT[dt], lens, hq, hk, d, d)
    at = cum(lens).tolist()
    for z in range(1, len(lens), 2):
        for y in x[:2]:
            y[at[z]:at[z + 1]] *= 64.0
    do, g = rand(7, len(x[0]), hq, d, dtype=DT[dt]) * 2.0 ** -16, decays(hk)
    first = packed_grads(x, do, g, lens)
    for _ in range(6):
        for a, b in zip(first, packed_grads(x, do, g, lens)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ scales far from 1
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (2, 1, 128)])
@pytest.mark.parametrize("scale,sizes", [(64.0, (1500.0, 2.0 ** -6, 2.0 ** -6, 2.0 ** -12)), (2.0 ** -20, (1.0, 1.0, 1.0, 256.0)), (-0.3, (1.0, 1.0, 1.0, 1.0)),
                                         (1e-5, (8.0, 1.0, 1.0, 64.0)), (3e4, (2.0, 2.0 ** -10, 2.0 ** -10, 2.0 ** -13)), (0.0, (1.0, 1.0, 1.0, 1.0)), (2.0 ** -100, (1.0, 1.0, 1.0, 1.0))])
def test_gradients_under_any_scale(dt, hq, hk, d, scale, sizes):
    """Chunks that meet through the state, with a scale that fp16 inputs times it do not bear.  So many sequences that each is one segment."""
    L, n, b = A.lib(), 300, 320
    L.fa_linear_plan.restype = C.c_longlong
    seg, nseg = C.c_int(), C.c_int()
    L.fa_linear_plan(b, n, C.c_longlong(0), hq, hq // hk, d, d, A.DT[dt], C.byref(seg), C.byref(nseg))
    assert nseg.value == 1
    dt = DT[dt]
    one = [(x.float() * s).to(dt) for x, s in zip((*inputs(dt, [n], hq, hk, d, d), rand(5, n, hq, d, dtype=dt)), sizes)]
    size = min(1.0, abs(scale) * sizes[3] * sizes[0] * 16 + 2.0 ** -14)       # a last state's gradient next to the outputs' own
    start = 1.0 / max(1.0, 16 * abs(scale) * sizes[0])                        # a first state whose outputs stay in fp16
    s0, ds, g = rand(3, hk, d, d) * start, rand(4, hk, d, d) * size, decays(hk, "-0.02")
    q, k, v, s = (x.expand(b, *x.shape).clone().requires_grad_() for x in (*one[:3], s0))
    out, final = fa.linear_attn_func(q, k, v, g, scale=scale, initial_state=s, return_final_state=True)
    grads = torch.autograd.grad((out, final), (q, k, v, s), (one[3].expand_as(out), ds.expand_as(final)))
    args = (*one[:3], g, scale, s0, one[3], ds)
    sizes_of = R.both(*one[:3], g, abs(scale), s0, one[3], ds)     # a term's size takes the scale's size; lin_ref's sums take the scale as it is
    for x, (want, _), (_, amp), floor, name in zip((out, final, *grads), R.both(*args), sizes_of, F.floors(*args),
                                                   ("out", "final", "dq", "dk", "dv", "dinitial")):
        for z in (0, b - 1):
            F.close(x[z], want, amp, floor, n * (hq // hk), (d, d), g, dt, name)


# ------------------------------------------------------------------ indices and lengths of 64 bits
@pytest.mark.parametrize("n", [1, 40])
def test_wide_indices_and_lengths(n):
    """Slots past 32 bits are outside the pool and not their low word's; that many tokens seen are not none."""
    b, h, d = 6, 2, 64
    x = [rand(i, b, n, h, d, dtype=torch.bfloat16) for i in range(3)]
    pool, g = rand(5, 4, h, d, d), decays(h)
    before, want = pool.clone(), pool.clone()
    at = torch.tensor([1, 2 ** 32 + 3, -2 ** 40, 2 ** 62, -1, 0]).cuda()
    seen = torch.tensor([2 ** 31, 1, 1, 1, 1, 2 ** 40 + 7]).cuda()
    fa.device_error(clear=True)
    out = fa.linear_attn_with_state(*x, pool, g, state_indices=at, cache_seqlens=seen)
    assert fa.device_error(clear=True) == SLOT
    narrow = torch.tensor([1, -1, -1, -1, -1, 0], dtype=torch.int32).cuda()
    assert torch.equal(out, fa.linear_attn_with_state(*x, want, g, state_indices=narrow)) and torch.equal(pool, want)
    assert torch.equal(pool[2:], before[2:]) and not out[1:5].any() and fa.device_error() == 0
    every = torch.stack((at, at), 1)[:, 0]                      # strided, and in each integer type that torch indexes with
    fa.linear_attn_with_state(*x, pool, g, state_indices=every, cache_seqlens=seen)
    fa.linear_attn_with_state(*x, want, g, state_indices=narrow.short())
    assert torch.equal(pool, want)
    fa.device_error(clear=True)


def test_wide_indices_on_another_stream_and_captured():
    x = [rand(i, 3, 1, 2, 64, dtype=torch.bfloat16) for i in range(3)]
    pool, g, at = rand(5, 4, 2, 64, 64), decays(2), torch.tensor([2, 0, 3]).cuda()
    new = torch.zeros_like(pool)
    run = lambda: fa.linear_attn_with_state(*x, pool, g, state_indices=at, state_out=new)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    at.copy_(torch.tensor([1, 3, 2]))
    graph.replay()
    got = out.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.zeros(64 << 20, device="cuda")
        at.copy_(torch.tensor([1, 3, 2], device="cuda"))
        want = run()
    side.synchronize()
    assert torch.equal(got, want) and not big.any()


def test_wide_offsets_of_rotary():
    from fable_attn.layers.rotary import apply_rotary_emb_qk, scaled_inv_freq
    freq, _ = scaled_inv_freq(64, device="cuda")
    q, k = (rand(i, 3, 5, 2, 64, dtype=torch.bfloat16).requires_grad_() for i in range(2))
    far = torch.tensor([2 ** 32 + 5, -2 ** 35, 2 ** 31]).cuda()
    pos = far[:, None] + torch.arange(5, device="cuda")
    a, b = (apply_rotary_emb_qk(q, k, freq, **kw) for kw in (dict(seqlen_offsets=far), dict(positions=pos)))
    ga, gb = (torch.autograd.grad(y, (q, k), (torch.ones_like(q), torch.ones_like(k))) for y in (a, b))
    assert all(torch.equal(x, y) for x, y in zip((*a, *ga), (*b, *gb)))
    near = torch.tensor([5, 0, 70000]).cuda()
    a, b = (apply_rotary_emb_qk(q, k, freq, seqlen_offsets=o) for o in (near, near.int()))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = [apply_rotary_emb_qk(q[i].detach(), k[i].detach(), freq, seqlen_offsets=far[i:i + 1]) for i in range(3)]      # packed: one offset
    want = apply_rotary_emb_qk(q, k, freq, pos)
    assert all(torch.equal(o[j], want[j][i]) for i, o in enumerate(one) for j in range(2))


def test_wide_lengths_of_the_cache():
    """The paged cache reads the same kind of lengths: 2^32 cached tokens are not none, and their pages are outside the table."""
    k = rand(1, 2, 1, 2, 64, dtype=torch.bfloat16)
    kc, vc = (torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.tensor([[0], [2]], dtype=torch.int32).cuda()
    fa.device_error(clear=True)
    fa.kvcache_append(k, k, kc, vc, torch.tensor([2 ** 32, 3]).cuda(), table)
    assert fa.device_error(clear=True) == 8192
    assert torch.equal(kc[2, 3], k[1, 0]) and int(kc.count_nonzero()) == int(k[1].count_nonzero())


# ------------------------------------------------------------------ forward-mode tangents
@pytest.mark.parametrize("which", [0, 1, 2, 3, 4])
def test_forward_mode_is_refused(which):
    """A tangent is not dropped in silence: not the queries', nor any other input's, with or without gradients."""
    from torch.autograd import forward_ad
    from fable_attn.layers.rotary import apply_rotary_emb_qk, scaled_inv_freq
    x = [rand(i, 2, 20, 2, 64) for i in range(3)] + [rand(3, 2, 2, 64, 64), decays(2)]
    freq, _ = scaled_inv_freq(64, device="cuda")
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        q, k, v, s, g = x
        cu = cum([20, 20])
        calls = [lambda: fa.linear_attn_func(q, k, v, g, initial_state=s), lambda: fa.linear_attn_with_state(q, k, v, s, g),
                 lambda: fa.linear_attn_varlen_func(*(y.flatten(0, 1) for y in (q, k, v)), g, cu, 20, initial_state=s)]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        if which < 2:
            with pytest.raises(NotImplementedError):
                apply_rotary_emb_qk(q, k, freq)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                apply_rotary_emb_qk(q, k, freq, inplace=True)
        if which == 0:
            turn = forward_ad.make_dual(freq, freq)
            with pytest.raises(NotImplementedError):
                apply_rotary_emb_qk(k, k, turn)
    if which < 2:
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda y: apply_rotary_emb_qk(y, k, freq)[0], (q,), (q,))
    q, k, v = (rand(i, 2, 20, 2, 64).requires_grad_() for i in range(3))
    out, turned = fa.linear_attn_func(q, k, v, decays(2)), apply_rotary_emb_qk(q, k, freq)[0]
    with forward_ad.dual_level():                    # of a gradient that comes in
        do = forward_ad.make_dual(torch.ones_like(q), torch.ones_like(q))
        for y in (out, turned):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, q, do)
    q, k = q.detach(), k.detach()
    a, b = apply_rotary_emb_qk(k, k, freq)
    assert torch.equal(a, b) and fa.linear_attn_func(*(rand(i, 2, 20, 2, 64) for i in range(3)), decays(2)).isfinite().all()


# ------------------------------------------------------------------ which kernels run
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (8, 40), (72, 128), (128, 16)])
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 2)])
def test_tensor_cores_take_16_bits(dt, dk, dv, hq, hk, monkeypatch):
    """With FABLE_ATTN_REQUIRE_TC nothing runs on the CUDA cores instead: every direction, grouped heads, packed, states, rows off 16 bytes."""
    monkeypatch.setenv("FABLE_ATTN_REQUIRE_TC", "1")
    check_run(DT[dt], [130, 130], hq, hk, dk, dv, decays(hk), True, False)
    check_run(DT[dt], [5, 300, 0, 40], hq, hk, dk, dv, decays(hk), True, True, strided=True)
    x = [rand(i, 2, 40, h, d, dtype=DT[dt]) for i, (h, d) in enumerate(((hq, dk), (hk, dk), (hk, dv)))]
    pool = torch.zeros(2, hk, dk, dv, device="cuda")
    assert fa.linear_attn_with_state(*x, pool, decays(hk)).isfinite().all()
    odd = [torch.cat((y[..., :1], y), -1)[..., 1:] for y in x]
    assert torch.equal(fa.linear_attn_func(*odd, decays(hk)), fa.linear_attn_func(*x, decays(hk)))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_cuda_cores_are_refused_where_tensor_cores_are_required(dt, monkeypatch):
    x = [rand(i, 2, 40, 2, 136, dtype=DT[dt]).requires_grad_() for i in range(3)]
    g = decays(2)
    out = fa.linear_attn_func(*x, g)
    monkeypatch.setenv("FABLE_ATTN_REQUIRE_TC", "1")
    for call in (lambda: fa.linear_attn_func(*x, g), lambda: torch.autograd.grad(out.sum(), x)):
        with pytest.raises(Exception, match="FABLE_ATTN_REQUIRE_TC"):
            call()
    with torch.no_grad():
        assert fa.linear_attn_func(*(y[:, :16] for y in x), g).isfinite().all()       # token by token
        assert fa.linear_attn_func(*(y[:, :0] for y in x), g).numel() == 0
        assert fa.linear_attn_func(*(y.float() for y in x), g).isfinite().all()


# ------------------------------------------------------------------ states off 16 bytes
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n", [40, 400])
def test_states_that_are_slices_of_flat_buffers(dt, n):
    """A first state and a last state's gradient at any place: the same bits.  A pool is refused there, since it is written in place."""
    b, h, d = 2, 2, 64
    x = [rand(i, b, n, h, d, dtype=DT[dt]).requires_grad_() for i in range(3)]
    g, flat = decays(h), rand(3, b * h * d * d + 1)
    for at in (0, 1):
        part = flat[at:at + b * h * d * d]
        s0 = part.view(b, h, d, d).requires_grad_()
        out, final = fa.linear_attn_func(*x, g, initial_state=s0, return_final_state=True)
        both = torch.cat((rand(4, 3 if at else 4), final.flatten()))      # the gradient of the second part starts 12 bytes, or 16, into one buffer
        weight = rand(5, 4 + len(both))[:len(both)]
        got = (out, final) + torch.autograd.grad((out, both), x + [s0], (torch.ones_like(out), weight))
        near = part.detach().clone().view(b, h, d, d).requires_grad_()
        out, final = fa.linear_attn_func(*x, g, initial_state=near, return_final_state=True)
        ds = weight[-final.numel():].clone().view_as(final)
        want = (out, final) + torch.autograd.grad((out, final), x + [near], (torch.ones_like(out), ds))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    pool = flat[1:].view(b, h, d, d).detach()
    with torch.no_grad(), pytest.raises(ValueError):
        fa.linear_attn_with_state(*x, pool, g)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("g", ["0", "-0.02", "-1.5"])
@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0, 2.0 ** -18, 1.0, 2.0 ** -10), (2.0 ** -9, 2.0 ** -9, 1.0, 1.0, 2.0 ** -8, 1.0), (2.0 ** 5, 2.0 ** 5, 2.0 ** -6, 2.0 ** -14, 1.0, 2.0 ** -9),
                                   (1.0, 2.0 ** -12, 2.0 ** 6, 2.0 ** -6, 1.0, 2.0 ** -4), (2.0 ** -6, 2.0 ** 6, 2.0 ** -10, 2.0 ** 6, 2.0 ** -6, 1.0)])
@pytest.mark.parametrize("carried", [False, True])
def test_operands_of_other_sizes(dt, hq, hk, d, g, sizes, carried):
    """Small gradients, small and large queries, keys and values, over several chunks, with and without states."""
    check_sizes(DT[dt], 300, hq, hk, d, decays(hk, g), sizes, carried)


def test_written_states_may_not_want_gradients():
    x = [rand(i, 2, 3, 2, 64) for i in range(3)]
    pool, out = torch.zeros(2, 2, 64, 64, device="cuda"), torch.zeros(2, 2, 64, 64, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError):
        fa.linear_attn_with_state(*x, pool, decays(2), state_out=out)
    with torch.no_grad():
        fa.linear_attn_with_state(*x, pool, decays(2), state_out=out)
    assert out.any()
