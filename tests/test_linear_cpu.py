"""What linear attention and the scaled rotary decide on the host: refusals of the C entries, the split into segments, the frequencies."""
import ctypes as C
import math

import pytest
import torch

import fa_abi as A
import lin_ref as R


class FaLinearParams(C.Structure):
    _fields_ = [("struct_size", C.c_uint)] + [(n, C.c_void_p) for n in ("q", "k", "v", "o")] + [
        (n, A.FaStrides) for n in ("sQ", "sK", "sV", "sO")] + [(n, C.c_void_p) for n in ("log_decay", "state_in", "state_out")] + [
        ("slots", C.c_longlong)] + [(n, C.c_void_p) for n in ("state_index", "seen", "cu")] + [("total", C.c_longlong)] + [
        (n, C.c_int) for n in ("batch", "S", "NH", "gqa", "dk", "dv")] + [("scale", C.c_float)] + [
        (n, C.c_int) for n in ("seg_len", "nseg", "keep_states")] + [("states", C.c_void_p)]


class FaLinearBwdParams(C.Structure):
    _fields_ = [("struct_size", C.c_uint)] + [(n, C.c_void_p) for n in ("q", "k", "v", "dO", "dQ", "dK", "dV")] + [
        (n, A.FaStrides) for n in ("sQ", "sK", "sV", "sdO", "sdQ", "sdK", "sdV")] + [
        (n, C.c_void_p) for n in ("log_decay", "initial", "dfinal", "dinitial", "cu")] + [("total", C.c_longlong)] + [
        (n, C.c_int) for n in ("batch", "S", "NH", "gqa", "dk", "dv")] + [("scale", C.c_float)] + [
        (n, C.c_int) for n in ("seg_len", "nseg")] + [(n, C.c_void_p) for n in ("states", "work")]


class FaRotaryQkParams(C.Structure):
    _fields_ = [("struct_size", C.c_uint)] + [(n, C.c_void_p) for n in ("q", "k", "q_out", "k_out")] + [
        (n, A.FaStrides) for n in ("sQ", "sK", "sQo", "sKo")] + [(n, C.c_void_p) for n in ("inv_freq", "positions", "offsets")] + [
        ("offset", C.c_longlong)] + [(n, C.c_int) for n in ("pos_bytes", "batch", "seqlen", "heads_q", "heads_k", "dim", "rot_dim",
                                                           "interleaved", "inverse")] + [("factor", C.c_float)]


def lin(**kw):
    p = FaLinearParams(struct_size=C.sizeof(FaLinearParams), q=16, k=16, v=16, o=16, log_decay=16, batch=1, S=64, NH=4, gqa=2, dk=64, dv=64,
                       seg_len=128, nseg=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw", [dict(q=None), dict(log_decay=None), dict(NH=5), dict(gqa=0), dict(dk=260), dict(dv=12), dict(dk=0), dict(S=-1),
                                dict(batch=-1), dict(state_in=20, slots=1), dict(state_in=16, slots=0), dict(state_out=16, slots=0),
                                dict(cu=16, batch=0, total=3), dict(S=500), dict(seg_len=0), dict(S=200, nseg=2), dict(total=-1)])
def test_forward_refusals(kw):
    L = A.lib()
    assert L.fa_linear_launch(C.byref(lin(**kw)), 1, None) == A.FA_ERR_INVALID
    assert L.fa_last_error()


def test_forward_refuses_types_and_layouts():
    L = A.lib()
    assert L.fa_linear_launch(C.byref(lin()), 3, None) == A.FA_ERR_INVALID
    assert L.fa_linear_launch(C.byref(lin(struct_size=8)), 1, None) == A.FA_ERR_ABI
    assert L.fa_linear_launch(None, 1, None) == A.FA_ERR_INVALID
    assert L.fa_linear_launch(C.byref(lin(batch=0)), 1, None) == A.FA_OK


@pytest.mark.parametrize("kw", [dict(dO=None), dict(dK=None), dict(NH=5), dict(dk=12), dict(dfinal=8), dict(S=500), dict(S=200, nseg=2),
                                dict(S=200, nseg=2, states=16), dict(struct_size=16)])
def test_backward_refusals(kw):
    L = A.lib()
    p = FaLinearBwdParams(struct_size=C.sizeof(FaLinearBwdParams), q=16, k=16, v=16, dO=16, dQ=16, dK=16, dV=16, log_decay=16, batch=1, S=64,
                          NH=4, gqa=2, dk=64, dv=64, seg_len=128, nseg=1)
    for k, v in kw.items():
        setattr(p, k, v)
    assert L.fa_linear_backward_launch(C.byref(p), 1, None) in (A.FA_ERR_INVALID, A.FA_ERR_ABI)


@pytest.mark.parametrize("kw", [dict(q=None), dict(inv_freq=None), dict(k=16), dict(rot_dim=7), dict(rot_dim=66), dict(rot_dim=0), dict(heads_q=0),
                                dict(positions=16, pos_bytes=2), dict(batch=-1), dict(dim=600, rot_dim=300), dict(struct_size=4)])
def test_rotary_refusals(kw):
    L = A.lib()
    p = FaRotaryQkParams(struct_size=C.sizeof(FaRotaryQkParams), q=16, q_out=16, inv_freq=16, batch=1, seqlen=1, heads_q=1, dim=64, rot_dim=64)
    for k, v in kw.items():
        setattr(p, k, v)
    assert L.fa_rotary_qk_launch(C.byref(p), 1, None) in (A.FA_ERR_INVALID, A.FA_ERR_ABI)


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    mirrors = {"FaLinearParams": FaLinearParams, "FaLinearBwdParams": FaLinearBwdParams, "FaRotaryQkParams": FaRotaryQkParams}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fable_attn.h"', "int main(void){"]
    for name, cls in mirrors.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.dirname(A.HEADER), str(src), "-o", str(tmp_path / "probe")], check=True)
    for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines():
        s, f, v = line.split()
        assert int(v) == (C.sizeof(mirrors[s]) if f == "size" else getattr(mirrors[s], f).offset), (s, f)


@pytest.mark.parametrize("batch,s,total", [(1, 1, 0), (1, 16384, 0), (256, 4096, 0), (1, 1 << 30, 0), (7, 300, 1000), (1000, 5, 17), (1, 0, 0), (0, 5, 0)])
@pytest.mark.parametrize("nh,gqa,dk,dv,dt", [(32, 1, 128, 128, 1), (64, 8, 64, 64, 0), (2, 1, 256, 80, 2)])
def test_plan_covers_every_token(batch, s, total, nh, gqa, dk, dv, dt):
    L = A.lib()
    L.fa_linear_plan.restype = C.c_longlong
    seg, n = C.c_int(), C.c_int()
    floats = L.fa_linear_plan(batch, s, C.c_longlong(total), nh, gqa, dk, dv, dt, C.byref(seg), C.byref(n))
    assert seg.value > 0 and n.value >= 1 and seg.value * n.value >= s and (n.value - 1) * seg.value < max(s, 1)
    slots = batch if n.value == 1 else batch * n.value if not total else -(-total // seg.value) if batch == 1 else total // seg.value + batch
    whole = slots * (nh // gqa) * dk * dv
    assert floats == whole if n.value > 1 else floats in (0, whole)     # one segment: a last state may need it


def test_segments_of_packed_sequences_have_slots_of_their_own():
    """The first slot of sequence z is floor(row0 / seg_len) + z: ranges of ceil(len / seg_len) slots that do not meet and end in
    total / seg_len + batch, and a bisection over them finds each slot's sequence."""
    gen = torch.Generator().manual_seed(3)
    for _ in range(300):
        batch, seg = int(torch.randint(1, 9, (), generator=gen)), int(torch.randint(1, 40, (), generator=gen))
        lens = (torch.randint(0, 90, (batch,), generator=gen) * (torch.rand(batch, generator=gen) > 0.3)).tolist()
        row0 = [sum(lens[:z]) for z in range(batch)]
        first = [r // seg + z for z, r in enumerate(row0)]
        spans = [range(f, f + -(-n // seg)) for f, n in zip(first, lens)]
        used = [s for r in spans for s in r]
        assert len(set(used)) == len(used) and max(used, default=0) < sum(lens) // seg + batch
        assert len(set(first)) == batch                                   # an empty sequence's slot is nobody else's
        assert all(f not in r for z, f in enumerate(first) for y, r in enumerate(spans) if y != z)
        for z, r in enumerate(spans):
            for s in r:
                lo, hi = 0, batch
                while hi - lo > 1:
                    mid = (lo + hi) // 2
                    lo, hi = (mid, hi) if first[mid] <= s else (lo, mid)
                assert lo == z


def test_reference_gradients_against_differences():
    """lin_ref's gradients against its own values: both are linear in each input, so a step of 1 is exact."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x = [r(9, 4, 5), r(9, 2, 5), r(9, 2, 3), r(2, 5, 3)]
    g, do, ds = torch.tensor([-0.3, -math.inf], dtype=torch.float64), r(9, 4, 3), r(2, 5, 3)
    loss = lambda y: sum((p * w).sum() for p, w in zip(R.one(*y[:3], g, 0.7, y[3]), (do, ds)))
    grads = R.one(*x[:3], g, 0.7, x[3], do, ds)[2:]
    for i in range(4):
        step = r(*x[i].shape)
        up, down = ([y + s * step if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        assert abs((loss(up) - loss(down)) / 2 - (grads[i] * step).sum()) < 1e-10


def test_reference_against_the_recurrence():
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(20, h, 4, generator=gen, dtype=torch.float64) for h in (4, 2, 2))
    g, s = torch.tensor([-0.2, 0.0], dtype=torch.float64), torch.randn(2, 4, 4, generator=gen, dtype=torch.float64)
    o, final = R.one(q, k, v, g, 0.5, s)
    for t in range(20):
        s = g.exp()[:, None, None] * s + k[t][:, :, None] * v[t][:, None]
        for h in range(4):
            assert torch.allclose(o[t, h], 0.5 * s[h // 2].t() @ q[t, h], atol=1e-12)
    assert torch.allclose(final, s, atol=1e-12)


def test_scaled_frequencies():
    from fable_attn.layers.rotary import rotary_tables, scaled_inv_freq
    f, m = scaled_inv_freq(64)
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32))
    lin_, _ = scaled_inv_freq(64, scaling="linear", factor=4.0)
    assert torch.allclose(lin_, f / 4)
    ntk, _ = scaled_inv_freq(64, scaling="ntk", factor=4.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4)
    y, m = scaled_inv_freq(64, scaling="yarn", factor=4.0, original_max_position=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 45], f[turns > 45]) and torch.allclose(y[turns < 0.7], f[turns < 0.7] / 4)
    assert bool((y <= f).all()) and bool((y >= f / 4 * (1 - 1e-12)).all()) and bool((y[1:] < y[:-1]).all()) and math.isclose(m, 1 + 0.1 * math.log(4))
    cos, sin = rotary_tables(y, 50, m)
    assert cos.shape == sin.shape == (50, 32) and cos.dtype == torch.float32 and torch.allclose(cos ** 2 + sin ** 2, torch.tensor(m * m).float())


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(scaling="other"), dict(scaling="yarn"), dict(factor=0.5),
                                dict(base=1.0), dict(scaling="ntk", rotary_dim=2), dict(scaling="yarn", original_max_position=10, beta_fast=1.0)])
def test_scaled_frequencies_refuse(kw):
    from fable_attn.layers.rotary import scaled_inv_freq
    with pytest.raises(ValueError):
        scaled_inv_freq(**{"rotary_dim": 64, "factor": 2.0, **kw})


def test_host_tensors_are_refused():
    import fable_attn as fa
    from fable_attn.layers.rotary import apply_rotary_emb_qk
    x, g = torch.zeros(1, 4, 2, 64), torch.zeros(2)
    with pytest.raises(ValueError):
        fa.linear_attn_func(x, x, x, g)
    with pytest.raises(ValueError):
        fa.linear_attn_varlen_func(x[0], x[0], x[0], g, torch.tensor([0, 4]), 4)
    with pytest.raises(ValueError):
        fa.linear_attn_with_state(x, x, x, torch.zeros(1, 2, 64, 64), g)
    with pytest.raises(TypeError):
        fa.linear_attn_func(x, x, x, -0.1)
    with pytest.raises(ValueError):
        apply_rotary_emb_qk(x, x, torch.ones(32))
