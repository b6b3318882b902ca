"""CPU tests of the paged 8-bit cache operators: the parameter blocks' layout, and every refusal that is
decided before any device work (C ABI and Python)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import fa_abi as A
import fable_attn as fa

P, I, L, F = C.c_void_p, C.c_int, C.c_longlong, C.c_float


class FaKvAppendParams(C.Structure):
    _fields_ = [("struct_size", C.c_uint), ("k", P), ("v", P), ("k_row", L), ("k_head", L), ("v_row", L), ("v_head", L),
                ("Kc", P), ("Vc", P), ("Ks", P), ("Vs", P), ("block_table", P), ("ctx_len", P), ("cu_new", P),
                ("tokens", I), ("total", L)] + [(n, I) for n in ("batch", "heads", "dim", "page", "block", "max_blocks", "code")] + [
                ("num_blocks", L), ("cos", P), ("sin", P), ("rot_dim", I), ("rot_seqlen_ro", I), ("rot_interleaved", I),
                ("rot_pos", P)]


class FaKvGatherParams(C.Structure):
    _fields_ = [("struct_size", C.c_uint), ("Kc", P), ("Vc", P), ("Ks", P), ("Vs", P), ("block_table", P), ("cu_k", P),
                ("starts", P), ("k", P), ("v", P), ("total", L)] + [
                (n, I) for n in ("batch", "heads", "dim", "page", "block", "max_blocks", "code")] + [("num_blocks", L)]


class FaDec8Params(C.Structure):
    _fields_ = [("struct_size", C.c_uint), ("q", P), ("q_row", L), ("q_head", L), ("Kc", P), ("Vc", P), ("Ks", P), ("Vs", P),
                ("block_table", P), ("ctx_len", P), ("cu_q", P), ("tokens", I), ("max_tokens", I), ("total", L), ("o", P),
                ("lse", P), ("scratch", P)] + [
                (n, I) for n in ("batch", "NH", "gqa", "dim", "page", "block", "max_blocks", "code")] + [
                ("num_blocks", L), ("scale", F), ("softcap", F), ("win_left", I), ("win_right", I), ("alibi", P),
                ("leftpad", P), ("cos", P), ("sin", P), ("rot_dim", I), ("rot_seqlen_ro", I), ("rot_interleaved", I),
                ("rot_pos", P)]


BLOCKS = (FaKvAppendParams, FaKvGatherParams, FaDec8Params)


def test_mirrors_match_the_header():
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fable_attn.h"', "int main(void){"]
    for cls in BLOCKS:
        n = cls.__name__
        lines.append(f'printf("{n} size %zu\\n", sizeof({n}));')
        lines += [f'printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for f, _ in cls._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(src, "w").write("\n".join(lines + ["return 0;}"]))
        subprocess.run(["gcc", "-I", os.path.dirname(A.HEADER), src, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out if x}
    for cls in BLOCKS:
        assert got[(cls.__name__, "size")] == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert got[(cls.__name__, f)] == getattr(cls, f).offset, (cls.__name__, f)


def block(cls, **kw):
    p = cls()
    p.struct_size = C.sizeof(cls)
    for f, t in cls._fields_:   # placeholders: refused before any pointer is followed
        if t is P and f not in ("cu_new", "cu_q", "starts", "cos", "sin", "rot_pos", "alibi", "leftpad", "lse"):
            setattr(p, f, 16)
    base = dict(batch=2, heads=2, dim=64, page=16, block=8, max_blocks=4, code=8, num_blocks=10, tokens=1, total=2, NH=4, gqa=2,
                scale=1.0, win_left=-1, win_right=0)
    for k, v in {**base, **kw}.items():
        if hasattr(p, k):
            setattr(p, k, v)
    return p


COMMON = [(dict(page=24), A.FA_ERR_INVALID), (dict(block=32), A.FA_ERR_INVALID), (dict(block=3), A.FA_ERR_INVALID),
          (dict(block=0), A.FA_ERR_INVALID), (dict(page=1024, block=512), A.FA_ERR_INVALID), (dict(max_blocks=0), A.FA_ERR_INVALID),
          (dict(num_blocks=0), A.FA_ERR_INVALID), (dict(code=5), A.FA_ERR_INVALID), (dict(Ks=None), A.FA_ERR_INVALID),
          (dict(dim=72), A.FA_ERR_UNSUPPORTED), (dict(dim=272), A.FA_ERR_UNSUPPORTED), (dict(Kc=None), A.FA_ERR_INVALID),
          (dict(total=-1), A.FA_ERR_INVALID), (dict(total=1 << 40, tokens=1 << 20, cu_new=16, cu_q=16), A.FA_ERR_SIZE),
          (dict(struct_size=8), A.FA_ERR_ABI)]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(total=3), A.FA_ERR_INVALID), (dict(code=0, Ks=None, Vs=None), A.FA_ERR_INVALID), (dict(code=1), A.FA_ERR_INVALID),
    (dict(cos=16), A.FA_ERR_INVALID), (dict(cos=16, sin=16, rot_dim=3, rot_seqlen_ro=4), A.FA_ERR_INVALID),
    (dict(cos=16, sin=16, rot_dim=80, rot_seqlen_ro=4), A.FA_ERR_INVALID), (dict(ctx_len=None), A.FA_ERR_INVALID)])
def test_append_refusals(kw, code):
    assert A.lib().fa_kv_append_launch(C.byref(block(FaKvAppendParams, **kw)), 1, None) == code


@pytest.mark.parametrize("kw,code", COMMON + [(dict(cu_k=None), A.FA_ERR_INVALID)])
def test_gather_refusals(kw, code):
    assert A.lib().fa_kv_gather_launch(C.byref(block(FaKvGatherParams, **kw)), 1, None) == code


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(total=3), A.FA_ERR_INVALID), (dict(NH=5), A.FA_ERR_INVALID), (dict(gqa=0), A.FA_ERR_INVALID), (dict(code=1), A.FA_ERR_INVALID),
    (dict(cos=16, sin=16, rot_dim=3, rot_seqlen_ro=4), A.FA_ERR_INVALID), (dict(o=None), A.FA_ERR_INVALID)])
def test_decode8_refusals(kw, code):
    assert A.lib().fa_decode8_launch(C.byref(block(FaDec8Params, **kw)), 1, None) == code


@pytest.mark.parametrize("fn,cls", [("fa_kv_append_launch", FaKvAppendParams), ("fa_kv_gather_launch", FaKvGatherParams),
                                    ("fa_decode8_launch", FaDec8Params)])
def test_dtype_codes_null_blocks_and_nothing_to_do(fn, cls):
    f = getattr(A.lib(), fn)
    assert f(C.byref(block(cls)), 8, None) == A.FA_ERR_INVALID
    assert f(None, 1, None) == A.FA_ERR_INVALID
    assert f(C.byref(block(cls, total=0, tokens=0)), 1, None) == A.FA_OK
    assert f(C.byref(block(cls, batch=0, total=0)), 1, None) == A.FA_OK


def test_python_refuses_cpu_tensors_and_wrong_types():
    k, v, ks, vs = fa.new_cache_8bit(4, 16, 2, 64, device="cpu")
    assert k.dtype == torch.int8 and ks.shape == (4, 2, 1)
    bt, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        fa.kvcache_append(x, x, k, v, n, bt, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="CUDA"):
        fa.kvcache_gather(k, v, bt, torch.zeros(2, dtype=torch.int32), 0, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="CUDA"):
        fa.flash_attn_with_kvcache_8bit(x, k, v, ks, vs, n, bt)
    with pytest.raises(ValueError, match="8-bit"):
        fa.flash_attn_with_kvcache_8bit(x, k.float(), v.float(), ks, vs, n, bt)


@pytest.mark.parametrize("kw", [dict(dtype=torch.float16), dict(block=3), dict(block=32), dict(block=0), dict(block=512)])
def test_new_cache_refusals(kw):
    with pytest.raises(ValueError):
        fa.new_cache_8bit(4, 16, 2, 64, device="cpu", **kw)


def test_new_cache_types():
    k, v, ks, vs = fa.new_cache_8bit(3, 64, 1, 32, dtype=torch.float8_e4m3fn, block=4, device="cpu")
    assert k.dtype == v.dtype == torch.float8_e4m3fn and k.shape == (3, 64, 1, 32) and vs.shape == (3, 1, 16)
    assert (k.float() == 0).all() and (ks == 0).all()
