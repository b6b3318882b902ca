"""Rotary embedding of one token a sequence whose sequence dimension comes first in memory: such a dimension has one entry and a
stride that says nothing.  Rotation alone gives the same bits as of the packed copy."""
import pytest
import torch

import fable_attn as fa
from fable_attn.layers.rotary import apply_rotary_emb

pytestmark = pytest.mark.gpu


def seq_first(x):
    """(batch, 1, heads, dim) as a view of (1, batch, heads, dim); the storage goes on to where its stride would lead."""
    b, _, h, d = x.shape
    wide = torch.zeros(b * b, h, d, dtype=x.dtype, device=x.device)
    wide[:b] = x[:, 0]
    return wide[:b][None].transpose(0, 1)


def tables(rows, half):
    ang = torch.arange(rows, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
    return ang.cos(), ang.sin()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_apply_rotary_emb(interleaved, inplace):
    x = torch.randn(4, 1, 3, 64, device="cuda", dtype=torch.bfloat16)
    cos, sin = tables(50, 32)
    offs = torch.tensor([7, 0, 33, 49], dtype=torch.int32, device="cuda")
    want = apply_rotary_emb(x.clone(), cos, sin, interleaved, seqlen_offsets=offs)
    y = seq_first(x)
    got = apply_rotary_emb(y, cos, sin, interleaved, inplace=inplace, seqlen_offsets=offs)
    assert got.shape == x.shape and torch.equal(got, want)
    assert torch.equal(y, want if inplace else x)


@pytest.mark.parametrize("sq", [1, 3])
def test_attention_that_rotates(sq):
    """k of one token a sequence, rotated on the way into the forward."""
    q = torch.randn(4, sq, 4, 64, device="cuda", dtype=torch.float16)
    k, v = (torch.randn(4, 1, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    cos, sin = tables(8, 32)
    with torch.no_grad():
        want = fa.flash_attn_func(q, k, v, rotary_cos=cos, rotary_sin=sin)
        got = fa.flash_attn_func(q, seq_first(k), v, rotary_cos=cos, rotary_sin=sin)
    assert torch.equal(got, want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_attention_that_rotates_a_slice_of_longer_sequences(interleaved):
    """k cut out of a longer buffer: its batches do not follow one another."""
    q = torch.randn(3, 5, 4, 64, device="cuda", dtype=torch.float16)
    wide = torch.randn(2, 3, 9, 2, 64, device="cuda", dtype=torch.float16)
    k, v = wide[0, :, 2:7], wide[1, :, 2:7]
    cos, sin = tables(8, 32)
    with torch.no_grad():
        want = fa.flash_attn_func(q, k.clone(), v.clone(), causal=True, rotary_cos=cos, rotary_sin=sin, rotary_interleaved=interleaved)
        got = fa.flash_attn_func(q, k, v, causal=True, rotary_cos=cos, rotary_sin=sin, rotary_interleaved=interleaved)
    assert torch.equal(got, want)


def test_attention_that_rotates_one_head_given_as_several():
    q = torch.randn(3, 5, 4, 64, device="cuda", dtype=torch.float16)
    k, v = (torch.randn(3, 5, 1, 64, device="cuda", dtype=torch.float16).expand(-1, -1, 2, -1) for _ in range(2))
    cos, sin = tables(8, 32)
    with torch.no_grad():
        want = fa.flash_attn_func(q, k.contiguous(), v.contiguous(), causal=True, rotary_cos=cos, rotary_sin=sin)
        got = fa.flash_attn_func(q, k, v, causal=True, rotary_cos=cos, rotary_sin=sin)
    assert torch.equal(got, want)
