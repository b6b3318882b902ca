"""Paged K/V caches held in 8 bits: writing, attending, reading back.

A cache is k_cache / v_cache (num_blocks, page_block_size, nheads_k, headdim), page_block_size a power of two,
with block_table (batch, max_blocks) int32, as flash_attn_with_kvcache takes it.  Held in 8 bits it is
torch.int8 or torch.float8_e4m3fn and comes with k_scale / v_scale (num_blocks, nheads_k,
page_block_size // block) fp32: one scale for `block` consecutive slots of a page and a head, block a power of two up to 256.  An
element's value is code * scale.  `new_cache_8bit` makes one.

    kvcache_append                rotates new keys and writes keys and values behind the cached ones
    flash_attn_with_kvcache_8bit  attention of one or several new tokens over the cache
    kvcache_gather                a range of the cache as packed keys and values, for the prefill of a
                                  further chunk with flash_attn_varlen_func

The reference has no counterpart: its caches hold the inputs' type and its FP8 arguments raise.
headdim is a multiple of 16 up to 256.  All calls run on the current stream and read lengths and
tables on the device, with no host synchronisation.  None of them carries gradients.
"""
import torch

from fable_attn import _C

_CODE_TYPES = (torch.int8, torch.float8_e4m3fn)


def new_cache_8bit(num_blocks, page_block_size, nheads_k, headdim, dtype=torch.int8, block=16, device="cuda"):
    """Empty (k_cache, v_cache, k_scale, v_scale) with one scale for `block` slots of a page and a head."""
    if dtype not in _CODE_TYPES:
        raise ValueError(f"fable_attn: an 8-bit cache is torch.int8 or torch.float8_e4m3fn, not {dtype}")
    if block < 1 or block & (block - 1) or block > 256 or page_block_size % block:
        raise ValueError(f"fable_attn: block={block} must be a power of two up to 256 that divides "
                         f"page_block_size={page_block_size}")
    shape = (num_blocks, page_block_size, nheads_k, headdim)
    k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(num_blocks, nheads_k, page_block_size // block, device=device) for _ in range(2))
    return k, v, ks, vs


def kvcache_append(k, v, k_cache, v_cache, cache_seqlens, block_table, *, k_scale=None, v_scale=None,
                   cu_seqlens_new=None, rotary_cos=None, rotary_sin=None, rotary_interleaved=True,
                   rotary_seqlens=None):
    """Write new keys and values behind each sequence's cached tokens, in place.

    k, v: (batch, seqlen_new, nheads_k, headdim) or, with cu_seqlens_new (batch + 1) int32, ragged counts packed
    as (total_new, nheads_k, headdim); fp16, bf16 or fp32.  cache_seqlens (batch): tokens in the cache BEFORE
    the call; token i goes to position cache_seqlens + i (the caller advances cache_seqlens).
    rotary_cos / rotary_sin (seqlen_ro, rotary_dim / 2) rotate k at its position, or at rotary_seqlens + i, in fp32
    with one rounding at the end.  A sequence with no new tokens is left alone, and so is what cu_seqlens_new names beyond
    the rows given.

    Fast are rows on 16-byte boundaries, a rotary_dim that is a multiple of 16 and, in 8 bits, pages of 16 slots or more; other
    calls go element by element and take 5 to 7 times as long.

    The cache has k's type, or is 8-bit with k_scale / v_scale.  Then each touched block of slots gets
    s = max(its scale so far, amax / Q, 2**-100), Q = 127 or 448, its scale so far counting only where the block holds
    earlier tokens of the sequence; new codes are round(x / s), and earlier codes are put on the new scale where it
    grew.  A NaN or an infinity makes its block's scale NaN until the block is begun anew, so that reading
    the block gives NaN.  Two sequences must not append to one page."""
    _C.kv_append(k, v, k_cache, v_cache, cache_seqlens, block_table, k_scale, v_scale, cu_seqlens_new, rotary_cos,
                 rotary_sin, bool(rotary_interleaved), rotary_seqlens)


def kvcache_gather(k_cache, v_cache, block_table, cu_seqlens_k, total_k, *, k_scale=None, v_scale=None,
                   seq_starts=None, dtype=None):
    """(k, v), each (total_k, nheads_k, headdim): of sequence b the positions seq_starts[b] + i (0 + i without
    seq_starts), i < cu_seqlens_k[b + 1] - cu_seqlens_k[b], as rows from cu_seqlens_k[b] on.  dtype: fp16,
    bf16 or fp32 (default: the cache's, bf16 for an 8-bit one); one rounding.  With cu_seqlens_k they are the k and
    v of flash_attn_varlen_func.  total_k (host int) must be cu_seqlens_k[-1]."""
    return tuple(_C.kv_gather(k_cache, v_cache, block_table, cu_seqlens_k, int(total_k), k_scale, v_scale, seq_starts,
                              dtype))


def flash_attn_with_kvcache_8bit(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale=None,
                                 causal=True, window_size=(-1, -1), softcap=0.0, alibi_slopes=None, *,
                                 cu_seqlens_q=None, max_seqlen_q=None, cache_leftpad=None, rotary_cos=None,
                                 rotary_sin=None, rotary_interleaved=True, rotary_seqlens=None,
                                 return_softmax_lse=False):
    """Attention of new tokens over an 8-bit paged cache that holds them already (kvcache_append first).

    q: (batch, seqlen_q, nheads, headdim) or, with cu_seqlens_q (batch + 1) int32, ragged counts packed as
    (total_q, nheads, headdim); fp16, bf16 or fp32.  cache_seqlens (batch): tokens in the cache, the new ones
    INCLUDED: query t of a sequence's n sits at position cache_seqlens - n + t, and masks are aligned to it as
    in flash_attn_func (causal, window_size, keys before cache_leftpad hidden).  rotary_cos / rotary_sin rotate q by
    its position, or by rotary_seqlens + t.  max_seqlen_q is a bound on the ragged counts that helps to choose the kernel.

    Returns out, shaped as q, or (out, softmax_lse) with return_softmax_lse: (batch, nheads, seqlen_q), or (nheads,
    total_q) with cu_seqlens_q.  Rows that see nothing, and packed rows outside [cu_seqlens_q[0], cu_seqlens_q[-1]) as
    padded batches have them, are 0 with an LSE of -infinity.  Meant for up to some tens of query rows (tokens times query heads of a kv
    head) per sequence; longer chunks: kvcache_gather and flash_attn_varlen_func.  V's values may be up to 2**100.  Pages of
    less than 16 slots take about 1.7 times as long."""
    if k_cache.dtype not in _CODE_TYPES:
        raise ValueError(f"fable_attn: an 8-bit cache is torch.int8 or torch.float8_e4m3fn, not {k_cache.dtype}")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    wl, wr = window_size
    wl = -1 if wl is None or wl < 0 else int(wl)
    wr = 0 if causal else -1 if wr is None or wr < 0 else int(wr)
    n = q.shape[0] if max_seqlen_q is None else int(max_seqlen_q)
    out = _C.dec8(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, float(softmax_scale), wl, wr,
                  float(softcap or 0.0), alibi_slopes, cu_seqlens_q, n, cache_leftpad, rotary_cos, rotary_sin,
                  bool(rotary_interleaved), rotary_seqlens, bool(return_softmax_lse))
    return tuple(out) if return_softmax_lse else out[0]
