"""Linear attention with a decay per head: training, prompts, and decode steps over a pool of states.

Per sequence and kv head, with lam = exp(log_decay):

    S_t = lam S_{t-1} + k_t v_t^T        (headdim x headdim_v, fp32)
    o_t = scale * S_t^T q_t              = scale * sum_{s <= t} lam^(t - s) (q_t . k_s) v_s   from an empty state

so that a sequence costs the same for each token however long it is, and all it needs to be continued is S.  Layouts, types and
grouped heads are those of flash_attn_func: q (batch, seqlen, nheads, headdim), k (batch, seqlen, nheads_k, headdim), v (batch, seqlen,
nheads_k, headdim_v), fp16, bf16 or fp32; the nheads / nheads_k query heads of a group read one state, states are fp32
(.., nheads_k, headdim, headdim_v).  headdim and headdim_v are multiples of 8 up to 256.

    linear_attn_func         a batch of sequences of one length, with gradients
    linear_attn_varlen_func  packed sequences, with gradients
    linear_attn_with_state   serving: new tokens (a chunk of a prompt, or one or a few) continue states that live in a pool

log_decay (nheads_k,) is the natural logarithm of the factor per token: 0 keeps everything, -infinity nothing but the token
itself, and a value above 0 counts as 0.  It carries no gradient, and forward-mode tangents are refused.  scale defaults to headdim ** -0.5.  A NaN or an infinity may
reach every output of its own sequence and heads, the tokens before it among them, and no other sequence.  All calls run on the
current stream and read lengths and indices on the device, with no host synchronisation.  The reference has no counterpart.
"""
import torch

from fable_attn import _C


def _check(q, log_decay):
    if not isinstance(log_decay, torch.Tensor):
        raise TypeError(f"fable_attn: log_decay must be a tensor of (nheads_k,), got {type(log_decay).__name__}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("fable_attn: log_decay carries no gradient; pass log_decay.detach()")
    if not q.is_cuda:
        raise ValueError("fable_attn: tensors must be on a CUDA device (q.is_cuda is False)")


class _LinearAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial, cu_seqlens, max_seqlen, want_final, keep):
        batch = q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
        final = None
        if initial is not None:
            initial = initial.contiguous()
            if initial.data_ptr() % 16:              # a slice of a flat buffer
                initial = initial.clone()
        if want_final:
            final = torch.empty(batch, k.shape[-2], k.shape[-1], v.shape[-1], dtype=torch.float32, device=q.device)
        out, states, seg_len, nseg = _C.linear_fwd(q, k, v, log_decay, scale, initial, final, None, None, cu_seqlens, max_seqlen, keep)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial, cu_seqlens, states)
        ctx.rest = (scale, max_seqlen, seg_len, nseg)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, initial, cu_seqlens, states = ctx.saved_tensors
        scale, max_seqlen, seg_len, nseg = ctx.rest
        if dout is None:
            dout = q.new_zeros(*q.shape[:-1], v.shape[-1])
        want = initial is not None and ctx.needs_input_grad[5]
        dq, dk, dv, dinitial = _C.linear_bwd(dout, q, k, v, log_decay, scale, initial, dfinal, want, cu_seqlens, max_seqlen, states,
                                             seg_len, nseg)
        return dq, dk, dv, None, None, dinitial if want else None, None, None, None, None


def _linear(q, k, v, log_decay, scale, initial, cu_seqlens, max_seqlen, want_final):
    _check(q, log_decay)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    keep = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, initial))
    out, final = _LinearAttn.apply(q, k, v, log_decay, float(scale), initial, cu_seqlens, int(max_seqlen), bool(want_final), keep)
    return (out, final) if want_final else out


def linear_attn_func(q, k, v, log_decay, scale=None, initial_state=None, return_final_state=False):
    """out (batch, seqlen, nheads, headdim_v), or (out, final_state) with return_final_state.

    initial_state (batch, nheads_k, headdim, headdim_v) fp32: S before the first token (0 without it); final_state, shaped
    alike, is S after the last.  Gradients flow to q, k, v and initial_state, from out and final_state; a group's share of dk and dv
    is summed over its query heads in fp32, in a fixed order, so that runs repeat bit for bit."""
    return _linear(q, k, v, log_decay, scale, initial_state, None, 0, return_final_state)


def linear_attn_varlen_func(q, k, v, log_decay, cu_seqlens, max_seqlen, scale=None, initial_state=None,
                            return_final_state=False):
    """linear_attn_func over packed sequences: q (total, nheads, headdim), k and v alike, sequence b in the rows [cu_seqlens[b],
    cu_seqlens[b + 1]) (int32, batch + 1).  max_seqlen is a bound on the lengths that chooses the work's split; a longer
    sequence is still computed whole, only slower.  Rows of no sequence, as padded batches have them, give 0 in out and in the gradients.
    An empty sequence's final_state is its initial_state."""
    return _linear(q, k, v, log_decay, scale, initial_state, cu_seqlens, max_seqlen, return_final_state)


def linear_attn_with_state(q, k, v, state, log_decay, scale=None, *, state_indices=None, cache_seqlens=None, cu_seqlens=None,
                           max_seqlen=None, state_out=None):
    """Continue sequences whose states live in a pool, and write the new states back; out, shaped as linear_attn_func's.

    q, k, v: (batch, seqlen, heads, dim) or, with cu_seqlens (batch + 1) int32, ragged counts packed as (total, heads, dim), where
    max_seqlen is a bound on the counts that helps to choose the kernel.  state (slots, nheads_k, headdim, headdim_v)
    fp32, contiguous and on a 16-byte boundary, is updated in place, or, with state_out of the same shape, left as it is while the new states go there (drafted tokens
    that are not accepted then cost nothing but the step back).  Sequence b has slot state_indices[b] (slot b, and
    slots == batch, without it); a negative index is padding, whose rows of out are 0.  cache_seqlens (batch): tokens seen before; where it
    is 0 the sequence starts from an empty state whatever its slot holds.

    An index outside the pool, and the later of two sequences that name one slot, give 0, leave the state alone and are
    recorded in fable_attn.device_error().  Up to 16 tokens a sequence go through the state one by one; longer ones in
    chunks.  No gradients."""
    _check(q, log_decay)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad or
                                    (state_out is not None and state_out.requires_grad)):
        raise NotImplementedError("fable_attn: linear_attn_with_state carries no gradients; use linear_attn_func")
    if scale is None:
        scale = q.shape[-1] ** -0.5
    out = state if state_out is None else state_out
    return _C.linear_fwd(q, k, v, log_decay, float(scale), state, out, state_indices, cache_seqlens, cu_seqlens,
                         0 if max_seqlen is None else int(max_seqlen), False)[0]
