"""One layer of linear attention with a decay per head: a training step, and the same sequences served.

Queries and keys are turned by their positions (apply_rotary_emb_qk, frequencies scaled for long contexts), then
  training  linear_attn_varlen_func over packed sequences, with gradients through both;
  serving   linear_attn_with_state: the prompts in chunks, then tokens one by one, over a pool of states; drafted tokens go to a
            second pool first, and count only once they are accepted.
Served outputs and last states are compared with the training pass over whole sequences, and the relative distance is printed: what
rounding to bf16 costs, about 0.2 %.

    python flash-attention-rdna2_b200/examples/linear_layer.py [--chunk N]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fable_attn as fa  # noqa: E402
from fable_attn.layers.rotary import apply_rotary_emb_qk, scaled_inv_freq  # noqa: E402


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--chunk", type=int, default=256)
    a = ap.parse_args(argv)
    dev = torch.device("cuda")
    torch.manual_seed(0)
    hq, hk, d, lens, tail = 16, 4, 128, [700, 33, 1025, 256], 5       # the last `tail` tokens are decoded
    batch, total = len(lens), sum(lens)
    cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
    starts = cu[:-1].tolist()
    pos = torch.cat([torch.arange(n, device=dev) for n in lens]).to(torch.int32)
    inv, factor = scaled_inv_freq(d, scaling="yarn", factor=8.0, original_max_position=4096, device=dev)
    log_decay = -torch.logspace(-0.5, -3, hk, device=dev)
    q, k, v = (torch.randn(total, h, d, device=dev, dtype=torch.bfloat16, requires_grad=True) for h in (hq, hk, hk))
    turn = lambda q, k, pos: apply_rotary_emb_qk(q, k, inv, pos, factor=factor)

    whole, last = fa.linear_attn_varlen_func(*turn(q, k, pos), v, log_decay, cu, max(lens), return_final_state=True)
    whole.backward(torch.randn_like(whole))
    assert all(x.grad.isfinite().all() for x in (q, k, v))
    print(f"training step over {lens} tokens: gradients of q, k and v")

    pool = torch.empty(batch + 2, hk, d, d, device=dev)               # whatever the slots held
    drafts = torch.empty_like(pool)
    slots = torch.randperm(batch + 2, device=dev)[:batch].to(torch.int32)
    out, done = torch.empty_like(whole), [0] * batch

    def serve(counts, states_to=None):                                # the next counts[z] tokens of each sequence
        rows = torch.cat([torch.arange(s + n, s + n + c, device=dev) for s, n, c in zip(starts, done, counts)])
        with torch.no_grad():
            got = fa.linear_attn_with_state(*turn(q[rows], k[rows], pos[rows]), v[rows], pool, log_decay, state_indices=slots,
                                            cache_seqlens=torch.tensor(done, dtype=torch.int32, device=dev),
                                            cu_seqlens=torch.tensor([0] + counts, device=dev).cumsum(0).to(torch.int32),
                                            max_seqlen=max(counts), state_out=states_to)
        return rows, got

    while any(n < m - tail for n, m in zip(done, lens)):
        counts = [max(0, min(a.chunk, m - tail - n)) for n, m in zip(done, lens)]
        rows, got = serve(counts)
        out[rows] = got
        done = [n + c for n, c in zip(done, counts)]
    serve([3] * batch, drafts)                                        # drafted, and not accepted: the pool is as it was
    for _ in range(tail):
        rows, got = serve([1] * batch)
        out[rows] = got
        done = [n + 1 for n in done]
    worst = max(rel(out, whole), rel(pool[slots.long()], last))
    print(f"served in chunks of {a.chunk} and {tail} tokens one by one: {worst:.4f} from the whole sequences")
    return worst


if __name__ == "__main__":
    main()
