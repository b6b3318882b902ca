"""Calls from threads that have used no GPU before: the same kernels run, and give the same bits.

A tensor map needs a current context, which such a thread gets with its first runtime call; autograd runs backward passes on a thread of
its own."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import fable_attn as fa

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def prompt():
    x = [rand(i, 2, 300, 4, 64) for i in range(3)]
    g, pool, new = torch.full((4,), -0.02).cuda(), torch.zeros(2, 4, 64, 64, device="cuda"), torch.empty(2, 4, 64, 64, device="cuda")
    return lambda: (fa.linear_attn_with_state(*x, pool, g, state_out=new), new)


def forward(d):
    x = [rand(i, 2, 300, 4, d) for i in range(3)]
    return lambda: (fa.flash_attn_func(*x, causal=True),)


def packed():
    x = [rand(i, 600, 4, 128) for i in range(3)]
    cu = torch.tensor([0, 200, 600], dtype=torch.int32).cuda()
    return lambda: (fa.flash_attn_varlen_func(*x, cu, cu, 400, 400, causal=True),)


def paged(nq):
    q, kc, vc = rand(1, 2, nq, 32, 128), rand(2, 40, 256, 8, 128), rand(3, 40, 256, 8, 128)
    table, lens = torch.arange(40, dtype=torch.int32).view(2, 20).cuda(), torch.tensor([5000, 777], dtype=torch.int32).cuda()
    return lambda: (fa.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=lens, block_table=table, causal=True),)


def paged8(kind):
    k8, v8, ks, vs = fa.new_cache_8bit(40, 64, 2, 128, kind, device="cuda")
    table, lens = torch.arange(40, dtype=torch.int32).view(2, 20).cuda(), torch.tensor([1000, 777], dtype=torch.int32).cuda()
    x = rand(4, 1777, 2, 128)
    cu = torch.tensor([0, 1000, 1777], dtype=torch.int32).cuda()
    fa.kvcache_append(x, x, k8, v8, torch.zeros_like(lens), table, k_scale=ks, v_scale=vs, cu_seqlens_new=cu)
    q = rand(5, 2, 1, 16, 128)
    return lambda: (fa.flash_attn_with_kvcache_8bit(q, k8, v8, ks, vs, lens, table),)


CALLS = {"prompt": prompt, "forward64": lambda: forward(64), "forward128": lambda: forward(128), "forward256": lambda: forward(256), "packed": packed,
         "paged1": lambda: paged(1), "paged64": lambda: paged(64), "int8": lambda: paged8(torch.int8), "e4m3": lambda: paged8(torch.float8_e4m3fn)}


@pytest.mark.parametrize("name", list(CALLS))
def test_first_call_of_a_thread(name):
    call = CALLS[name]()
    want = [x.clone() for x in call()]
    call()                                       # the allocator has the memory: the thread's first call to the GPU is the operator's
    got = []

    def run():
        try:
            got.extend(x.clone() for x in call())
        except Exception as e:                   # shown by the assertion below
            got.append(e)

    torch.cuda.synchronize()
    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), got


BACKWARD = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import fable_attn as fa
torch.manual_seed(0)
x = [torch.randn(2, 300, 4, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3)]
do, g = torch.randn_like(x[0]), torch.full((4,), -0.02, device="cuda")
s0 = torch.randn(2, 4, 64, 64, device="cuda", requires_grad=True)
held = [torch.empty(4 << 20, device="cuda", dtype=t) for t in (torch.uint8, torch.float32) for _ in range(8)]
del held                                         # the allocator has the memory
if sys.argv[2] == "linear":
    out = fa.linear_attn_func(*x, g, initial_state=s0)
    leaves = x + [s0]
else:
    out = fa.flash_attn_func(*x, causal=True)
    leaves = x
a, b = (torch.autograd.grad(out, leaves, do, retain_graph=True) for _ in range(2))
print([bool(torch.equal(i, j)) for i, j in zip(a, b)])
"""


@pytest.mark.parametrize("kind", ["linear", "attention"])
def test_first_backward_of_a_process(kind):
    root = os.path.dirname(os.path.dirname(os.path.abspath(fa.__file__)))
    r = subprocess.run([sys.executable, "-c", BACKWARD, root, kind], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "True" in r.stdout and "False" not in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("name", ["prompt", "forward128", "packed"])
def test_two_threads_at_once(name):
    """Each on a stream of its own, many times over: nothing is shared that the calls write."""
    calls = [CALLS[name]() for _ in range(2)]
    want = [[x.clone() for x in c()] for c in calls]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not all(torch.equal(a, b) for a, b in zip(calls[i](), want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


CAPTURED = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import fable_attn as fa
from fable_attn.layers.rotary import apply_rotary_emb_qk, scaled_inv_freq
torch.manual_seed(0)
x = [torch.randn(2, 300, 4, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3)]
do, g = torch.randn_like(x[0]), torch.full((4,), -0.02, device="cuda")
freq = scaled_inv_freq(64, device="cuda")[0]

def step():
    q, k = apply_rotary_emb_qk(x[0], x[1], freq)
    out = fa.linear_attn_func(q, k, x[2], g)
    return (out,) + torch.autograd.grad(out, x, do)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
print([bool(torch.equal(a, b)) for a, b in zip(got, step())], fa.device_error())
"""


def test_first_calls_of_a_process_captured():
    """No call before the capture: kernels are loaded, and their limits raised, inside it."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(fa.__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED, root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split("]")[0] == "[True, True, True, True" and r.stdout.split()[-1] == "0", r.stdout + r.stderr
