"""Linear attention and the rotary of q and k at the edges of what they are given: the parts that run on the host."""
import ctypes as C
import math
import os
import random
import subprocess

import pytest

import fa_abi as A

CSRC = os.path.join(A.ROOT, "flash-attention-rdna2_b200", "csrc")

SLOTS = r"""
#include <cstdio>
#include <vector>
#include "linear_common.cuh"
// lines of: total S batch seg_len nseg cu[0] .. cu[batch]
int main() {
  long long total;
  int S, batch, len, nseg, line = 0;
  while (scanf("%lld %d %d %d %d", &total, &S, &batch, &len, &nseg) == 5) {
    std::vector<int> cu(batch + 1);
    for (int& x : cu) if (scanf("%d", &x) != 1) return 2;
    ++line;
    const long long slots = fa::lin_slots(true, total, batch, len, nseg);
    const fa::LinSeqs q{cu.data(), nullptr, total, batch, S, 1, len, nseg, (int)slots};
    std::vector<int> walked(slots, 0);
    for (int z = 0; z < batch; ++z) {                                  // as the join walks the workspace
      const fa::LinSpan s = fa::lin_span(q, z);
      const long long first = fa::lin_first_slot(q, z, s.row0);
      for (int m = 0; m < fa::lin_segments(q, s.len); ++m) {
        if (first + m < 0 || first + m >= slots) return printf("line %d: sequence %d has slot %lld of %lld\n", line, z, first + m, slots), 1;
        ++walked[first + m];
      }
    }
    long long rows = 0;
    for (int i = 0; i < slots; ++i) {                                  // as the states and outputs find their tokens
      int z, t0, t1;
      const fa::LinSpan s = fa::lin_segment(q, i, z, t0, t1);
      if ((t1 > t0) != walked[i]) return printf("line %d: slot %d has tokens [%d, %d) and is joined %d times\n", line, i, t0, t1, walked[i]), 1;
      if (t1 > t0) rows += t1 - t0;
    }
    long long want = 0;
    for (int z = 0; z < batch; ++z) want += fa::lin_span(q, z).len;
    if (rows != want) return printf("line %d: %lld rows of %lld\n", line, rows, want), 1;
  }
  return printf("%d", line) > 0 ? 0 : 3;
}
"""


@pytest.fixture(scope="module")
def slots_program(tmp_path_factory):
    """The segments' arithmetic of the kernels' own header, compiled for the host."""
    at = tmp_path_factory.mktemp("slots")
    (at / "slots.cu").write_text(SLOTS)
    subprocess.run([os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC,
                    "-I", os.path.dirname(A.HEADER), str(at / "slots.cu"), "-o", str(at / "slots")], check=True)
    return str(at / "slots")


def test_the_join_stays_in_its_workspace(slots_program):
    """Packed sequences, empty ones anywhere, offsets past the rows: the join touches slots of its own inside the workspace, the ones
    that have tokens.  One sequence has ceil(total / seg_len) slots and no more, so an empty one at the end has none."""
    rng = random.Random(0)
    lines = []
    for _ in range(4000):
        batch, seg = rng.choice([1, 1, 2, 3, 8]), rng.choice([1, 7, 32, 64, 128, 384])
        cut = lambda hi: min(hi, rng.choice([0, seg, 2 * seg, 3 * seg, rng.randrange(5 * seg + 1)]))
        total = rng.choice([seg, 4 * seg, 4 * seg - 1, rng.randrange(1, 6 * seg + 1)])
        cu = sorted(cut(total) for _ in range(batch + 1))
        if rng.random() < 0.5:
            cu[-1] = total
        if rng.random() < 0.3:
            cu = [total - (total % seg if rng.random() < 0.5 else 0)] * (batch + 1)      # nobody has a token
        if rng.random() < 0.2:
            cu = [x + total for x in cu]                                                   # past the rows
        nseg = max(1, -(-total // seg)) if rng.random() < 0.9 else 1
        lines.append(f"{total} {total} {batch} {seg} {nseg} " + " ".join(map(str, cu)))
    lines.append("512 512 1 128 4 512 512")
    r = subprocess.run([slots_program], input="\n".join(lines), capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == str(len(lines)), r.stdout


def test_narrowing_refusals():
    L = A.lib()
    L.fa_narrow_index_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]
    assert L.fa_narrow_index_launch(None, None, 0, None) == A.FA_OK
    for args in ((None, 16, 3, None), (16, None, 3, None), (16, 16, -1, None)):
        assert L.fa_narrow_index_launch(*args) == A.FA_ERR_INVALID


@pytest.mark.parametrize("dim,base,factor,length", [(64, 10000.0, 4.0, 4096), (128, 500000.0, 32.0, 8192), (16, 10000.0, 8.0, 256), (128, 10000.0, 1.0, 2048)])
def test_yarn_between_the_kept_and_the_divided(dim, base, factor, length):
    """Pair i turns length * base^(-2 i / dim) / (2 pi) times over the original length.  From the pair below the one that turns beta_fast = 32 times to the
    pair above the one that turns once, the share that is divided by `factor` grows by equal steps; every element against that, pair by pair."""
    from fable_attn.layers.rotary import scaled_inv_freq
    got, times = scaled_inv_freq(dim, base, "yarn", factor, length)
    of = lambda turns: dim / 2 * math.log(length / (2 * math.pi * turns)) / math.log(base)      # the (real) pair that turns so often
    first, last = max(math.floor(of(32.0)), 0), min(math.ceil(of(1.0)), dim - 1)
    assert first < last and 0 < sum(first < i < last for i in range(dim // 2))
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        share = 0.0 if i <= first else 1.0 if i >= last else (i - first) / (last - first)
        assert math.isclose(float(got[i]), f * ((1 - share) + share / factor), rel_tol=1e-12), i
    assert math.isclose(times, 1 + 0.1 * math.log(factor))
    slow, _ = scaled_inv_freq(dim, base, "yarn", factor, length, beta_fast=8.0, beta_slow=2.0)
    assert bool((slow <= got * (1 + 1e-12)).any()) and float(slow[0]) == 1.0
