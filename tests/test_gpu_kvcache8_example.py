"""The serving example end to end: chunked prefill and decode over an 8-bit cache against the same layer over an
unquantised one.

Tolerance: N(0, 1) values in blocks of 16 x 128 reach about 3.9, so an int8 step is 0.031 and its error 0.0089 of a value's
rms; e4m3 codes err by up to 2^-4, 0.027 rms of a value.  V carries that into the output as it is, K as a random error of
the same size in each score (q is N(0, 1), the score scale 1 / sqrt(d)), hence of each weight: sqrt(2) times it, 0.0126 and
0.038, with bf16's 0.002 beside them.  The bars are 1.5 times that."""
import importlib.util
import os

import pytest

import fa_abi as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bar", [("int8", 0.019), ("e4m3", 0.057)])
def test_example(dtype, bar):
    path = os.path.join(A.ROOT, "flash-attention-rdna2_b200", "examples", "serve_8bit_cache.py")
    spec = importlib.util.spec_from_file_location("serve_8bit_cache", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(["--dtype", dtype, "--steps", "8"]) <= bar
