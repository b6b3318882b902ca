"""CPU tests of the paged 8-bit cache operators' refusals where a call has rows but no sequences."""
import ctypes as C

import pytest

import fa_abi as A
from test_kvcache8_cpu import FaDec8Params, FaKvAppendParams, FaKvGatherParams, block


@pytest.mark.parametrize("fn,cls", [("fa_kv_append_launch", FaKvAppendParams), ("fa_kv_gather_launch", FaKvGatherParams),
                                    ("fa_decode8_launch", FaDec8Params)])
def test_rows_without_sequences(fn, cls):
    """Rows that nothing would write are refused, not passed over."""
    f = getattr(A.lib(), fn)
    assert f(C.byref(block(cls, batch=0, total=3, cu_new=16, cu_q=16)), 1, None) == A.FA_ERR_INVALID
    assert f(C.byref(block(cls, batch=0, total=0, cu_new=16, cu_q=16)), 1, None) == A.FA_OK
