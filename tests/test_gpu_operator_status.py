"""The status of the row operators' launches covers the work of every stream."""
import ctypes as C

import pytest
import torch

import mgg_osdi23_b200 as mgg
from mgg_osdi23_b200._lib import check, lib

pytestmark = pytest.mark.gpu


def test_the_status_waits_for_other_streams():
    """A launch that gives up behind a tenth of a second of work on a stream that does not block the default one."""
    z, labels, lp = torch.randn(1000, 47, device="cuda"), torch.zeros(1000, device="cuda", dtype=torch.int32), torch.empty(1000, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(2):                                  # the second time nothing has to be loaded any more
        mgg.class_logprob_forward(lp, z, labels)
        assert mgg.operator_status() == 0
        side.wait_stream(torch.cuda.current_stream())
        check(lib.mggb_operator_wait_limit(0, None))
        try:
            with torch.cuda.stream(side):
                torch.cuda._sleep(200_000_000)
                mgg.class_logprob_forward(lp, z, labels)
        finally:
            check(lib.mggb_operator_wait_limit(-1, None))
        code = mgg.operator_status(reset=True)
        assert side.query()
        torch.cuda.synchronize()
        assert code == 1 and mgg.operator_status() == 0


def test_a_status_that_is_not_reset_stays():
    z, labels, lp = torch.randn(100, 5, device="cuda"), torch.zeros(100, device="cuda", dtype=torch.int32), torch.empty(100, device="cuda")
    check(lib.mggb_operator_wait_limit(0, None))
    try:
        mgg.class_logprob_forward(lp, z, labels)
    finally:
        check(lib.mggb_operator_wait_limit(-1, None))
    assert mgg.operator_status() != 0 and mgg.operator_status() != 0
    assert mgg.operator_status(reset=True) != 0 and mgg.operator_status() == 0
    mgg.class_logprob_forward(lp, z, labels)
    assert mgg.operator_status() == 0
    want = torch.log_softmax(z.double(), 1)[:, 0]
    # five exponentials of relative error 2^-21 in a sum, and the roundings of a difference and a logarithm
    assert float((lp.double() - want).abs().max()) <= 2.0 ** -18


def test_the_status_is_the_current_devices():
    st = C.c_int(-1)
    check(lib.mggb_operator_device_status(C.byref(st), 0))
    assert st.value == mgg.operator_status() == 0
