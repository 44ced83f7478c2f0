"""The status of the row operators' launches and the limit of their waits, on the host (no GPU)."""
import ctypes as C

import pytest

import mgg_osdi23_b200 as mgg
from mgg_osdi23_b200._lib import check, lib


def test_the_limit_of_waits_is_checked_and_restored():
    before = C.c_int64()
    for bad in (-2, 2 ** 22 + 1, 2 ** 40):
        with pytest.raises(mgg.MggbError, match="operator_wait_limit"):
            check(lib.mggb_operator_wait_limit(bad, None))
    check(lib.mggb_operator_wait_limit(5, C.byref(before)))
    assert before.value == 2 ** 22
    check(lib.mggb_operator_wait_limit(-1, C.byref(before)))
    assert before.value == 5
    check(lib.mggb_operator_wait_limit(2 ** 22, C.byref(before)))
    assert before.value == 2 ** 22


def test_the_status_wants_a_place_to_write():
    with pytest.raises(mgg.MggbError, match="operator_device_status"):
        check(lib.mggb_operator_device_status(None, 0))
