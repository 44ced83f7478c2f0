"""The status calls whose description says that they synchronise the device wait for streams that do not block the default one."""
import ctypes as C

import pytest
import torch

from mgg_osdi23_b200._lib import check, lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["mggb_agg_device_status", "mggb_dense_device_status", "mggb_operator_device_status"])
def test_the_status_waits_for_other_streams(name):
    side, st = torch.cuda.Stream(), C.c_int(-1)
    for _ in range(2):                                  # the second time nothing has to be loaded any more
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
        check(getattr(lib, name)(C.byref(st), 0))
        assert side.query() and st.value == 0
