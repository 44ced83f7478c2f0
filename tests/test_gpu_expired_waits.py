"""A bounded wait that runs out: the launch ends, the status tells, a reset clears it, and the next call is right.

The waits are made to run out by the limit itself (no data is ever missing): with a limit of 0 a wait gives up at once or
after one poll, while the copies it asked for are still under way."""
import contextlib
import ctypes as C

import pytest
import torch

import mgg_osdi23_b200 as mgg
from mgg_osdi23_b200._lib import check, lib

pytestmark = pytest.mark.gpu


def status(reset=0):
    torch.cuda.synchronize()
    st = C.c_int(-1)
    check(lib.mggb_operator_device_status(C.byref(st), reset))
    return st.value


@contextlib.contextmanager
def limit(polls):
    before = C.c_int64()
    check(lib.mggb_operator_wait_limit(polls, C.byref(before)))
    try:
        yield
    finally:
        check(lib.mggb_operator_wait_limit(before.value, None))


def guarded(shape, t):
    """A tensor of this shape with 64 elements of 7 on each side of it, and the whole of it."""
    n = 1
    for s in shape:
        n *= s
    whole = torch.full((n + 128,), 7.0, device="cuda", dtype=t)
    return whole[64: 64 + n].view(shape), whole


def expires_and_recovers(call, outputs):
    """call(outputs) with and without time to wait; outputs: (shape, type) each."""
    assert status() == 0
    want = [guarded(*o) for o in outputs]
    call([v for v, _ in want])
    assert status() == 0
    for polls in (0, 1, 0):
        got = [guarded(*o) for o in outputs]
        with limit(polls):
            call([v for v, _ in got])
        code = status(reset=1)
        assert code != 0 or polls > 0                       # one poll may last long enough
        assert status() == 0
        for _, whole in got:
            assert (whole[:64] == 7).all() and (whole[-64:] == 7).all()
        if code == 0:
            assert all(torch.equal(a, b) for (a, _), (b, _) in zip(got, want))
        again = [guarded(*o) for o in outputs]
        call([v for v, _ in again])
        assert status() == 0
        assert all(torch.equal(a, b) for (a, _), (b, _) in zip(again, want))


def grouped(sizes, k, m, t):
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)
    n = sum(sizes)
    x, w, dy = r(n, k), r(len(sizes), k, m), r(n, m)
    ptr = torch.tensor([0] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    expires_and_recovers(lambda o: mgg.grouped_dense_forward(o[0], x, w, ptr), [((n, m), t)])
    expires_and_recovers(lambda o: mgg.grouped_dense_backward(o[0], None, dy, x, w, ptr), [((n, k), t)])
    expires_and_recovers(lambda o: mgg.grouped_dense_backward(None, o[0], dy, x, w, ptr), [((len(sizes), k, m), torch.float32)])


# a weight that stays in shared memory, sums of two k-chunks, a weight that does not stay, many units per block, an empty group; 16-bit rows that no tensor map takes
@pytest.mark.parametrize("t,k,m", [(torch.float32, 128, 128), (torch.float32, 64, 72), (torch.float32, 602, 132), (torch.bfloat16, 129, 131), (torch.float16, 100, 210)])
@pytest.mark.parametrize("sizes", [[70], [40_000, 0, 3, 20_000]])
def test_grouped_products_through_registers(sizes, t, k, m):
    grouped(sizes, k, m, t)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_class_log_probabilities_of_narrow_rows(t):
    n, c = 5000, 47
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(n, c, generator=g, device="cuda").to(t)
    labels = torch.randint(0, c, (n,), generator=g, device="cuda", dtype=torch.int32)
    lp, stats = torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda")
    mgg.class_logprob_forward(lp, z, labels, stats=stats)
    f32, i32 = torch.float32, torch.int32
    expires_and_recovers(lambda o: mgg.class_logprob_forward(o[0], z, labels, top_ids=o[1], top_logprobs=o[2]), [((n,), f32), ((n, 5), i32), ((n, 5), f32)])
    expires_and_recovers(lambda o: mgg.class_logprob_backward(o[0], z, labels, stats, lp), [((n, c), t)])



# tensor copies: fewer k-chunks than the ring has stages (all asked for before any wait of the copying thread), and many more
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,k,m", [([70], 128, 128), ([40_000, 0, 3, 20_000], 128, 192), ([300, 61], 2048, 256), ([900] * 5, 640, 1024)])
def test_grouped_products_through_tensor_copies(sizes, k, m, t):
    grouped(sizes, k, m, t)


# lane groups of a warp and teams of warps, fewer rows than the rings hold and many more, rows that are no multiple of 16 bytes
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(3, 16), (20_000, 41), (9, 602), (5000, 602), (40, 4096), (3000, 4099), (700, 8192)])
def test_layer_norm_backward(n, d, t):
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dy, w = r(n, d).to(t), r(n, d).to(t), r(d)
    mean, rstd, y = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x)
    mgg.layer_norm_forward(y, x, w, None, mean=mean, rstd=rstd)
    expires_and_recovers(lambda o: mgg.layer_norm_backward(o[0], dy, x, mean, rstd, w, dweight=o[1], dbias=o[2]),
                         [((n, d), t), ((d,), torch.float32), ((d,), torch.float32)])
