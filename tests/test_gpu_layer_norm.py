"""Layer norm, forward and backward, against the formulas in 64 bits."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                        # half a step of fp32, relative
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one feature to wide rows, odd widths, widths whose rows are not 16- or 8- or 4-byte aligned
SHAPES = [(1, 1), (3, 2), (5, 7), (64, 16), (33, 31), (129, 33), (70, 100), (257, 128), (97, 602), (40, 601), (1000, 64),
          (17, 1000), (9, 1024), (6, 1025), (5, 4096), (3, 4099), (2, 8192), (4, 8200), (3, 16384), (2, 16390), (1, 40000), (2500, 41)]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps     # a whole step below the normal range


def adds(d):
    """Roundings on the way of one term into a row's sum: every lane of 32 adds its share, then a tree."""
    return d / 32 + 16


def inputs(n, d, t, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=g, device="cuda") * 0.7 + torch.randn(n, 1, generator=g, device="cuda") * 3
    return x.to(t), torch.randn(n, d, generator=g, device="cuda").to(t), 1 + 0.2 * torch.randn(d, generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda")


def forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    var = ((x - mean[:, None]) ** 2).mean(1)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (x - mean[:, None]) * rstd[:, None]
    w = torch.ones(x.shape[1], device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], device=x.device, dtype=torch.float64) if b is None else b.double()
    return xhat * w + b, mean, rstd, xhat


def check_forward(out, mean, rstd, x, w, b, eps):
    want, m, r, xhat = forward64(x, w, b, eps)
    d = x.shape[1]
    x64 = x.double()
    e_mean = adds(d) * U * x64.abs().mean(1)
    # the squared deviations carry twice the error of one deviation; the root halves it again
    e_rstd = (adds(d) + 8) * U + (e_mean * r)
    dev = (x64 - m[:, None]).abs()
    aw = 1.0 if w is None else w.double().abs()
    ab = 0.0 if b is None else b.double().abs()
    tol = (half(out.dtype) * want.abs() + tiny(out.dtype)
           + aw * (r[:, None] * (e_mean[:, None] + 2 * U * dev) + (e_rstd[:, None] + 2 * U) * xhat.abs()) + 2 * U * (want.abs() + ab))
    assert ((out.double() - want).abs() <= tol * (1 + 2.0 ** -7)).all()
    assert ((mean.double() - m).abs() <= e_mean + U * m.abs()).all()
    assert ((rstd.double() - r).abs() <= (e_rstd + 4 * U) * r).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,d", SHAPES)
def test_forward_matches_the_formula(n, d, t):
    x, _, w, b = inputs(n, d, t)
    for weight, bias in ((w, b), (None, None), (w, None)):
        out = torch.full_like(x, 7.0)
        mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        mgg.layer_norm_forward(out, x, weight, bias, 1e-5, mean=mean, rstd=rstd)
        check_forward(out, mean, rstd, x, weight, bias, 1e-5)
        again = torch.empty_like(x)
        mgg.layer_norm_forward(again, x, weight, bias, 1e-5)                 # without the statistics: the same bits
        assert torch.equal(out, again)


def backward64(dy, x, mean, rstd, w):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xhat = (x - mean) * rstd
    g = dy if w is None else dy * w.double()
    a, c = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - a - xhat * c)
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0), size, (dy * xhat).abs().sum(0), dy.abs().sum(0), (dy.abs() * (x.abs() + mean.abs()) * rstd).sum(0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,d", SHAPES)
def test_backward_matches_the_formula(n, d, t):
    x, dy, w, b = inputs(n, d, t, seed=1)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    mean, rstd = m.float(), r.float()
    for weight in (w, None):
        dx, dw, db = torch.full_like(x, 7.0), torch.full((d,), 7.0, device="cuda"), torch.full((d,), 7.0, device="cuda")
        mgg.layer_norm_backward(dx, dy, x, mean, rstd, weight, dweight=dw, dbias=db)
        want, want_w, want_b, size, size_w, size_b, cancel = backward64(dy, x, mean, rstd, weight)
        # xhat itself is formed with one rounding of x - mean and one of the product
        tol = half(t) * want.abs() + tiny(t) + (adds(d) + 12) * U * size
        assert ((dx.double() - want).abs() <= tol * (1 + 2.0 ** -7)).all()
        # a sum over n rows: at most n additions on a term's way, two roundings in the term
        assert ((dw.double() - want_w).abs() <= (n + 4) * U * size_w + 2 * U * cancel).all()
        assert ((db.double() - want_b).abs() <= (n + 2) * U * size_b).all()
        # each output alone, and the same bits again
        only = torch.empty_like(x)
        mgg.layer_norm_backward(only, dy, x, mean, rstd, weight)
        assert torch.equal(only, dx)
        ow, ob = torch.empty_like(dw), torch.empty_like(db)
        mgg.layer_norm_backward(None, dy, x, mean, rstd, weight, dweight=ow)
        mgg.layer_norm_backward(None, dy, x, mean, rstd, weight, dbias=ob)
        assert torch.equal(ow, dw) and torch.equal(ob, db)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,d", [(1, 5), (7, 16), (5000, 16), (4099, 41), (300_007, 3), (20_011, 100), (3000, 602), (2049, 1024), (777, 4099), (300, 16384), (37, 20000)])
def test_the_weights_gradient_misses_no_row(n, d, t):
    """With mean 0, rstd 1 and small whole numbers every product and sum is exact in fp32, whatever the order."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-2, 3, (n, d), generator=g, device="cuda").to(t)
    dy = torch.randint(-3, 4, (n, d), generator=g, device="cuda").to(t)
    dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    mgg.layer_norm_backward(None, dy, x, torch.zeros(n, device="cuda"), torch.ones(n, device="cuda"), dweight=dw, dbias=db)
    assert torch.equal(dw.double(), (dy.double() * x.double()).sum(0))
    assert torch.equal(db.double(), dy.double().sum(0))


def test_gradient_agrees_with_differences():
    n, d = 5, 24
    x, dy, w, b = inputs(n, d, torch.float32, seed=4)
    mean, rstd, out = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x)
    mgg.layer_norm_forward(out, x, w, b, 1e-3, mean=mean, rstd=rstd)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)

    def loss(x, w, b):
        return float((forward64(x, w, b, 1e-3)[0] * dy.double()).sum())
    h = 1e-5
    for grad, var, at in ((dx, x, (2, 3)), (dx, x, (4, 23)), (dw, w, (5,)), (db, b, (7,))):
        hi, lo = var.double().clone(), var.double().clone()
        hi[at] += h
        lo[at] -= h
        args = lambda v: tuple(v if a is var else a for a in (x, w, b))
        diff = (loss(*args(hi)) - loss(*args(lo))) / (2 * h)
        # differences in 64 bits: h^2 times a third derivative of a few hundred, and the kernel's fp32 sums of d or n terms
        assert abs(float(grad[at]) - diff) <= 1e-6 + 64 * U * (1 + abs(diff)) * 16


@pytest.mark.parametrize("t", TYPES)
def test_rows_far_apart_and_odd_offsets(t):
    """Views of some columns: rows that start at any element, strides of any length."""
    n = 67
    for d, off, wide in ((16, 1, 19), (100, 3, 131), (64, 8, 96), (602, 2, 610), (4096, 5, 4111), (1500, 4, 1504)):
        g = torch.Generator(device="cuda").manual_seed(d)
        big = torch.randn(n, wide, generator=g, device="cuda").to(t)
        big_dy = torch.randn(n, wide + 3, generator=g, device="cuda").to(t)
        x, dy = big[:, off:off + d], big_dy[:, 1:1 + d]
        w, b = torch.randn(d, generator=g, device="cuda"), torch.randn(d, generator=g, device="cuda")
        holder = torch.full((n, wide + 5), 9.0, device="cuda", dtype=t)
        out = holder[:, 2:2 + d]
        mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        mgg.layer_norm_forward(out, x, w, b, mean=mean, rstd=rstd)
        check_forward(out, mean, rstd, x, w, b, 1e-5)
        assert (holder[:, :2] == 9).all() and (holder[:, 2 + d:] == 9).all()
        holder.fill_(9.0)
        dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
        mgg.layer_norm_backward(out, dy, x, mean, rstd, w, dweight=dw, dbias=db)
        want, want_w, want_b, size, size_w, size_b, cancel = backward64(dy, x, mean, rstd, w)
        assert ((out.double() - want).abs() <= (half(t) * want.abs() + tiny(t) + (adds(d) + 12) * U * size) * (1 + 2.0 ** -7)).all()
        assert ((dw.double() - want_w).abs() <= (n + 4) * U * size_w + 2 * U * cancel).all()
        assert (holder[:, :2] == 9).all() and (holder[:, 2 + d:] == 9).all()
        # a weight that starts off a 16-byte boundary: the same bits
        odd_w, odd_b = torch.empty(d + 1, device="cuda")[1:].copy_(w), torch.empty(d + 1, device="cuda")[1:].copy_(b)
        one, two = torch.empty(n, d, device="cuda", dtype=t), torch.empty(n, d, device="cuda", dtype=t)
        mgg.layer_norm_forward(one, x, w, b)
        mgg.layer_norm_forward(two, x, odd_w, odd_b)
        assert torch.equal(one, two)


@pytest.mark.parametrize("n,d", [(200, 64), (50, 602), (9, 4096), (3, 20000)])
def test_in_place(n, d):
    x, dy, w, b = inputs(n, d, torch.float32, seed=5)
    mean, rstd, out = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x)
    mgg.layer_norm_forward(out, x, w, b, mean=mean, rstd=rstd)
    y = x.clone()
    mgg.layer_norm_forward(y, y, w, b)
    assert torch.equal(y, out)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)
    for which in ("dy", "x"):
        a, c = dy.clone(), x.clone()
        dw2, db2 = torch.empty_like(w), torch.empty_like(b)
        mgg.layer_norm_backward(a if which == "dy" else c, a, c, mean, rstd, w, dweight=dw2, dbias=db2)
        assert torch.equal(a if which == "dy" else c, dx)
        assert torch.equal(dw2, dw) and torch.equal(db2, db)


def test_constant_rows_large_offsets_and_bad_values():
    d = 256
    x = torch.zeros(6, d, device="cuda")
    x[1] = 5.0
    x[2] = 1e4 + torch.arange(d, device="cuda") / 16        # spread 4.6 on an offset of 10^4
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    x[5] = torch.arange(d, device="cuda", dtype=torch.float32)
    out, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    b = torch.randn(d, device="cuda")
    mgg.layer_norm_forward(out, x, None, b, mean=mean, rstd=rstd)
    assert torch.equal(out[0], b) and torch.equal(out[1], b)     # no spread: the bias alone
    ok = [0, 1, 2, 5]
    check_forward(out[ok], mean[ok], rstd[ok], x[ok], None, b, 1e-5)
    assert out[3].isnan().all() and out[4].isnan().all() and out[ok].isfinite().all()


def test_no_rows():
    x = torch.empty(0, 8, device="cuda")
    mgg.layer_norm_forward(torch.empty_like(x), x)
    dw, db = torch.full((8,), 7.0, device="cuda"), torch.full((8,), 7.0, device="cuda")
    mgg.layer_norm_backward(torch.empty_like(x), x, x, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), dweight=dw, dbias=db)
    assert (dw == 0).all() and (db == 0).all()


def test_captured_and_replayed_on_another_stream():
    n, d = 700, 100
    x, dy, w, b = inputs(n, d, torch.bfloat16, seed=6)
    out, mean, rstd = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def step():
        mgg.layer_norm_forward(out, x, w, b, mean=mean, rstd=rstd)
        mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs = []
    for _ in range(2):                       # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            step()
        graphs.append(graph)
    for k in range(4):
        nx, ndy, _, _ = inputs(n, d, torch.bfloat16, seed=10 + k)
        x.copy_(nx)
        dy.copy_(ndy)
        graphs[k % 2].replay()
        got = [t.clone() for t in (out, mean, rstd, dx, dw, db)]
        step()
        assert all(torch.equal(a, b_) for a, b_ in zip(got, (out, mean, rstd, dx, dw, db)))


def test_no_bounded_wait_expired():
    import ctypes as C
    from mgg_osdi23_b200._lib import check, lib
    st = C.c_int(-1)
    check(lib.mggb_operator_device_status(C.byref(st), 0))
    assert st.value == 0


def test_offsets_beyond_32_bits():
    n, d = 560_000, 4096
    x = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    tail, dy_tail, w, b = inputs(64, d, torch.bfloat16, seed=8)
    x[-64:] = tail
    mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    out = torch.empty_like(x)
    mgg.layer_norm_forward(out, x, w, b, mean=mean, rstd=rstd)
    check_forward(out[-64:], mean[-64:], rstd[-64:], tail, w, b, 1e-5)
    assert torch.equal(out[0], b.to(torch.bfloat16)) and torch.equal(out[n // 2], out[0])
    dy = torch.zeros_like(x)
    dy[-64:] = dy_tail
    dx, dw, db = out, torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)
    small = [torch.empty_like(tail), torch.empty_like(dw), torch.empty_like(db)]
    mgg.layer_norm_backward(small[0], dy_tail, tail, mean[-64:].contiguous(), rstd[-64:].contiguous(), w, dweight=small[1], dbias=small[2])
    assert torch.equal(dx[-64:], small[0]) and (dx[:-64] == 0).all()
    # the same 64 terms per column, in another order
    _, _, _, _, size_w, size_b, _ = backward64(dy_tail, tail, mean[-64:], rstd[-64:], w)
    assert ((dw - small[1]).abs().double() <= 130 * U * size_w).all() and ((db - small[2]).abs().double() <= 130 * U * size_b).all()


def test_two_streams_with_workspaces_of_their_own():
    import ctypes as C
    from mgg_osdi23_b200._lib import check, lib
    n, d = 20_000, 602
    x, dy, w, b = inputs(n, d, torch.float32, seed=9)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    mean, rstd = m.float(), r.float()
    need = C.c_size_t()
    check(lib.mggb_layer_norm_backward_scratch_bytes(n, d, C.byref(need)))
    want = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)]
    mgg.layer_norm_backward(want[0], dy, x, mean, rstd, w, dweight=want[1], dbias=want[2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(v) for v in want] + [torch.empty(need.value, dtype=torch.uint8, device="cuda")] for _ in streams]
    for _ in range(5):
        for st, (dx, dw, db, scratch) in zip(streams, got):
            with torch.cuda.stream(st):
                mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db, scratch=scratch)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, c) for a, c in zip(g, want))
    with pytest.raises(mgg.MggbError, match="scratch"):
        mgg.layer_norm_backward(None, dy, x, mean, rstd, w, dweight=want[1], scratch=torch.empty(need.value - 1, dtype=torch.uint8, device="cuda"))
