"""Products grouped by node type, forward and both gradients, against 64-bit products."""
import math

import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# (sizes of the groups, dim1, dim2): single rows, empty groups at every place, sizes around the tiles, odd and narrow widths
CASES = [([1], 1, 1), ([3], 2, 5), ([0, 1, 0], 7, 3), ([5, 0, 9], 16, 16), ([130, 1, 127], 32, 64), ([64, 64, 0, 200], 100, 47),
         ([33, 257, 1], 41, 602), ([300], 602, 16), ([1] * 40, 64, 128), ([0, 0, 0, 17], 128, 128), ([255, 256, 257], 64, 256),
         ([20, 500, 3, 0, 77], 129, 130), ([61], 1024, 48), ([10, 2, 0, 0, 30, 1], 256, 512), ([1000, 2000], 96, 33), ([4000], 8, 8), ([129, 640], 72, 200),
         ([2, 3, 1], 300, 1000), ([700], 513, 257)]


def half(t):
    return torch.finfo(t).eps / 2


def rows_of(sizes, first=0):
    out, a = [], first
    for s in sizes:
        out.append(slice(a, a + s))
        a += s
    return out


def pointers(sizes, first=0):
    return torch.tensor([first] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)


def random_case(sizes, k, m, t, seed=0, first=0, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = first + sum(sizes) + tail
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return r(n, k).to(t), (r(len(sizes), k, m) / math.sqrt(k)).to(t), r(n, m).to(t), pointers(sizes, first)


def bound(t, terms):
    """What a sum of `terms` products may be off relative to the sum of their magnitudes, before it is rounded: fp32
    operands go in with at least 21 bits each (2^-21 for the pair's dropped parts), every product is added in fp32."""
    return (2.0 ** -21 if t == torch.float32 else 0.0) + (terms + 2) * 2.0 ** -23


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sizes,k,m", CASES)
def test_products_match(sizes, k, m, t):
    for first, tail in ((0, 0), (3, 5)):
        x, w, dy, ptr = random_case(sizes, k, m, t, first=first, tail=tail)
        n = x.shape[0]
        out, dx = torch.full((n, m), 7.0, device="cuda", dtype=t), torch.full((n, k), 7.0, device="cuda", dtype=t)
        dw = torch.full((len(sizes), k, m), 7.0, device="cuda")
        mgg.grouped_dense_forward(out, x, w, ptr)
        mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
        X, W, D = x.double(), w.double(), dy.double()
        for g, r in enumerate(rows_of(sizes, first)):
            for got, a, b, terms in ((out[r], X[r], W[g], k), (dx[r], D[r], W[g].T, m), (dw[g], X[r].T, D[r], r.stop - r.start)):
                want, size = a @ b, a.abs() @ b.abs()
                tol = (half(t) * (1 + 2.0 ** -7) * want.abs() + 2.0 ** -25 if got.dtype != torch.float32 else 0) + bound(t, terms) * size
                assert ((got.double() - want).abs() <= tol).all()
        for whole in (out, dx):                                # rows of no group stay as they were
            assert (whole[:first] == 7).all() and (whole[n - tail:] == 7).all()
        # each gradient alone, and again: the same bits
        a, b = torch.full_like(dx, 7.0), torch.empty_like(dw)
        mgg.grouped_dense_backward(a, None, dy, x, w, ptr)
        mgg.grouped_dense_backward(None, b, dy, x, w, ptr)
        assert torch.equal(a, dx) and torch.equal(b, dw)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sizes,k,m", [([40_000, 3, 0, 9000], 24, 40), ([5, 70_001], 41, 16), ([3000] * 20, 64, 64), ([2500, 1, 900], 640, 384), ([100] * 100, 48, 100)])
def test_whole_numbers_are_exact(sizes, k, m, t):
    """Entries of -1, 0, 1: every product and every sum below 2^24 is exact, so a missed or doubled row or column shows.
    16-bit outputs hold the sums as long as those stay within 256; the entries of x and dy are sparse enough for that."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n = sum(sizes)
    few = lambda *s: (torch.randint(-1, 2, s, generator=g, device="cuda") * (torch.rand(*s, generator=g, device="cuda") < 0.2)).to(t)
    x, w, dy, ptr = few(n, k), torch.randint(-1, 2, (len(sizes), k, m), generator=g, device="cuda").to(t), few(n, m), pointers(sizes)
    out, dx, dw = torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(len(sizes), k, m, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    for i, r in enumerate(rows_of(sizes)):
        X, W, D = x[r].double(), w[i].double(), dy[r].double()
        assert torch.equal(out[r].double(), X @ W)
        assert torch.equal(dx[r].double(), D @ W.T)
        assert torch.equal(dw[i].double(), X.T @ D)


@pytest.mark.parametrize("t", TYPES)
def test_any_pointers_stay_inside(t):
    """Pointers below 0, past the rows or falling: clamped to the rows and made monotone, nothing else is touched."""
    n, k, m = 50, 24, 40
    x, w, dy, _ = random_case([n], k, m, t)
    w = torch.randn(4, k, m, device="cuda").to(t) / 5
    for raw, fixed in (([-7, 10, 20, 30, 40], [0, 10, 20, 30, 40]), ([0, 30, 10, 45, 90], [0, 30, 30, 45, 50]), ([60, 70, 0, 5, 2 ** 31 - 1], [50, 50, 50, 50, 50]),
                       ([5, 5, 5, 5, 5], [5] * 5), ([-2 ** 31, -1, 0, 50, 50], [0, 0, 0, 50, 50]), ([10, -3, 12, 11, 49], [10, 10, 12, 12, 49])):
        res = []
        for p in (raw, fixed):
            ptr = torch.tensor(p, device="cuda", dtype=torch.int32)
            out, dx, dw = torch.full((n, m), 7.0, device="cuda", dtype=t), torch.full((n, k), 7.0, device="cuda", dtype=t), torch.full((4, k, m), 7.0, device="cuda")
            mgg.grouped_dense_forward(out, x, w, ptr)
            mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
            res.append((out, dx, dw))
        assert all(torch.equal(a, b) for a, b in zip(*res))
        assert (res[0][0][: fixed[0]] == 7).all() and (res[0][0][fixed[-1]:] == 7).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k,m", [(64, 64), (40, 24), (33, 17), (128, 256)])
def test_neighbours_do_not_leak(k, m, t):
    """NaN in the other groups' rows and weights, and behind the last group, reaches no group's own results."""
    sizes = [70, 5, 0, 131]
    n = sum(sizes) + 9
    x, w, dy, ptr = random_case(sizes, k, m, t, tail=9)
    clean = [torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(4, k, m, device="cuda")]
    mgg.grouped_dense_forward(clean[0], x, w, ptr)
    mgg.grouped_dense_backward(clean[1], clean[2], dy, x, w, ptr)
    rows = rows_of(sizes)
    for g in (0, 1, 3):
        x2, w2, dy2 = torch.full_like(x, math.nan), torch.full_like(w, math.nan), torch.full_like(dy, math.nan)
        x2[rows[g]], w2[g], dy2[rows[g]] = x[rows[g]], w[g], dy[rows[g]]
        out, dx, dw = torch.empty_like(clean[0]), torch.empty_like(clean[1]), torch.empty_like(clean[2])
        mgg.grouped_dense_forward(out, x2, w2, ptr)
        mgg.grouped_dense_backward(dx, dw, dy2, x2, w2, ptr)
        assert torch.equal(out[rows[g]], clean[0][rows[g]]) and torch.equal(dx[rows[g]], clean[1][rows[g]]) and torch.equal(dw[g], clean[2][g])
        assert (dw[2] == 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_odd_addresses(t):
    """Matrices that start at any element of their storage: the same bits as aligned ones, nothing written beside them."""
    sizes, k, m = [90, 200, 1], 64, 72
    x, w, dy, ptr = random_case(sizes, k, m, t)
    n = x.shape[0]

    def odd(v, by):
        return torch.empty(v.numel() + by + 8, device="cuda", dtype=v.dtype).fill_(7.0)[by: by + v.numel()].view(v.shape).copy_(v)
    want = [torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(3, k, m, device="cuda")]
    mgg.grouped_dense_forward(want[0], x, w, ptr)
    mgg.grouped_dense_backward(want[1], want[2], dy, x, w, ptr)
    for by in (1, 2, 4):
        got = [odd(torch.zeros_like(v), by) for v in want]
        mgg.grouped_dense_forward(got[0], odd(x, by), odd(w, by), ptr)
        mgg.grouped_dense_backward(got[1], got[2], odd(dy, by), odd(x, by), odd(w, by), ptr)
        for a, b in zip(got, want):
            # another order of the same sums is allowed where another kernel takes unaligned matrices
            size = float(b.double().abs().max())
            assert float((a.double() - b.double()).abs().max()) <= (2 * half(t) + 2.0 ** -14) * size


def test_gradients_agree_with_differences():
    sizes, k, m = [3, 0, 4], 5, 6
    x, w, dy, ptr = random_case(sizes, k, m, torch.float32, seed=8)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)

    def loss(x, w):
        return float(sum(((x[r].double() @ w[g].double()) * dy[r].double()).sum() for g, r in enumerate(rows_of(sizes))))
    h = 1e-4
    for grad, var, at in ((dx, x, (1, 2)), (dx, x, (6, 4)), (dw, w, (0, 4, 1)), (dw, w, (1, 2, 2)), (dw, w, (2, 0, 5))):
        hi, lo = var.double().clone(), var.double().clone()
        hi[at] += h
        lo[at] -= h
        args = lambda v: (v, w) if var is x else (x, v)
        diff = (loss(*args(hi)) - loss(*args(lo))) / (2 * h)            # the loss is linear in each: differences are exact but for 64-bit roundings
        assert abs(float(grad[at]) - diff) <= 1e-9 + 20 * 2.0 ** -21 * (1 + abs(diff))


def test_no_rows_and_no_members():
    w = torch.randn(3, 16, 24, device="cuda")
    x, dy = torch.empty(0, 16, device="cuda"), torch.empty(0, 24, device="cuda")
    ptr = torch.zeros(4, device="cuda", dtype=torch.int32)
    mgg.grouped_dense_forward(torch.empty(0, 24, device="cuda"), x, w, ptr)
    dw = torch.full((3, 16, 24), 7.0, device="cuda")
    mgg.grouped_dense_backward(torch.empty(0, 16, device="cuda"), dw, dy, x, w, ptr)
    assert (dw == 0).all()
    x, dy, out = torch.randn(20, 16, device="cuda"), torch.randn(20, 24, device="cuda"), torch.full((20, 24), 7.0, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    dw.fill_(7.0)
    mgg.grouped_dense_backward(None, dw, dy, x, w, ptr)
    assert (out == 7).all() and (dw == 0).all()


def test_many_groups():
    """The largest number of types, most of them empty."""
    groups, k, m, n = 4096, 8, 8, 3000
    g = torch.Generator().manual_seed(9)
    cuts = torch.sort(torch.randint(0, n + 1, (groups - 1,), generator=g)).values
    ptr = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), n)]).to(device="cuda", dtype=torch.int32)
    x, dy = torch.randint(-2, 3, (n, k), device="cuda").float(), torch.randint(-2, 3, (n, m), device="cuda").float()
    w = torch.randint(-2, 3, (groups, k, m), device="cuda").float()
    gid = torch.repeat_interleave(torch.arange(groups, device="cuda"), (ptr[1:] - ptr[:-1]).long())
    out, dx, dw = torch.empty(n, m, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty_like(w)
    mgg.grouped_dense_forward(out, x, w, ptr)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    assert torch.equal(out, torch.einsum("nk,nkm->nm", x, w[gid]))
    assert torch.equal(dx, torch.einsum("nm,nkm->nk", dy, w[gid]))
    assert torch.equal(dw, torch.zeros_like(w).index_add_(0, gid, x[:, :, None] * dy[:, None, :]))


@pytest.mark.parametrize("t", TYPES)
def test_captured_replayed_with_new_sizes(t):
    """The sizes are read at run time: a replayed graph takes the groups it finds in group_ptr."""
    n, k, m = 400, 64, 96
    x, w, dy, _ = random_case([n], k, m, t)
    w = (torch.randn(3, k, m, device="cuda") / 8).to(t)
    ptr = pointers([100, 200, 100])
    out, dx, dw = torch.zeros(n, m, device="cuda", dtype=t), torch.zeros(n, k, device="cuda", dtype=t), torch.zeros(3, k, m, device="cuda")

    def step():
        mgg.grouped_dense_forward(out, x, w, ptr)
        mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        step()
    for sizes in ([400, 0, 0], [1, 2, 397], [0, 130, 270]):
        ptr.copy_(pointers(sizes))
        for v in (out, dx, dw):
            v.fill_(7.0)
        graph.replay()
        got = [v.clone() for v in (out, dx, dw)]
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, dx, dw)))


def test_no_bounded_wait_expired():
    import ctypes as C
    from mgg_osdi23_b200._lib import check, lib
    st = C.c_int(-1)
    check(lib.mggb_operator_device_status(C.byref(st), 0))
    assert st.value == 0


@pytest.mark.parametrize("t", TYPES)
def test_many_groups_of_wide_weights(t):
    """The largest number of types through the tensor cores: what is left of shared memory beside the lists is enough."""
    groups, k, m, n = 4096, 72, 80, 6000
    g = torch.Generator().manual_seed(10)
    cuts = torch.sort(torch.randint(0, n + 1, (groups - 1,), generator=g)).values
    ptr = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), n)]).to(device="cuda", dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(10)
    whole = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(t)
    x, dy, w = whole(n, k), whole(n, m), whole(groups, k, m)
    gid = torch.repeat_interleave(torch.arange(groups, device="cuda"), (ptr[1:] - ptr[:-1]).long())
    out, dx, dw = torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(groups, k, m, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    per_row = w[gid].float()
    assert torch.equal(out.float(), torch.bmm(x[:, None].float(), per_row)[:, 0])
    assert torch.equal(dx.float(), torch.bmm(per_row, dy[:, :, None].float())[:, :, 0])
    assert torch.equal(dw, torch.zeros_like(dw).index_add_(0, gid, x[:, :, None].float() * dy[:, None, :].float()))


@pytest.mark.parametrize("t", TYPES)
def test_long_sums_stay_fp32(t):
    """A tensor-core instruction cuts up to 2^-23 off the accumulator; a sum leaves it after at most 48 of them (768 terms), so
    fp32 results are within 48 * 2^-23 + 2^-21 of their norm however long the sum."""
    sizes, k, m = [9000, 50], 2048, 96
    x, w, dy, ptr = random_case(sizes, k, m, t, seed=11)
    n = sum(sizes)
    out, dx, dw = torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(2, k, m, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    for g, r in enumerate(rows_of(sizes)):
        X, W, D = x[r].double(), w[g].double(), dy[r].double()
        for got, want in ((out[r], X @ W), (dx[r], D @ W.T), (dw[g], X.T @ D)):
            off = float((got.double() - want).norm() / want.norm())
            assert off <= 48 * 2.0 ** -23 + 2.0 ** -21 + (half(got.dtype) if got.dtype != torch.float32 else 0.0)


def test_two_streams_with_workspaces_of_their_own():
    """Calls that overlap share nothing but their inputs."""
    import ctypes as C
    from mgg_osdi23_b200._lib import check, lib
    sizes, k, m = [30_000, 20_000], 100, 47
    x, w, dy, ptr = random_case(sizes, k, m, torch.float32, seed=12)
    n = sum(sizes)
    need = C.c_size_t()
    check(lib.mggb_grouped_dense_backward_scratch_bytes(n, 2, k, m, 0, C.byref(need)))
    assert need.value > 0
    want = [torch.empty_like(x), torch.empty(2, k, m, device="cuda")]
    mgg.grouped_dense_backward(want[0], want[1], dy, x, w, ptr)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(x), torch.empty(2, k, m, device="cuda"), torch.empty(need.value, dtype=torch.uint8, device="cuda")] for _ in streams]
    for _ in range(5):
        for st, (dx, dw, scratch) in zip(streams, got):
            with torch.cuda.stream(st):
                mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr, scratch=scratch)
    torch.cuda.synchronize()
    for dx, dw, _ in got:
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    with pytest.raises(mgg.MggbError, match="scratch"):
        mgg.grouped_dense_backward(None, want[1], dy, x, w, ptr, scratch=torch.empty(need.value - 1, dtype=torch.uint8, device="cuda"))


def test_offsets_beyond_32_bits():
    """Rows whose element offsets pass 2^31."""
    n, k, m = 1_100_000, 2048, 8
    x = torch.zeros(n, k, device="cuda", dtype=torch.bfloat16)
    tail = torch.randint(-2, 3, (300, k), device="cuda").to(torch.bfloat16)
    x[-300:] = tail
    w = torch.randint(-1, 2, (2, k, m), device="cuda").to(torch.bfloat16)
    ptr = pointers([n - 300, 300])
    out = torch.empty(n, m, device="cuda", dtype=torch.bfloat16)
    mgg.grouped_dense_forward(out, x, w, ptr)
    assert torch.equal(out[-300:].double(), (tail.double() @ w[1].double()).to(torch.bfloat16).double()) and (out[:-300] == 0).all()
    w16 = torch.randint(-1, 2, (2, k, 16), device="cuda").to(torch.bfloat16)
    out = torch.empty(n, 16, device="cuda", dtype=torch.bfloat16)
    mgg.grouped_dense_forward(out, x, w16, ptr)
    assert torch.equal(out[-300:].double(), (tail.double() @ w16[1].double()).to(torch.bfloat16).double()) and (out[:-300] == 0).all()
    dw = torch.empty(2, k, 16, device="cuda")
    dy = torch.ones(n, 16, device="cuda", dtype=torch.bfloat16)
    mgg.grouped_dense_backward(None, dw, dy, x, w16, ptr)
    assert (dw[0] == 0).all() and torch.equal(dw[1].double(), tail.double().sum(0)[:, None].expand(k, 16))
