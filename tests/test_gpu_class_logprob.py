"""Class log probabilities, entropy, alternatives and their gradient against the definitions in 64 bits."""
import math

import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (5, 2), (33, 3), (64, 16), (300, 41), (129, 47), (1000, 32), (65, 33), (257, 64), (40, 65), (77, 128), (31, 172), (9, 256), (20, 257),
          (6, 1000), (8, 1023), (5, 2048), (3, 4097), (2, 20_000), (3, 33_001), (1, 100_000), (2, 262_144), (130, 5000), (700, 1500)]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def inputs(n, c, t, seed=0, masked=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(n, c, generator=g, device="cuda") * 3 + torch.randn(n, 1, generator=g, device="cuda") * 8
    if c > 1 and masked:
        z[:, 1:].masked_fill_(torch.rand(n, c - 1, generator=g, device="cuda") < masked, -math.inf)
    labels = torch.randint(0, c, (n,), generator=g, device="cuda", dtype=torch.int32)
    labels[torch.rand(n, generator=g, device="cuda") < 0.3] = -1
    return z.to(t), labels


def forward64(z):
    z = z.double()
    m = z.amax(1, keepdim=True)
    d = torch.where(z == -math.inf, -math.inf, z - m)
    e = d.exp()
    s = e.sum(1, keepdim=True)
    L = torch.where((s == 0) & (m == -math.inf), 0.0, s.log())
    h = L - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / torch.where(s == 0, 1.0, s)
    return m, L, d - L, h


def best(z, k):
    """Classes by score, equal scores by class, NaN first."""
    return torch.sort(z.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :k].int()


def sum_error(c):
    """Relative error of the sum of c exponentials: 2^-21 for one of them (two units in the last place and the rounding
    of its argument, which is below 2^-22 where the term counts), c/32 + 16 additions on a term's way."""
    return 2.0 ** -21 + (c / 32 + 16) * U


def run_forward(z, labels, k):
    n = z.shape[0]
    o = dict(logprob=torch.full((n,), 7.0, device="cuda"), stats=torch.full((n, 2), 7.0, device="cuda"), entropy=torch.full((n,), 7.0, device="cuda"),
             top_ids=torch.full((n, k), -7, device="cuda", dtype=torch.int32) if k else None, top_logprobs=torch.full((n, k), 7.0, device="cuda") if k else None)
    mgg.class_logprob_forward(o["logprob"], z, labels, stats=o["stats"], entropy=o["entropy"], top_ids=o["top_ids"], top_logprobs=o["top_logprobs"])
    return o


def check_forward(o, z, labels):
    n, c = z.shape
    m, L, lp, h = forward64(z)
    y = labels.long()
    has = (y >= 0) & (y < c)
    want = torch.where(has, lp.gather(1, y.clamp(0, c - 1)[:, None])[:, 0], 0.0)
    tol_L = sum_error(c) + 2 * U * L[:, 0].abs()

    def close(got, want, tol):
        same = got.double() == want                            # infinities
        assert (same | ((got.double() - want).abs() <= tol)).all()
    close(o["logprob"], want, tol_L + 3 * U * want.abs())
    assert torch.equal(o["stats"][:, 0].double(), m[:, 0])
    close(o["stats"][:, 1], L[:, 0], tol_L)
    # the entropy is a sum of terms p |log p| <= L + log c: their relative error is the sums'
    close(o["entropy"], h[:, 0], 4 * sum_error(c) * (1 + math.log(c)) + 4 * U)
    if o["top_ids"] is not None:
        ids = best(z, o["top_ids"].shape[1])
        assert torch.equal(o["top_ids"], ids)
        if o["top_logprobs"] is not None:
            want = lp.gather(1, ids.long())
            close(o["top_logprobs"], want, tol_L[:, None] + 3 * U * want.abs().nan_to_num(posinf=0, neginf=0))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward_matches_the_definition(n, c, t):
    z, labels = inputs(n, c, t)
    for k in sorted({0, 1, min(c, 5), min(c, 32)}):
        o = run_forward(z, labels, k)
        check_forward(o, z, labels)
    # every output alone gives the same bits
    one = torch.empty_like(o["logprob"])
    mgg.class_logprob_forward(one, z, labels)
    assert torch.equal(one, o["logprob"])
    ent = torch.empty_like(one)
    mgg.class_logprob_forward(None, z, None, entropy=ent)
    assert torch.equal(ent, o["entropy"])
    if o["top_ids"] is not None:
        ids = torch.empty_like(o["top_ids"])
        mgg.class_logprob_forward(None, z, None, top_ids=ids)
        assert torch.equal(ids, o["top_ids"])


def backward64(z, labels, dlp, dh):
    n, c = z.shape
    m, L, lp, h = forward64(z)
    p = lp.exp()
    y = labels.long()
    has = (y >= 0) & (y < c)
    up = torch.where(has, dlp.double(), 0.0)[:, None] if dlp is not None else torch.zeros(n, 1, device="cuda", dtype=torch.float64)
    hot = torch.zeros_like(p)
    hot.scatter_(1, y.clamp(0, c - 1)[:, None], has.double()[:, None])
    first = torch.where(hot > 0, up * (1 - p), -up * p)
    second = torch.zeros_like(p) if dh is None else -dh.double()[:, None] * p * torch.where(p > 0, lp + h, 0.0)
    # error: of p relative (its exponent's rounding and the exponential's), of lp + h absolute
    size = up.abs() * (p + hot) + (0 if dh is None else dh.double().abs()[:, None] * p * (2 + torch.where(p > 0, (lp + h).abs() + lp.abs(), 0.0)))
    return first + second, size, L


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,c", SHAPES)
def test_backward_matches_the_formula(n, c, t):
    z, labels = inputs(n, c, t, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    dlp = torch.randn(n, generator=g, device="cuda")
    dh = torch.randn(n, generator=g, device="cuda")
    o = run_forward(z, labels, 0)
    for a, b in ((dlp, None), (dlp, dh), (None, dh)):
        dz = torch.full_like(z, 7.0)
        mgg.class_logprob_backward(dz, z, labels if a is not None else None, o["stats"], a, entropy=o["entropy"] if b is not None else None, dentropy=b)
        want, size, L = backward64(z, labels, a, b)
        lp = forward64(z)[2].abs().nan_to_num(posinf=0, neginf=0)
        tol = half(t) * want.abs() + tiny(t) + (4 * sum_error(c) * (1 + math.log(c)) + 4 * U * (lp + L.abs())) * size + 2.0 ** -140
        assert ((dz.double() - want).abs() <= tol * (1 + 2.0 ** -7)).all()
        inplace = z.clone()
        mgg.class_logprob_backward(inplace, inplace, labels if a is not None else None, o["stats"], a, entropy=o["entropy"] if b is not None else None, dentropy=b)
        assert torch.equal(inplace, dz)


def test_gradient_agrees_with_differences():
    n, c = 4, 11
    z, labels = inputs(n, c, torch.float32, seed=7, masked=0.0)
    labels[:] = torch.tensor([3, 0, 10, -1], device="cuda")
    dlp, dh = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    o = run_forward(z, labels, 0)
    dz = torch.empty_like(z)
    mgg.class_logprob_backward(dz, z, labels, o["stats"], dlp, entropy=o["entropy"], dentropy=dh)

    def loss(z):
        _, _, lp, h = forward64(z)
        y = labels.long()
        return float((torch.where(y >= 0, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0) * dlp.double()).sum() + (h[:, 0] * dh.double()).sum())
    step = 1e-5
    for at in ((0, 3), (0, 4), (1, 0), (2, 5), (3, 6)):
        hi, lo = z.double().clone(), z.double().clone()
        hi[at] += step
        lo[at] -= step
        diff = (loss(hi) - loss(lo)) / (2 * step)
        assert abs(float(dz[at]) - diff) <= 1e-8 + 200 * U * (1 + float(dlp.abs().max()) + float(dh.abs().max()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("c", [1, 2, 31, 47, 64, 200, 1500, 40_000])
def test_masked_rows_and_bad_values(c, t):
    """Rows with nothing left, masks of the type's lowest value, one class left, NaN and infinities, ties, signed zeros."""
    lowest = torch.finfo(t).min
    z = torch.zeros(9, c, device="cuda").to(t)
    z[0] = -math.inf                       # nothing left
    z[1] = lowest                          # masked by the lowest value as a whole: uniform
    z[2] = lowest
    z[2, c // 2] = 3.0                     # one class left
    z[3] = -math.inf
    z[3, c - 1] = torch.finfo(t).max       # one class left, the largest value
    z[4, c // 3] = math.nan
    z[5, c // 2] = math.inf
    z[6] = 0.0                             # all equal
    z[7] = 0.0
    z[7, ::2] = -0.0                       # equal too
    z[8] = math.nan
    labels = torch.tensor([0, 0, c // 2, c - 1, 0, 0, c - 1, 0, -1], device="cuda", dtype=torch.int32)
    k = min(c, 8)
    o = run_forward(z, labels, k)
    ok = [0, 1, 2, 3, 6, 7]
    check_forward({key: v[ok].contiguous() for key, v in o.items()}, z[ok], labels[ok])
    assert torch.equal(o["top_ids"][ok + [4, 8]], best(z, k)[ok + [4, 8]])
    assert o["logprob"][0] == -math.inf and o["entropy"][0] == 0 and (o["top_logprobs"][0] == -math.inf).all()
    for r in (4, 5):
        assert o["logprob"][r].isnan() and o["entropy"][r].isnan() and o["top_logprobs"][r].isnan().all()
    assert o["top_ids"][5, 0] == c // 2 and o["logprob"][8] == 0 and o["entropy"][8].isnan()
    dz = torch.full_like(z, 7.0)
    mgg.class_logprob_backward(dz, z, labels, o["stats"], torch.ones(9, device="cuda"), entropy=o["entropy"], dentropy=torch.ones(9, device="cuda"))
    assert (dz[0] == 0).all() and dz[ok].isfinite().all() and dz[4].isnan().all() and dz[5].isnan().all()
    want, _, _ = backward64(z[ok[1:]], labels[ok[1:]], torch.ones(5, device="cuda"), torch.ones(5, device="cuda"))
    assert ((dz[ok[1:]].double() - want).abs() <= half(t) * want.abs() + tiny(t) + 2.0 ** -17).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("c", [5, 47, 300, 3000, 50_000])
def test_ties_go_to_the_lowest_class(c, t):
    """Few distinct scores, so that every place in the ranking is tied, also across warps and blocks."""
    g = torch.Generator(device="cuda").manual_seed(c)
    z = torch.randint(-2, 3, (50 if c < 10_000 else 3, c), generator=g, device="cuda").to(t)
    labels = torch.zeros(z.shape[0], device="cuda", dtype=torch.int32)
    for k in (1, min(c, 4), min(c, 17), min(c, 32)):
        check_forward(run_forward(z, labels, k), z, labels)
    # sorted rows, rising and falling: the ranking is replaced at every step, or never again
    z = torch.sort(z, dim=1).values.contiguous()
    check_forward(run_forward(z, labels, min(c, 8)), z, labels)
    z = z.flip(1).contiguous()
    check_forward(run_forward(z, labels, min(c, 8)), z, labels)


def test_large_scores_keep_their_probabilities():
    """Scores of 10^5 in a row: L is not lost beside the maximum."""
    z = 1e5 + torch.arange(100, device="cuda", dtype=torch.float32).repeat(3, 1) / 16
    labels = torch.tensor([0, 50, 99], device="cuda", dtype=torch.int32)
    o = run_forward(z, labels, 3)
    check_forward(o, z, labels)
    dz = torch.empty_like(z)
    mgg.class_logprob_backward(dz, z, labels, o["stats"], torch.ones(3, device="cuda"))
    want, size, _ = backward64(z, labels, torch.ones(3, device="cuda"), None)
    assert ((dz.double() - want).abs() <= 16 * sum_error(100) * size + 1e-30).all()


def test_labels_outside_the_classes_are_no_label():
    z, _ = inputs(6, 10, torch.float32)
    labels = torch.tensor([-1, -5, 10, 2 ** 31 - 1, -2 ** 31, 3], device="cuda", dtype=torch.int32)
    o = run_forward(z, labels, 0)
    assert (o["logprob"][:5] == 0).all() and o["logprob"][5] < 0
    dz = torch.full_like(z, 7.0)
    # an unlabelled row's upstream gradient takes no part, whatever it holds
    dlp = torch.tensor([math.nan, math.inf, 1.0, 1.0, 1.0, 1.0], device="cuda")
    mgg.class_logprob_backward(dz, z, labels, o["stats"], dlp)
    assert (dz[:5] == 0).all() and (dz[5] != 0).any()


@pytest.mark.parametrize("t", TYPES)
def test_rows_far_apart_and_odd_offsets(t):
    n = 37
    for c, off, wide in ((41, 1, 50), (47, 0, 48), (172, 3, 177), (1000, 8, 1016), (5000, 1, 5003), (40_000, 5, 40_007)):
        big = torch.full((n, wide), 60.0, device="cuda").to(t)               # what lies beside the rows would win
        z, labels = inputs(n, c, t, seed=c)
        big[:, off:off + c] = z
        view = big[:, off:off + c]
        k = min(8, c)
        o, p = run_forward(view, labels, k), run_forward(z, labels, k)
        check_forward(o, z, labels)
        assert torch.equal(o["top_ids"], p["top_ids"])
        holder = torch.full((n, wide + 2), 9.0, device="cuda", dtype=t)
        dz, dense = holder[:, 1:1 + c], torch.empty_like(z)
        dlp = torch.randn(n, device="cuda")
        mgg.class_logprob_backward(dz, view, labels, p["stats"], dlp, entropy=p["entropy"], dentropy=dlp)
        mgg.class_logprob_backward(dense, z, labels, p["stats"], dlp, entropy=p["entropy"], dentropy=dlp)
        assert torch.equal(dz, dense)
        assert (holder[:, :1] == 9).all() and (holder[:, 1 + c:] == 9).all()
        mgg.class_logprob_backward(view, view, labels, p["stats"], dlp, entropy=p["entropy"], dentropy=dlp)      # in place in a view
        assert torch.equal(view, dense) and (big[:, off + c:] == 60).all() and (big[:, :off] == 60).all()


def test_no_rows():
    z = torch.empty(0, 8, device="cuda")
    none = torch.empty(0, device="cuda")
    mgg.class_logprob_forward(none, z, torch.empty(0, device="cuda", dtype=torch.int32))
    mgg.class_logprob_backward(torch.empty_like(z), z, torch.empty(0, device="cuda", dtype=torch.int32), torch.empty(0, 2, device="cuda"), none)


@pytest.mark.parametrize("n,c", [(500, 47), (3, 60_000)])
def test_captured_and_replayed(n, c):
    z, labels = inputs(n, c, torch.bfloat16, seed=3)
    o = run_forward(z, labels, 5)
    dz, dlp = torch.empty_like(z), torch.randn(n, device="cuda")

    def step():
        mgg.class_logprob_forward(o["logprob"], z, labels, stats=o["stats"], entropy=o["entropy"], top_ids=o["top_ids"], top_logprobs=o["top_logprobs"])
        mgg.class_logprob_backward(dz, z, labels, o["stats"], dlp, entropy=o["entropy"], dentropy=dlp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        step()
    for k in range(3):
        nz, nl = inputs(n, c, torch.bfloat16, seed=20 + k)
        z.copy_(nz)
        labels.copy_(nl)
        graph.replay()
        got = [v.clone() for v in o.values()] + [dz.clone()]
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, list(o.values()) + [dz]))
        check_forward(o, z, labels)


def test_offsets_beyond_32_bits():
    n, c = 70_000, 32_768
    z = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16)
    tail, labels_tail = inputs(40, c, torch.bfloat16, seed=9)
    z[-40:] = tail
    labels = torch.zeros(n, device="cuda", dtype=torch.int32)
    labels[-40:] = labels_tail
    o = run_forward(z, labels, 4)
    check_forward({k: v[-40:].contiguous() for k, v in o.items()}, tail, labels_tail)
    assert (o["logprob"][:-40] == o["logprob"][0]).all()
    dlp = torch.ones(n, device="cuda")
    want = torch.empty_like(tail)
    mgg.class_logprob_backward(want, tail, labels_tail, o["stats"][-40:].contiguous(), dlp[-40:].contiguous())
    first = z[:1].clone()
    mgg.class_logprob_backward(first, first, labels[:1], o["stats"][:1].contiguous(), dlp[:1])
    mgg.class_logprob_backward(z, z, labels, o["stats"], dlp)
    assert torch.equal(z[-40:], want) and torch.equal(z[n // 2], first[0]) and torch.equal(z[0], first[0])


def test_no_bounded_wait_expired():
    import ctypes as C
    from mgg_osdi23_b200._lib import check, lib
    st = C.c_int(-1)
    check(lib.mggb_operator_device_status(C.byref(st), 0))
    assert st.value == 0
