"""Narrow grouped products on both sides of every rule that chooses a kernel for them, against 64-bit products."""
import math

import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# at, below and above the longest sums of each width, the widths where it changes, row dots of both kinds and their ends
WIDTHS = [(64, 2), (65, 2), (64, 4), (65, 4), (112, 5), (113, 5), (64, 8), (65, 8), (112, 8), (113, 8), (512, 3), (513, 3), (513, 4), (512, 5), (513, 5),
          (600, 8), (3300, 7), (1, 1), (9, 31), (24, 31), (25, 31), (40, 31), (41, 31), (80, 4), (81, 4), (16, 32), (33, 9), (48, 16), (49, 16), (64, 16), (65, 16),
          (88, 16), (89, 16), (32, 16), (33, 16), (88, 12)]
ROWS = [[1], [33, 0, 100, 257], [20_000, 3]]


def half(t):
    return torch.finfo(t).eps / 2


def bound(t, terms):
    """fp32 operands go in with at least 21 bits each; a sum of `terms` in fp32, rounded or cut."""
    return (2.0 ** -21 if t == torch.float32 else 0.0) + (terms + 2) * 2.0 ** -23


def check(got, a, b, t):
    want, size = a @ b, a.abs() @ b.abs()
    tol = (half(t) * (1 + 2.0 ** -7) * want.abs() + 2.0 ** -25 if got.dtype != torch.float32 else 0) + bound(t, a.shape[1]) * size
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sizes", ROWS)
@pytest.mark.parametrize("k,m", WIDTHS)
def test_products_match(k, m, sizes, t):
    g = torch.Generator(device="cuda").manual_seed(100 * k + m)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    n, groups = sum(sizes) + 5, len(sizes)
    x, w, dy = r(n, k).to(t), (r(groups, k, m) / math.sqrt(k)).to(t), r(n, m).to(t)
    ptr = torch.tensor([2] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    out, dx = torch.full((n, m), 7.0, device="cuda", dtype=t), torch.full((n, k), 7.0, device="cuda", dtype=t)
    dw = torch.full((groups, k, m), 7.0, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
    for i in range(groups):
        s = slice(int(ptr[i]), int(ptr[i + 1]))
        X, W, D = x[s].double(), w[i].double(), dy[s].double()
        check(out[s], X, W, t)
        check(dx[s], D, W.T, t)
        check(dw[i], X.T, D, t)
    for whole in (out, dx):
        assert (whole[:2] == 7).all() and (whole[n - 3:] == 7).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", [(65_536, 64, 64), (65_537, 64, 64), (65_536, 68, 60), (70_000, 64, 16), (70_000, 11, 132), (16_384, 16, 16),
                                   (16_385, 16, 16), (16_385, 17, 16), (70_000, 24, 19), (70_000, 602, 4)])
def test_the_weights_gradient_misses_no_row(n, k, m, t):
    """Entries of -1, 0 and 1, sparse: every sum is exact whatever kernel adds it up."""
    g = torch.Generator(device="cuda").manual_seed(7)
    few = lambda *s: (torch.randint(-1, 2, s, generator=g, device="cuda") * (torch.rand(*s, generator=g, device="cuda") < 0.2)).to(t)
    x, dy = few(n, k), few(n, m)
    cuts = [0, n // 3, n // 3, n]
    ptr = torch.tensor(cuts, device="cuda", dtype=torch.int32)
    dw = torch.empty(3, k, m, device="cuda")
    mgg.grouped_dense_backward(None, dw, dy, x, torch.empty(3, k, m, device="cuda", dtype=t), ptr)
    for i in range(3):
        assert torch.equal(dw[i].double(), x[cuts[i]: cuts[i + 1]].double().T @ dy[cuts[i]: cuts[i + 1]].double())


@pytest.mark.parametrize("m", [2, 4])
def test_row_dots_beyond_32_bits(m):
    """Rows whose element offsets pass 2^31."""
    n, k = 1_100_000, 2048
    x = torch.zeros(n, k, device="cuda", dtype=torch.bfloat16)
    tail = torch.randint(-2, 3, (300, k), device="cuda").to(torch.bfloat16)
    x[-300:] = tail
    w = torch.randint(-1, 2, (2, k, m), device="cuda").to(torch.bfloat16)
    out = torch.empty(n, m, device="cuda", dtype=torch.bfloat16)
    mgg.grouped_dense_forward(out, x, w, torch.tensor([0, n - 300, n], device="cuda", dtype=torch.int32))
    assert torch.equal(out[-300:].double(), (tail.double() @ w[1].double()).to(torch.bfloat16).double()) and (out[:-300] == 0).all()
