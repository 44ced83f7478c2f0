"""Infinities and NaN in the operands of grouped products: what they take part in is not finite, and nothing else."""
import math

import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

# narrow rows, row dots, weights kept in shared memory or not, 16-bit rows with and without tensor copies, narrow and wide dw
SHAPES = [(16, 16), (64, 4), (4, 64), (128, 128), (602, 132), (129, 131), (100, 47), (2048, 64), (8200, 40), (700, 3), (3, 700), (600, 8)]


def bound(t, terms):
    """As for finite operands: fp32 ones go in with at least 21 bits each; what a sum in fp32 may lose, cut or rounded."""
    return (2.0 ** -21 if t == torch.float32 else 0.0) + (terms + 2) * 2.0 ** -23


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,m", SHAPES)
def test_only_what_they_take_part_in(k, m, t):
    sizes = [70, 5, 0, 131]
    n = sum(sizes)
    g = torch.Generator(device="cuda").manual_seed(k + m)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x0, w0, dy0 = r(n, k).to(t), (r(4, k, m) / math.sqrt(k)).to(t), r(n, m).to(t)
    ptr = torch.tensor([0] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    rows = [slice(a, a + s) for a, s in zip(ptr.tolist(), sizes)]
    for which in ("x", "w", "dy"):
        x, w, dy = x0.clone(), w0.clone(), dy0.clone()
        for i, bad in enumerate((math.inf, -math.inf, math.nan, math.inf)):
            if which == "x":
                x[40 + 30 * i, (7 * i) % k] = bad
            elif which == "w":
                w[(0, 0, 3, 3)[i], (5 * i) % k, (3 * i) % m] = bad
            else:
                dy[40 + 30 * i, (7 * i) % m] = bad
        out, dx, dw = torch.empty(n, m, device="cuda", dtype=t), torch.empty(n, k, device="cuda", dtype=t), torch.empty(4, k, m, device="cuda")
        mgg.grouped_dense_forward(out, x, w, ptr)
        mgg.grouped_dense_backward(dx, dw, dy, x, w, ptr)
        X, W, D = x.double(), w.double(), dy.double()
        for i, s in enumerate(rows):
            for got, a, b in ((out[s], X[s], W[i]), (dx[s], D[s], W[i].T), (dw[i], X[s].T, D[s])):
                # in 64 bits from the definition: 0 times an infinity and sums of opposite ones are not finite either
                reached = (~a.isfinite()).double() @ torch.ones_like(b) + torch.ones_like(a) @ (~b.isfinite()).double() > 0
                assert torch.equal(~got.isfinite(), reached)
                clean = lambda v: torch.where(v.isfinite(), v, 0.0)
                want, size = clean(a) @ clean(b), clean(a).abs() @ clean(b).abs()
                tol = (torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -7) * want.abs() + 2.0 ** -25 if got.dtype != torch.float32 else 0) + bound(t, a.shape[1]) * size
                assert ((got.double() - want).abs() <= tol)[~reached].all()


@pytest.mark.parametrize("k,m", [(16, 16), (128, 128)])
def test_a_16_bit_infinity_stays_one(k, m):
    """16-bit operands go in whole: a row with one infinity and factors without a zero is infinite, with the product's sign."""
    for t in (torch.bfloat16, torch.float16):
        x, w = torch.ones(20, k, device="cuda", dtype=t), torch.ones(1, k, m, device="cuda", dtype=t)
        w[0, :, 1::2] = -1.0
        x[3, 5], x[4, 6] = math.inf, -math.inf
        out = torch.empty(20, m, device="cuda", dtype=t)
        mgg.grouped_dense_forward(out, x, w, torch.tensor([0, 20], device="cuda", dtype=torch.int32))
        assert (out[3, ::2] == math.inf).all() and (out[3, 1::2] == -math.inf).all()
        assert (out[4, ::2] == -math.inf).all() and (out[4, 1::2] == math.inf).all()
        rest = [i for i in range(20) if i not in (3, 4)]
        assert (out[rest][:, ::2] == k).all() and (out[rest][:, 1::2] == -k).all()
