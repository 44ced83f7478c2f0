"""Layer norm's gradients in rows whose statistics are extreme."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [5, 40, 41, 100, 602, 1001, 4099])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_constant_rows_of_huge_values_have_finite_gradients(d, t):
    """mean * rstd beyond fp32's range with every value of the row at the mean: xhat is 0, dx = rstd (g - mean(g))."""
    n = 37
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.zeros(n, d, device="cuda", dtype=t)
    x[::2] = 2.0 ** 120
    x[1::4] = -2.0 ** 119
    dy, w = torch.randn(n, d, generator=g, device="cuda").to(t), torch.randn(d, generator=g, device="cuda")
    mean, rstd = x[:, 0].float().contiguous(), torch.full((n,), 316.0, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)
    gr = dy.double() * w.double()
    want = 316.0 * (gr - gr.mean(1, keepdim=True))
    # a sum of d terms, a product and a difference in fp32; then the one rounding
    size = 316.0 * (gr.abs() + gr.abs().mean(1, keepdim=True))
    tol = torch.finfo(t).eps / 2 * want.abs() + (d / 32 + 28) * 2.0 ** -24 * size
    assert dx.isfinite().all() and ((dx.double() - want).abs() <= tol * (1 + 2.0 ** -7)).all()
    assert (dw == 0).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= (n + 2) * 2.0 ** -24 * dy.double().abs().sum(0)).all()


@pytest.mark.parametrize("d", [8, 40, 1000, 20_000])
def test_sums_beyond_the_range(d):
    """A row whose values add up beyond fp32's range is NaN, one whose squared deviations do has rstd 0; their neighbours are as ever."""
    x = torch.randn(4, d, device="cuda")
    other = x.clone()
    x[1] = 2.0 ** 127                                   # from two of them on the sum is infinite
    x[2, ::2], x[2, 1::2] = 2.0 ** 100, -2.0 ** 100
    b = torch.randn(d, device="cuda")
    out, mean, rstd = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    mgg.layer_norm_forward(out, x, None, b, mean=mean, rstd=rstd)
    assert out[1].isnan().all()
    assert float(rstd[2]) == 0 and torch.equal(out[2], b)
    want = torch.empty_like(x)
    mgg.layer_norm_forward(want, other, None, b)
    assert torch.equal(out[[0, 3]], want[[0, 3]])
