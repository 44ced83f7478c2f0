"""Inputs and outputs in one matrix side by side, which share no element, are taken."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,gap", [(1, 64, 0), (300, 64, 0), (300, 41, 3), (50, 602, 1), (5, 4096, 8)])
def test_columns_side_by_side_and_rows_in_between(n, d, gap, t):
    g = torch.Generator(device="cuda").manual_seed(d)
    x, dy = torch.randn(n, d, generator=g, device="cuda").to(t), torch.randn(n, d, generator=g, device="cuda").to(t)
    mean, rstd, out, dx = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    mgg.layer_norm_forward(out, x, mean=mean, rstd=rstd)
    mgg.layer_norm_backward(dx, dy, x, mean, rstd)
    labels, lp, stats, dz = torch.zeros(n, device="cuda", dtype=torch.int32), torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda"), torch.empty_like(x)
    mgg.class_logprob_forward(lp, x, labels, stats=stats)
    mgg.class_logprob_backward(dz, x, labels, stats, lp)
    close = lambda a, b: float((a.double() - b.double()).abs().max()) <= 4 * torch.finfo(t).eps * float(b.double().abs().max())
    whole = torch.zeros(n, 3 * (d + gap), device="cuda", dtype=t)
    at = lambda i: whole[:, i * (d + gap): i * (d + gap) + d]
    for xi, yi, oi in ((0, 1, 2), (2, 1, 0), (1, 2, 0)):
        at(xi).copy_(x), at(yi).copy_(dy)
        mgg.layer_norm_forward(at(oi), at(xi))
        assert close(at(oi), out)
        mgg.layer_norm_backward(at(oi), at(yi), at(xi), mean, rstd)
        assert close(at(oi), dx)
        mgg.class_logprob_backward(at(oi), at(xi), labels, stats, lp)
        assert close(at(oi), dz) and torch.equal(at(xi), x) and torch.equal(at(yi), dy)
    # every second row
    rows = torch.zeros(2 * n, d, device="cuda", dtype=t)
    rows[::2] = x
    mgg.layer_norm_forward(rows[1::2], rows[::2])
    assert close(rows[1::2], out) and torch.equal(rows[::2], x)
    with pytest.raises(mgg.MggbError, match="partly over"):
        mgg.layer_norm_forward(rows[:n], rows[:n].flatten()[1:].new_empty(0).set_(rows.untyped_storage(), 1, (n, d), (d, 1)))
