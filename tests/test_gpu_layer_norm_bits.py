"""When the gradients of layer norm's weight and bias have the same bits."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(3000, 100), (999, 602), (5000, 41), (300, 4096), (40, 16_384)])
def test_the_same_bits_where_type_strides_and_alignment_agree(n, d, t):
    """Matrices at other addresses of the same alignment, whatever lies between the rows, with dx or (aligned like it) without."""
    g = torch.Generator(device="cuda").manual_seed(d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x0, dy0, w = r(n, d).to(t), r(n, d).to(t), r(d)
    mean, rstd = x0.float().mean(1), (x0.float().var(1, unbiased=False) + 1e-5).rsqrt()
    step = 16 // x0.element_size()

    def place(v, off, gap):
        ld = d + gap
        whole = torch.full((n * ld + off + step,), 3.0, device="cuda", dtype=t)
        out = whole[off: off + n * ld].view(n, ld)[:, :d]
        return out.copy_(v)
    for gap, off in ((0, 0), (0, 1), (3, 2), (step, 0)):
        want = None
        for shift in (0, step, 5 * step):
            for with_dx in (True, False) if off % step == 0 else (True,):
                x, dy = place(x0, off + shift, gap), place(dy0, off + shift, gap)
                dx = place(torch.zeros_like(x0), off + shift, gap) if with_dx else None
                dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
                mgg.layer_norm_backward(dx, dy, x, mean, rstd, w, dweight=dw, dbias=db)
                if want is None:
                    want = [dw, db]
                assert torch.equal(dw, want[0]) and torch.equal(db, want[1])
