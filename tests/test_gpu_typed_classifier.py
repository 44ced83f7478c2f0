"""The operators together, as a classifier over nodes of several types uses them: grouped products, layer norm, the dense
layer and the class log probabilities, forward and backward, against 64-bit automatic differentiation."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes,din,hid,classes", [([200, 0, 57, 311], 100, 64, 47), ([3, 1], 41, 16, 5), ([1500, 700], 128, 128, 172)])
def test_one_training_step(sizes, din, hid, classes):
    g = torch.Generator(device="cuda").manual_seed(0)
    n, types = sum(sizes), len(sizes)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w1, w2 = r(n, din), r(types, din, hid) / din ** 0.5, r(hid, classes) / hid ** 0.5
    gamma, beta = 1 + 0.1 * r(hid), 0.1 * r(hid)
    ptr = torch.tensor([0] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    labels = torch.randint(0, classes, (n,), generator=g, device="cuda", dtype=torch.int32)
    labels[::3] = -1
    weight = -torch.ones(n, device="cuda") / n
    e = lambda *s: torch.empty(*s, device="cuda")

    h, hn, mean, rstd, logits, lp, stats, ent = e(n, hid), e(n, hid), e(n), e(n), e(n, classes), e(n), e(n, 2), e(n)
    mgg.grouped_dense_forward(h, x, w1, ptr)
    mgg.layer_norm_forward(hn, h, gamma, beta, mean=mean, rstd=rstd)
    mgg.dense_forward(logits, hn, w2)
    mgg.class_logprob_forward(lp, logits, labels, stats=stats, entropy=ent)
    dlogits, dhn, dh, dx, dw1, dgamma, dbeta = e(n, classes), e(n, hid), e(n, hid), e(n, din), e(types, din, hid), e(hid), e(hid)
    mgg.class_logprob_backward(dlogits, logits, labels, stats, weight, entropy=ent, dentropy=0.1 * weight)
    # the untyped layer's gradients are the grouped ones with a single type
    one = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    dw2 = e(1, hid, classes)
    mgg.grouped_dense_backward(dhn, dw2, dlogits, hn, w2[None].contiguous(), one)
    mgg.layer_norm_backward(dh, dhn, h, mean, rstd, gamma, dweight=dgamma, dbias=dbeta)
    mgg.grouped_dense_backward(dx, dw1, dh, x, w1, ptr)

    leaves = [t.double().requires_grad_() for t in (x, w1, gamma, beta, w2)]
    X, W1, G, B, W2 = leaves
    H = torch.cat([a @ b for a, b in zip(X.split(sizes), W1)])
    HN = torch.nn.functional.layer_norm(H, (hid,), G, B, 1e-5)
    LP = torch.log_softmax(HN @ W2, 1)
    y = labels.long()
    LPY = torch.where(y >= 0, LP.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    ENT = -(LP.exp() * LP).sum(1)
    ((LPY + 0.1 * ENT) * weight.double()).sum().backward()
    # Each of the eight operators in the chain adds at most about 2^-19 of its output's scale (sums of at most a few hundred
    # terms in fp32, products with 21-bit operands), and each norm or product multiplies what came before by a factor of
    # order one: 2^-14 of the largest entry leaves room for all of them and for the gain of small rows' rstd.
    for name, got, want in (("lp", lp, LPY.detach()), ("entropy", ent, ENT.detach()), ("dx", dx, X.grad), ("dw1", dw1, W1.grad),
                            ("dgamma", dgamma, G.grad), ("dbeta", dbeta, B.grad), ("dw2", dw2[0], W2.grad)):
        assert float((got.double() - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max()), name
