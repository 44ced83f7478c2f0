"""Grouped products with sums of many thousand terms: 16-bit results carry their one rounding, not the cuts of a long sum."""
import math

import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

# A sum leaves the tensor core after 2048 terms, 128 instructions of 16 terms.  An instruction adds 16 products to the
# accumulator, and each of these 17 numbers is cut towards zero 25 places below the largest: at most 17 * 2^-25 of it, half
# of that on the average (measured: 2.0e-7 of the accumulator, 17 * 2^-26 is 2.5e-7).  With terms of one sign the accumulator
# grows evenly, so that the cuts of n instructions come to (n + 1) / 2 of one at its end.  What is added outside is
# rounded to nearest, 2^-24 at most for each of up to 32 additions.
SEGMENT = 2048
CUT, ADDS = 17 * 2.0 ** -25, 32 * 2.0 ** -24


def cuts(k):
    return (min(SEGMENT, k + 15) / 16 + 1) / 2 * CUT


def positive(sizes, k, m, t, seed=0):
    """All terms are positive, so that the accumulator grows with every instruction and every cut goes the same way; 65,536 of
    them stay below fp16's largest value."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: 0.5 + 0.5 * torch.rand(*s, generator=g, device="cuda")
    x, w = r(sum(sizes), k).to(t), r(len(sizes), k, m).to(t)
    return x, w, torch.tensor([0] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)


def products(sizes, k, m, t, backward):
    x, w, ptr = positive(sizes, k, m, t)
    out = torch.empty(sum(sizes), m, device="cuda", dtype=t)
    if backward:                       # dx = dy w^T: the same sums with the weight the other way round
        wt = w.transpose(1, 2).contiguous()
        mgg.grouped_dense_backward(out, None, x, out.new_empty(sum(sizes), m), wt, ptr)
    else:
        mgg.grouped_dense_forward(out, x, w, ptr)
    want = torch.cat([a.double() @ b.double() for a, b in zip(x.split(sizes), w)])
    return out.double(), want


# one segment and the first term behind it, several, rows that no tensor map takes, the longest sum
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,k,m", [([40, 3], 2048, 24), ([300, 0, 70], 2056, 136), ([33], 2049, 41), ([260, 1], 8191, 64), ([17, 600], 12_288, 100),
                                       ([200, 5], 65_536, 40)])
def test_every_result_is_within_its_rounding(sizes, k, m, t, backward):
    got, want = products(sizes, k, m, t, backward)
    step = torch.exp2(torch.floor(torch.log2(want))) * torch.finfo(t).eps
    assert ((got - want).abs() <= step / 2 * (1 + 2.0 ** -7) + (cuts(k) + ADDS) * want).all()


@pytest.mark.parametrize("backward", [False, True])
def test_long_sums_are_not_cut_short(backward):
    """The mean of the relative errors of 65,536-term fp16 sums.  Rounding to fp16 has no direction: uniform within half a
    step (2^-11 of the value at most), the mean of 60,000 of them is within 5 * 2^-11 / sqrt(3 * 60,000) of 0.  The cuts have
    one, half of their most on the average.  Without an end to the segments they took 4.1e-4 off every sum."""
    sizes, k, m = [400, 200], 65_536, 100
    got, want = products(sizes, k, m, torch.float16, backward)
    assert abs(float(((got - want) / want).mean())) <= cuts(k) / 2 + 5 * 2.0 ** -11 / math.sqrt(3 * got.numel())


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
def test_whole_numbers_are_exact_and_the_calls_beside_them_undisturbed(t):
    """Entries of 0 and 1 with at most 200 of them in a row: exact in 16 bits, over every segment; rows of no group are left."""
    sizes, k, m = [130, 0, 300], 20_000, 72
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 2 + sum(sizes) + 3
    x = torch.zeros(n, k, device="cuda", dtype=t)
    x.scatter_(1, torch.randint(0, k, (n, 200), generator=g, device="cuda"), 1.0)
    w = torch.randint(0, 2, (3, k, m), generator=g, device="cuda").to(t)
    ptr = torch.tensor([2] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    out = torch.full((n, m), 7.0, device="cuda", dtype=t)
    mgg.grouped_dense_forward(out, x, w, ptr)
    rows, at = out[2:-3], 2
    for s, b in zip(sizes, w):
        assert torch.equal(out[at: at + s].double(), x[at: at + s].double() @ b.double())
        at += s
    assert rows.shape[0] == sum(sizes) and (out[:2] == 7).all() and (out[-3:] == 7).all()
