"""fp32 grouped products of up to 128 terms keep the precision of longer ones."""
import pytest
import torch

import mgg_osdi23_b200 as mgg

pytestmark = pytest.mark.gpu

# Terms of one sign between 1/4 and 1.  The products of the parts' upper bf16 numbers have 16 bits and are never 2^9 times
# smaller than their sum, so the tensor core, which cuts 25 places below the largest, adds them exactly.  The five smaller
# products are at most 2^-7 of the sum together and lose 17 * 2^-25 per instruction, (5 * 8 + 1) / 2 times: 2^-19.6 of 2^-7.
# The three products that are left out are below 2 * 2^-24; the final addition rounds by 2^-24.
BOUND = (41 / 2) * 17 * 2.0 ** -25 * 2.0 ** -7 + 3 * 2.0 ** -24


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("sizes", [[50], [700, 0, 40_000, 3]])
@pytest.mark.parametrize("k,m", [(20, 128), (32, 100), (33, 128), (47, 100), (64, 128), (64, 72), (96, 130), (100, 100), (127, 72), (128, 128), (128, 300)])
def test_every_sum_is_exact_to_fp32(sizes, k, m, backward):
    g = torch.Generator(device="cuda").manual_seed(k * m)
    r = lambda *s: 0.5 + 0.5 * torch.rand(*s, generator=g, device="cuda")
    x, w = r(sum(sizes), k), r(len(sizes), k, m)
    ptr = torch.tensor([0] + sizes).cumsum(0).to(device="cuda", dtype=torch.int32)
    out = torch.empty(sum(sizes), m, device="cuda")
    if backward:
        mgg.grouped_dense_backward(out, None, x, torch.empty_like(out), w.transpose(1, 2).contiguous(), ptr)
    else:
        mgg.grouped_dense_forward(out, x, w, ptr)
    want = torch.cat([a.double() @ b.double() for a, b in zip(x.split(sizes), w)])
    assert float(((out.double() - want) / want).abs().max()) <= BOUND


@pytest.mark.parametrize("k,m", [(64, 80), (33, 128), (48, 300)])
def test_many_groups(k, m):
    """The largest number of types, most of them empty, with what their lists leave of shared memory."""
    groups, n = 4096, 9000
    g = torch.Generator().manual_seed(k)
    cuts = torch.sort(torch.randint(0, n + 1, (groups - 1,), generator=g)).values
    ptr = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), n)]).to(device="cuda", dtype=torch.int32)
    whole = lambda *s: torch.randint(-3, 4, s, device="cuda").float()
    x, w = whole(n, k), whole(groups, k, m)
    gid = torch.repeat_interleave(torch.arange(groups, device="cuda"), (ptr[1:] - ptr[:-1]).long())
    out = torch.empty(n, m, device="cuda")
    mgg.grouped_dense_forward(out, x, w, ptr)
    assert torch.equal(out, torch.bmm(x[:, None].double(), w[gid].double())[:, 0].float())
    wt = w.transpose(1, 2).contiguous()                # dx = dy w^T with sums over k
    mgg.grouped_dense_backward(out, None, x, torch.empty(n, m, device="cuda"), wt, ptr)
    assert torch.equal(out, torch.bmm(x[:, None].double(), w[gid].double())[:, 0].float())
