"""read_pages says so when starts decrease, as prompt_attention does; every row is written all the same."""
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, Cache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("starts", [[0, 50, 20, 100], [100, 0, 0, 0], [0, 30, 60, 59], [5, 2 ** 31 - 1, -2 ** 31, 100]])
def test_starts_that_decrease(eight, starts):
    c = (Cache8 if eight else Cache)(1, [100, 100, 100], 2, 64, 16, torch.float16)
    kw = dict(dtype=torch.float16, **c.scales) if eight else {}
    out = fa.read_pages(c.k_pages, c.v_pages, c.table, torch.tensor(starts, dtype=torch.int32, device="cuda"), 100, **kw)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError):
        fa.check_status()
    fa.check_status()  # (said once)
    assert all(torch.isfinite(x).all() for x in out)


def test_of_many_requests():
    """One of 1500, behind what a block of threads looks at at once."""
    lengths = [b % 2 for b in range(1500)]
    c = Cache(2, lengths, 1, 16, 4, torch.float16)
    starts = torch.tensor([0] + lengths).cumsum(0).int().cuda()
    fa.read_pages(c.k_pages, c.v_pages, c.table, starts, 750)
    torch.cuda.synchronize()
    fa.check_status()
    starts[1400] += 2
    fa.read_pages(c.k_pages, c.v_pages, c.table, starts, 750)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="0x2[04]"):
        fa.check_status()


def test_a_window_of_the_rows():
    """Starts in front of the first row and beyond the last are no error: rows are what the formula says."""
    c = Cache(3, [40, 70], 2, 64, 16, torch.bfloat16)
    starts = torch.tensor([-30, 10, 80], dtype=torch.int32, device="cuda")
    k, v = fa.read_pages(c.k_pages, c.v_pages, c.table, starts, 50)
    torch.cuda.synchronize()
    fa.check_status()
    for got, want in ((k, c.keys), (v, c.values)):
        assert torch.equal(got[0].cpu(), torch.cat([want[0][:, 30:], want[1][:, :40]], 1))
