"""Up to 16 query rows per kv head, paged attention is no further from 64 bits than the rounding of its results is."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, attend, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("G,Sq", [(1, 1), (8, 1), (3, 3), (4, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_nothing_but_the_result_is_rounded(dtype, G, Sq, D):
    """Values of mean 0 under thousands of weights alike, where a rounding of the probabilities is as large as that of the result.  In two parts it leaves
    2^-16 (bf16) of a probability, 0.4 % of the rounding of the result, and sums in fp32 less: 2 % covers both."""
    dt = DTYPES[dtype]
    c = Cache(41, [6000], 1, D, 16, dt)
    q = normal(np.random.default_rng(42), 1, G, Sq, D, dtype=dt)
    out = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, sm_scale=0.02)
    want = attend(q, c.keys, c.values, scale=0.02)[0]
    off = lambda x: (x.double() - want).norm().item()  # noqa: E731
    assert off(out.cpu()) <= 1.02 * off(want.to(dt))
