"""paged_attention at head dims above 128, from a few rows per kv head to several tiles of them: by TMA and in pieces, a CTA per segment and segments that are cut."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, attend, check_attention, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("D", [144, 192, 256])
@pytest.mark.parametrize("G,Sq", [(8, 1), (4, 3), (4, 5), (8, 5), (5, 14)])
def test_rows_of_wide_heads(dtype, D, G, Sq):
    dt, lengths = DTYPES[dtype], [0, 1, Sq, 45, 700]
    c = Cache(51, lengths, 2, D, 16, dt, width=50)
    q = normal(np.random.default_rng(52), len(lengths), 2 * G, Sq, D, dtype=dt)
    want = attend(q, c.keys, c.values)
    wide = torch.cat([c.table, torch.full((len(lengths), 1500), -1, dtype=torch.int32, device="cuda")], 1)
    for table, options in ((c.table, None), (wide, {"kernels": "general"} if D == 256 else None)):
        out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, table, c.lengths, return_lse=True, kernel_options=options)
        check_attention(out, lse, want, dt)
    torch.cuda.synchronize()
    fa.check_status()
