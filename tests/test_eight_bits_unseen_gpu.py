"""Caches of 8 bits: a value scale that is no number or infinite belongs to the rows that see its token, and to no others."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache8, normal

pytestmark = pytest.mark.gpu


def both(Hq, Hkv, Sq, D, sees, at, value, score=None, mask=None, window=None, kernels=None, prefix=0, page=16):
    """Requests whose token `at` (from the end, all heads) has `value` for the scale of its value, against the same with a finite one: rows that do not see it are the same to the bit, rows that
    do are no numbers."""
    lengths = [7, 40, 200, 65]
    c = Cache8(1, lengths, Hkv, D, page, torch.bfloat16)
    rng = np.random.default_rng(2)
    q = normal(rng, len(lengths), Hq, Sq, D, dtype=torch.bfloat16).cuda()
    pre = [normal(rng, 1, Hkv, prefix, D, dtype=torch.bfloat16).cuda() for _ in range(2)] if prefix else None
    outs = []
    for x in (1.0, value):
        scales = c.v_scales.clone()
        for b, n in enumerate(lengths):
            scales[c.table[b, (n - at) // page].item(), :, (n - at) % page] = x
        outs.append(fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, score, mask, window=window, return_lse=True, key_scales=c.k_scales, value_scales=scales,
                                       kernel_options={"kernels": kernels} if kernels else None, prefix=pre))
    (want, want_lse), (got, lse) = outs
    assert torch.equal(lse, want_lse) and torch.isfinite(want).all()
    n = torch.tensor(lengths)
    i, j = prefix + (n[:, None] - Sq + torch.arange(Sq)), prefix + (n - at)[:, None]
    seen = sees(i, j).cuda()[:, None].expand(-1, Hq, -1)
    assert seen.any() and not seen.all()
    assert torch.equal(got[~seen], want[~seen])
    assert torch.isnan(got[seen]).all() if math.isnan(value) else not torch.isfinite(got[seen]).any()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("Hq,Hkv,Sq,D", [(4, 2, 2, 64), (8, 2, 2, 128), (4, 2, 3, 256), (12, 2, 2, 128), (10, 2, 4, 80), (8, 2, 5, 64), (20, 2, 3, 128), (8, 2, 4, 256)])
def test_the_newest_of_several_tokens(Hq, Hkv, Sq, D, kernels, value):
    """Of 4 to 30 rows per kv head: one to three groups of eight, several row tiles."""
    both(Hq, Hkv, Sq, D, lambda i, j: i >= j, 1, value, kernels=kernels)


@pytest.mark.parametrize("Hq", [2, 8])
def test_out_of_the_window(Hq):
    """The oldest token that the first of three queries sees."""
    both(Hq, 2, 3, 64, lambda i, j: (i >= j) & (i - j <= 3), 6, math.nan, window=3, page=8)


@pytest.mark.parametrize("Hq", [2, 8])
@pytest.mark.parametrize("prefix", [0, 150])
def test_taken_out_by_mods(Hq, prefix):
    both(Hq, 2, 2, 128, lambda i, j: (i >= j) & ((i + j) % 2 == 0), 3, math.nan, mask=lambda b, h, q_idx, kv_idx: (q_idx + kv_idx) % 2 == 0, prefix=prefix)
    lowest = lambda s, b, h, q_idx, kv_idx: torch.where((q_idx + kv_idx) % 2 == 0, s, -3.4028234663852886e38)  # noqa: E731
    both(Hq, 2, 2, 128, lambda i, j: (i >= j) & ((i + j) % 2 == 0), 3, math.nan, score=lowest, prefix=prefix)


@pytest.mark.parametrize("Hq", [2, 8])
def test_a_probability_of_next_to_nothing_is_seen(Hq):
    far = lambda s, b, h, q_idx, kv_idx: torch.where(q_idx - kv_idx == 1, s - 300.0, s)  # noqa: E731
    both(Hq, 2, 2, 64, lambda i, j: i >= j, 1, math.nan)
    both(Hq, 2, 3, 64, lambda i, j: i >= j, 2, math.nan, score=far)
