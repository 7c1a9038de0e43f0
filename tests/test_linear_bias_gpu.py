"""Biases that are linear over the keys, in prompts and behind a prefix, to half of what the other tests of them allow."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, Prompts, attend, check_attention, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu


def distance(score, b, h, q_idx, kv_idx):
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


def bound(want, tcgen05):
    """The tcgen05 kernels take the bias of a key from that of the middle of its tile, which the sums of up to 64 slopes are added to: three roundings of 64 slopes at most, 3 * 2^-24 * 64
    times the steepest, 2^-0.5, written as 2^-20 of a larger `top`.  The general kernel works it out key by key."""
    return (*want[:3], want[3] + (3 * 2.0 ** -24 * 64 * 2.0 ** -0.5 / 2.0 ** -20 if tcgen05 else 0.0))


@pytest.mark.parametrize("kernels,D,dtype", [(None, 64, "f16"), (None, 128, "bf16"), (None, 80, "f16"), ("general", 64, "f16"), (None, 256, "bf16"), (None, 64, "f32")])
@pytest.mark.parametrize("window", [None, 0, 40])
def test_prompts(kernels, D, dtype, window):
    p = Prompts(1, [1, 3, 129, 700, 1500], 4, 2, D, DTYPES[dtype], past=[700, 0, 30, 200, 1])
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, distance, key_starts=p.key_starts, window=window, return_lse=True, kernel_options={"kernels": kernels} if kernels else None)
    p.check(out, lse, bound(p.want(distance, None, window), kernels is None and D <= 128 and dtype != "f32"))


@pytest.mark.parametrize("kernels,D", [(None, 64), (None, 128), ("general", 128)])
def test_prefix(kernels, D):
    lengths = [1, 90, 33] + [5] * 20
    c = Cache(2, lengths, 2, D, 16, torch.float16)
    rng = np.random.default_rng(3)
    q, k, v = (normal(rng, *s, D, dtype=torch.float16) for s in ((23, 4, 1), (1, 2, 1300), (1, 2, 1300)))
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, distance, return_lse=True, prefix=(k.cuda(), v.cuda()),
                                  kernel_options={"kernels": kernels} if kernels else None)
    check_attention(out, lse, bound(attend(q, [torch.cat([k[0], x], 1) for x in c.keys], [torch.cat([v[0], x], 1) for x in c.values], distance), kernels is None), torch.float16)
