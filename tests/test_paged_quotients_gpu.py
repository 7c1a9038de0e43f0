"""Quotients in mods under paged_attention: what decides which key is seen or which entry of a table is read is exact, as under flax_attention."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, attend, check_attention, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu

# a divisor for each of 32 query heads: quotients that are whole numbers, and ones that are not
DIVISORS = torch.tensor([1, 2, 3, 5, 6, 7, 9, 10, 11, 12, 13, 14, 15, 17, 19, 21, 22, 23, 25, 27, 29, 31, 33, 35, 37, 39, 41, 43, 45, 47, 49, 0.1])
BIAS = torch.linspace(-1.0, 1.0, 101)[torch.randperm(101, generator=torch.Generator().manual_seed(5))]


def whole(x):
    """To an int32, towards 0: of a value that is traced, or of a tensor."""
    return x.to(torch.int32) if isinstance(x, torch.Tensor) else x.astype(np.int32)


def mods(kind, dev):
    """(score_mod, mask_mod) over tensors on `dev`"""
    d, bias = DIVISORS.to(dev), BIAS.to(dev)

    def same_part(b, h, q_idx, kv_idx):
        return torch.floor(q_idx / d[h]) == torch.floor(kv_idx / d[h])

    def same_part_whole(b, h, q_idx, kv_idx):
        return whole(q_idx / d[h]) == whole(kv_idx / d[h])

    def same_part_floordiv(b, h, q_idx, kv_idx):
        return (q_idx * 1.0) // d[h] == (kv_idx * 1.0) // d[h]

    def same_remainder(b, h, q_idx, kv_idx):
        return kv_idx / d[h] - torch.floor(kv_idx / d[h]) == 0.0

    def bucket(score, b, h, q_idx, kv_idx):
        return score + bias[whole((q_idx - kv_idx) / d[h]) % 101]

    def chosen(score, b, h, q_idx, kv_idx):
        return torch.where(torch.floor(kv_idx / d[h]) % 2 == 0, score / d[h], -score)

    def by_seven(b, h, q_idx, kv_idx):
        return torch.floor(q_idx / 7.0) == torch.floor(kv_idx / 7.0)

    return {"floor": (None, same_part), "cast": (None, same_part_whole), "floordiv": (None, same_part_floordiv), "equal": (None, same_remainder),
            "table": (bucket, None), "where": (chosen, None), "constant": (None, by_seven)}[kind]


@pytest.mark.parametrize("kind", ["floor", "cast", "floordiv", "equal", "table", "where", "constant"])
@pytest.mark.parametrize("dtype,Sq", [("f16", 1), ("bf16", 5), ("f32", 1)])
def test_quotients_that_decide(kind, dtype, Sq):
    dt = DTYPES[dtype]
    lengths = [1, 48, 50, 100, 148, 206, 778]
    c = Cache(31, lengths, 8, 64, 16, dt)
    q = normal(np.random.default_rng(32), len(lengths), 32, Sq, 64, dtype=dt)
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, *mods(kind, "cuda"), return_lse=True)
    want = attend(q, c.keys, c.values, *mods(kind, "cpu"))
    torch.cuda.synchronize()
    fa.check_status()
    check_attention(out, lse, want, dt)
