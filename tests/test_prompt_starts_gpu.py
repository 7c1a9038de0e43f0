"""Starts of requests in front of the first row or beyond the last are cut to the rows that there are, and reported.  (Of starts that decrease nothing is promised but the report.)"""
import math

import pytest
import torch

import flaxattention_b200 as fa
from _pages import Prompts, attend, check_attention
from _util import DTYPES

pytestmark = pytest.mark.gpu


def cut(starts, n):
    return [min(max(s, 0), n) for s in starts]


@pytest.mark.parametrize("dtype,D", [("f16", 64), ("bf16", 128), ("f16", 256), ("f32", 64)])
@pytest.mark.parametrize("requests", [1, 300])
@pytest.mark.parametrize("tokens,starts,key_starts", [(200, [-5, 60, 200], None), (200, [0, 60, 5000], None), (200, [30, 230, 231], None), (200, [-50, -20, 120, 2 ** 31 - 1], None),
                                                      (20, [0, 7, 40], [-100, 900, 5000])])
def test_starts_outside_the_rows(tokens, starts, key_starts, requests, dtype, D):
    dt = DTYPES[dtype]
    p = Prompts(1, [tokens], 4, 2, D, dt, past=None if key_starts is None else [1500 - tokens])
    # (300: so many in front, of no tokens, that requests are found in the other way)
    given, given_keys = ([s[0]] * (requests - 1) + s for s in (starts, key_starts or starts))
    on = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = fa.prompt_attention(p.q, p.k, p.v, on(given), key_starts=None if key_starts is None else on(given_keys), return_lse=True)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="starts"):
        fa.check_status()
    at, keys_at = cut(starts, tokens), cut(key_starts or starts, p.k.shape[2])
    q, k, v = p.queries[0], p.keys[0], p.values[0]
    rows = torch.zeros(tokens, dtype=torch.bool)
    for a, b, c, d in zip(at, at[1:], keys_at, keys_at[1:]):
        if a < b:
            rows[a:b] = True
            check_attention(out[:, :, a:b], lse[:, :, a:b], attend(q[None, :, a:b], [k[:, c:d]], [v[:, c:d]]), dt)
    out, lse = out.cpu(), lse.cpu()
    assert (out[:, :, ~rows] == 0).all() and (lse[:, :, ~rows] == -math.inf).all()
