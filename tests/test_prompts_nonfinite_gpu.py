"""A key whose score is no number or infinite makes the rows that see it no numbers, wherever it lies in a tile, and no others; so a query does to its own row."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu

softcap = lambda s, b, h, q_idx, kv_idx: 20.0 * torch.tanh(s / 20.0)  # noqa: E731
distance = lambda s, b, h, q_idx, kv_idx: s - (q_idx - kv_idx) * 0.25  # noqa: E731
cube = lambda s, b, h, q_idx, kv_idx: s * s * s  # noqa: E731


def spoil(k, j, value):
    k = k.clone()
    k[:, :, j] = value
    return k


def check(out, lse, want, want_lse, seen):
    """seen: rows (last dimension but one of out) that see the key"""
    assert torch.isnan(out[..., seen, :]).all() and torch.isnan(lse[..., seen]).all()
    assert torch.equal(out[..., ~seen, :], want[..., ~seen, :]) and torch.equal(lse[..., ~seen], want_lse[..., ~seen])


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("value,score,window", [(math.nan, None, None), (math.inf, None, None), (math.nan, softcap, None), (math.nan, distance, 40), (math.inf, distance, None), (math.nan, cube, None),
                                                (math.inf, cube, 3)])
def test_every_place_of_a_tile(kernels, D, dtype, value, score, window):
    """Two requests, of which one has the key; beside them one so long that it is not the short prompts' kernel.  (Queries are positive, so that infinite keys have infinite scores.)"""
    rng = np.random.default_rng(1)
    lengths = [300, 200, 2000]
    n = sum(lengths)
    starts = torch.tensor([0, 300, 500, 2500], dtype=torch.int32, device="cuda")
    q = normal(rng, 1, 2, n, D, dtype=DTYPES[dtype]).abs().cuda() + 0.01
    k, v = (normal(rng, 1, 1, n, D, dtype=DTYPES[dtype]).cuda() for _ in range(2))
    call = lambda k: fa.prompt_attention(q, k, v, starts, score, window=window, return_lse=True, sm_scale=0.02, kernel_options={"kernels": kernels} if kernels else None)  # noqa: E731
    want = call(k)
    assert torch.isfinite(want[0]).all()
    row = torch.arange(n, device="cuda")
    for j in [*range(300, 440), 0, 299, 499, 1777, 2499]:
        end = 300 if j < 300 else 500 if j < 500 else 2500
        check(*call(spoil(k, j, value)), *want, (row >= j) & (row < end) & (row - j <= (n if window is None else window)))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("past,tokens", [(6000, 16), (4000, 100)])
def test_parts_of_the_keys(value, past, tokens):
    """Few rows over many keys: of several CTAs that share a row one has the key."""
    rng = np.random.default_rng(2)
    starts, key_starts = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (tokens, past + tokens))
    q = normal(rng, 1, 2, tokens, 128, dtype=torch.bfloat16).abs().cuda() + 0.01
    k, v = (normal(rng, 1, 1, past + tokens, 128, dtype=torch.bfloat16).cuda() for _ in range(2))
    call = lambda k: fa.prompt_attention(q, k, v, starts, key_starts=key_starts, return_lse=True, sm_scale=0.02)  # noqa: E731
    want = call(k)
    row = torch.arange(tokens, device="cuda") + past
    for j in [*range(2048, 2048 + 130), 0, past - 1, past + tokens - 9]:
        check(*call(spoil(k, j, value)), *want, row >= j)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("B,prefix", [(40, 700), (3, 300), (3, 3000)])
def test_prefix(value, B, prefix):
    """All requests see the prefix's key, but for those that its window leaves out."""
    rng = np.random.default_rng(3)
    lengths = [(7 * b) % 60 + 1 for b in range(B)]
    c = Cache(4, lengths, 2, 128, 16, torch.float16)
    q = normal(rng, B, 8, 1, 128, dtype=torch.float16).abs().cuda() + 0.01
    k, v = (normal(rng, 1, 2, prefix, 128, dtype=torch.float16).cuda() for _ in range(2))
    call = lambda k: fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, window=window, return_lse=True, sm_scale=0.02, prefix=(k, v))  # noqa: E731
    pos = prefix + torch.tensor(lengths, device="cuda") - 1
    for window in (None, 40):
        want, want_lse = call(k)
        for j in [*range(128, 200), 0, prefix - 1, prefix - 30]:
            seen = pos - j <= (prefix + 100 if window is None else window)
            out, lse = call(spoil(k, j, value))
            assert torch.isnan(out[seen]).all() and torch.isnan(lse[seen]).all() and torch.equal(out[~seen], want[~seen]) and torch.equal(lse[~seen], want_lse[~seen])


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries(kernels, value):
    rng = np.random.default_rng(5)
    q, k, v = (normal(rng, 1, 2, 2000, 64, dtype=torch.float16).cuda() for _ in range(3))
    starts = torch.tensor([0, 2000], dtype=torch.int32, device="cuda")
    call = lambda q: fa.prompt_attention(q, k, v, starts, return_lse=True, kernel_options={"kernels": kernels} if kernels else None)  # noqa: E731
    want = call(q)
    for i in (200, 511, 1999):  # (a score of inf and one of -inf among those that it sees)
        check(*call(spoil(q, i, value)), *want, torch.arange(2000, device="cuda") == i)
