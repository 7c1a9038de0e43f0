"""paged_attention behind a prefix that all requests share, against its definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, Cache8, attend, check_attention, normal, with_slope
from _util import DTYPES

pytestmark = pytest.mark.gpu


def run(seed, P, lengths, Hq, Hkv, Sq, D, page, dtype, Dv=None, score=None, mask=None, window=None, bhln=True, eight=False, kernels=None, scale=None):
    dt = DTYPES[dtype]
    c = (Cache8 if eight else Cache)(seed, lengths, Hkv, D, page, dt, Dv=Dv)
    rng = np.random.default_rng(seed + 1)
    Dv = D if Dv is None else Dv
    q, pk, pv = normal(rng, len(lengths), Hq, Sq, D, dtype=dt), normal(rng, 1, Hkv, P, D, dtype=dt), normal(rng, 1, Hkv, P, Dv, dtype=dt)
    given = [(x if bhln else x.transpose(1, 2).contiguous()).cuda() for x in (q, pk, pv)]
    out, lse = fa.paged_attention(given[0], c.k_pages, c.v_pages, c.table, c.lengths, score, mask, window=window, bhln=bhln, return_lse=True, sm_scale=scale,
                                  prefix=(given[1], given[2]), kernel_options={"kernels": kernels} if kernels else None, **(c.scales if eight else {}))
    assert out.dtype == dt

    def behind(b, h, i, j):  # (queries in front of a request's first token see nothing)
        see = i >= P
        return see if mask is None else see & mask(b, h, i, j)

    join = lambda x, y: [torch.cat([x[0].double(), t.double()], 1) for t in y]  # noqa: E731
    want = attend(q, join(pk, c.keys), join(pv, c.values), score, behind, window, scale)
    check_attention(out if bhln else out.transpose(1, 2), lse, with_slope(want, 2.0 ** -0.5 if score is distance else 0.0), dt)
    torch.cuda.synchronize()
    fa.check_status()


@pytest.mark.parametrize("kernels,dtype", [(None, "f16"), ("general", "bf16"), (None, "bf16"), (None, "f32")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [1, 31, 127, 128, 129, 1300])
def test_lengths(kernels, dtype, D, P):
    run(1, P, [0, 1, 33, 200] + [3] * 36, 4, 2, 1, D, 16, dtype, kernels=kernels)


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("Hq,Hkv,Sq,B", [(1, 1, 1, 1), (8, 1, 1, 40), (6, 2, 3, 7), (4, 2, 8, 3), (16, 2, 2, 30), (3, 1, 70, 3), (2, 2, 1, 300)])
def test_rows(kernels, Hq, Hkv, Sq, B):
    run(2, 300, [(i * 7) % 50 for i in range(B)], Hq, Hkv, Sq, 64, 8, "bf16", kernels=kernels)


@pytest.mark.parametrize("dtype,D,eight", [("bf16", 128, False), ("f16", 64, False), ("f32", 64, False), ("bf16", 128, True), ("f16", 64, True)])
@pytest.mark.parametrize("G,Sq", [(1, 1), (3, 1), (4, 3)])
def test_pages_beside_the_prefix(dtype, D, eight, G, Sq):
    """Requests and parts of the prefix that fill the SMs together: the pages' CTAs are of a form that has room beside the others."""
    run(20, 2100, [0, 1, 31, 500] + [5 * i for i in range(1, 33)], 4 * G, 4, Sq, D, 16, dtype, eight=eight, score=softcap if G == 3 else None)


@pytest.mark.parametrize("dtype,D,Dv", [*(("f16", *x) for x in ((16, 16), (80, 80), (96, 32), (192, 128))), ("f32", 48, 48), ("f32", 256, 256)])
def test_head_dims(dtype, D, Dv):
    run(3, 200, [3, 70], 4, 2, 2, D, 16, dtype, Dv=Dv)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bhln", [True, False])
@pytest.mark.parametrize("Sq", [1, 3])
def test_eight_bits(D, bhln, Sq):
    run(4, 500, [0, 2, 100, 700], 8, 2, Sq, D, 16, "bf16", bhln=bhln, eight=True)


def softcap(score, b, h, q_idx, kv_idx):
    return 5.0 * torch.tanh(score / 5.0)


def distance(score, b, h, q_idx, kv_idx):
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


def parity(b, h, q_idx, kv_idx):
    return (q_idx + kv_idx + h + b) % 2 == 0


def nothing(b, h, q_idx, kv_idx):
    return (kv_idx < 0) & (q_idx < 0)


def not_in_front(b, h, q_idx, kv_idx):
    return (kv_idx >= 300) & (q_idx >= 0)


@pytest.mark.parametrize("dtype,D", [("f16", 64), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("score,mask", [(softcap, None), (distance, parity), (None, nothing), (None, not_in_front)])
def test_mods(dtype, score, mask, D):
    run(5, 300, [0, 1, 70, 400], 4, 2, 3, D, 16, dtype, score=score, mask=mask)


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("window", [0, 1, 50, 128, 300, 5000])
def test_windows(kernels, window):
    run(6, 333, [0, 2, 40, 200], 4, 1, 4, 64, 16, "bf16", window=window, kernels=kernels)
    run(6, 333, [0, 2, 40, 200], 4, 1, 4, 128, 16, "f16", window=window, kernels=kernels, score=distance)


@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_scales(scale):
    run(7, 140, [10, 60], 2, 2, 1, 64, 16, "f16", scale=scale)


def test_more_sums_than_one_launch_holds():
    """One request over a long prefix (many parts), cut segments of the pages."""
    run(8, 9000, [5000], 8, 2, 1, 128, 64, "bf16")


def test_no_prefix_is_none():
    c = Cache(9, [5, 70], 2, 64, 16, torch.float16)
    q = normal(np.random.default_rng(10), 2, 4, 1, 64, dtype=torch.float16).cuda()
    none = torch.zeros(1, 2, 0, 64, dtype=torch.float16, device="cuda")
    want = fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths)
    assert torch.equal(fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, prefix=(none, none)), want)


def test_what_lies_beyond_the_prefix():
    """Rows of a wider buffer behind the prefix are NaN."""
    c = Cache(11, [5, 70], 2, 128, 16, torch.bfloat16)
    rng = np.random.default_rng(12)
    q, k, v = normal(rng, 2, 4, 1, 128, dtype=torch.bfloat16), normal(rng, 1, 2, 200, 128, dtype=torch.bfloat16), normal(rng, 1, 2, 200, 128, dtype=torch.bfloat16)
    wide = [torch.full((1, 2, 300, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    wide[0][:, :, :200], wide[1][:, :, :200] = k, v
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, prefix=[w[:, :, :200] for w in wide])
    check_attention(out, lse, attend(q, [torch.cat([k[0], x], 1) for x in c.keys], [torch.cat([v[0], x], 1) for x in c.values]), torch.bfloat16)


def test_graphs_that_share_nothing():
    """Two captured calls, replayed in turn on one stream, each over its own lengths."""
    cs = [Cache(13 + i, [40, 9 + i, 300], 2, 64, 16, torch.float16) for i in range(2)]
    rng = np.random.default_rng(14)
    q = normal(rng, 3, 4, 1, 64, dtype=torch.float16)
    pre = [normal(rng, 1, 2, 250, 64, dtype=torch.float16) for _ in range(2)]
    on = [t.cuda() for t in (q, *pre)]
    call = lambda c: fa.paged_attention(on[0], c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, prefix=(on[1], on[2]))  # noqa: E731
    call(cs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for c, (out, lse) in zip(cs, outs):
        check_attention(out, lse, attend(q, [torch.cat([pre[0][0], x], 1) for x in c.keys], [torch.cat([pre[1][0], x], 1) for x in c.values]), torch.float16)


def test_refusals():
    c = Cache(15, [20, 30], 2, 64, 16, torch.float16)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.float16, device="cuda")
    p = torch.zeros(1, 2, 50, 64, dtype=torch.float16, device="cuda")
    call = lambda prefix: fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, prefix=prefix)  # noqa: E731
    call((p, p))
    with pytest.raises(TypeError, match="pair"):
        call(p)
    with pytest.raises(TypeError, match="tensor"):
        call((p, None))
    for bad in ((p[:, :1], p), (p, p[:, :, :40]), (torch.cat([p, p]), torch.cat([p, p])), (p[..., :48], p), (p.float(), p), (p, p.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call(bad)


@pytest.mark.parametrize("D,P", [(64, 300), (128, 1400)])
def test_scores_that_take_keys_out(D, P):
    """The lowest value as a score, for the whole prefix and for the requests' own keys in turn."""
    for cut in (lambda j: j < P, lambda j: j >= P, lambda j: j >= 0):
        def lowest(score, b, h, q_idx, kv_idx):
            return torch.where(cut(kv_idx), -3.4028234663852886e38, score)

        lengths = [4] * 40 + [50, 1]
        c = Cache(16, lengths, 2, D, 16, torch.bfloat16)
        rng = np.random.default_rng(17)
        q, pk, pv = normal(rng, 42, 4, 1, D, dtype=torch.bfloat16), *(normal(rng, 1, 2, P, D, dtype=torch.bfloat16) for _ in range(2))
        out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, lowest, return_lse=True, prefix=(pk.cuda(), pv.cuda()))
        keys, values = ([torch.cat([x[0], t], 1) for t in y] for x, y in ((pk, c.keys), (pv, c.values)))
        check_attention(out, lse, attend(q, keys, values, None, lambda b, h, i, j: ~cut(j) & (j >= 0)), torch.bfloat16)
