"""Caches of 8 bits: what rotary_append writes, what read_pages makes of it, and paged_attention over it, against the definitions."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, Cache8, ROUNDOFF, attend, eight_bits, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu


def attend8(q, keys, values, *args):
    """(out, lse, spread, top) and, per row, the mean of the values' largest sizes under its probabilities."""
    tops = attend(q, keys, [v.abs().amax(-1, keepdim=True) for v in values], *args)[0]
    return (*attend(q, keys, values, *args), tops)


def check(out, lse, want, dtype):
    """The output is rounded once (u |o|); a score is off by some fp32 roundings of the largest, and probabilities by as much in proportion.  Times their scales they are whole
    numbers for the product with the values, each off by 2^-16 of the largest of 32 keys at most.  That largest is no more than the sum of the 32, and a value no more than
    the largest of its row, so that a result is off by 32 * 2^-16 of the mean of those at most, and in the mean over many, whose roundings have nothing to do with each other, by
    sqrt(32) * 2^-16 < 2^-13 of it.  (Up to 8 rows; with more, probabilities go in as two bf16 parts, 2^-17 of each.)"""
    ref, ref_lse, spread, top, tops = want
    off = 2.0 ** -20 * (4 + top)
    got = out.detach().cpu().double()
    assert got.shape == ref.shape and torch.isfinite(got).all()
    err = (got - ref).abs()
    bound = ROUNDOFF[dtype] * ref.abs() + (2.0 ** -16 + off) * spread + 2.0 ** -24
    assert (err <= bound + 2.0 ** -11 * tops).all(), (err / bound).max().item()
    assert err.mean() <= (bound + 2.0 ** -13 * tops).mean()
    lse = lse.cpu().double()
    empty = torch.isneginf(ref_lse)
    assert torch.equal(torch.isneginf(lse), empty)
    assert ((lse - ref_lse)[~empty].abs() <= off + 2.0 ** -22 * ref_lse[~empty].abs()).all()
    assert (got[empty] == 0).all()


def run(seed, lengths, Hq, Hkv, Sq, D, page, dtype, Dv=None, score=None, mask=None, window=None, token_major=False, bhln=True, kernel_options=None, width=None):
    dt = DTYPES[dtype]
    c = Cache8(seed, lengths, Hkv, D, page, dt, Dv=Dv, token_major=token_major, width=width)
    q = normal(np.random.default_rng(seed + 1), len(lengths), Hq, Sq, D, dtype=dt)
    given = q.cuda() if bhln else q.transpose(1, 2).contiguous().cuda()
    out, lse = fa.paged_attention(given, c.k_pages, c.v_pages, c.table, c.lengths, score, mask, window=window, bhln=bhln, return_lse=True,
                                  kernel_options=kernel_options, **c.scales)
    assert out.dtype == dt
    check(out if bhln else out.transpose(1, 2), lse, attend8(q, c.keys, c.values, score, mask, window), dt)
    torch.cuda.synchronize()
    fa.check_status()


LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1023]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [1, 8, 12, 16, 64, 128])
def test_lengths_and_pages(dtype, D, page):
    run(1, LENGTHS, 4, 2, 1, D, page, dtype)


@pytest.mark.parametrize("page,D,Dv", [(16, 16, 16), (6, 32, 16), (16, 48, 48), (6, 80, 80), (16, 96, 96), (6, 112, 64), (16, 128, 64), (16, 192, 128), (6, 256, 256), (16, 256, 16)])
def test_head_dims(page, D, Dv):
    run(2, [1, 40, 333], 4, 4, 2, D, page, "f16", Dv=Dv)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(1, 1, 1), (8, 1, 1), (16, 1, 1), (17, 1, 1), (8, 2, 3), (4, 2, 8), (6, 2, 7), (32, 1, 2), (4, 1, 17), (3, 1, 70)])
def test_rows(Hq, Hkv, Sq, D):
    """Rows of one to three groups of eight, and of several tiles; requests shorter than their new tokens."""
    for page in (16, 5):
        run(3, [0, 1, Sq, Sq + 1, 200], Hq, Hkv, Sq, D, page, "bf16")


@pytest.mark.parametrize("token_major,bhln", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_layouts(token_major, bhln, D):
    run(4, [5, 77, 300], 8, 2, 2, D, 16, "bf16", token_major=token_major, bhln=bhln)


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("width", [None, 4000])
@pytest.mark.parametrize("D", [64, 128])
def test_kernels(general, width, D):
    """Loads by TMA and in pieces, segments of a CTA each and cut ones."""
    run(5, [1, 100, 700, 2500], 8, 2, 1, D, 16, "bf16", kernel_options={"kernels": "general"} if general else None, width=width)


def softcap(score, b, h, q_idx, kv_idx):
    return 5.0 * torch.tanh(score / 5.0)


def distance(score, b, h, q_idx, kv_idx):
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


def nothing(b, h, q_idx, kv_idx):
    return (kv_idx < 0) & (q_idx < 0)


def parity(b, h, q_idx, kv_idx):
    return (q_idx + kv_idx + h) % 2 == 0


@pytest.mark.parametrize("score,mask,window", [(None, parity, None), (None, nothing, None), (None, None, 0), (softcap, None, 33), (distance, None, 100), (distance, None, 33)])
def test_mods_and_windows(score, mask, window):
    run(6, [0, 1, 70, 400], 4, 2, 3, 64, 16, "f16", score=score, mask=mask, window=window)
    run(6, [0, 1, 70, 400], 4, 2, 3, 96, 10, "bf16", score=score, mask=mask, window=window)


@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** 12, 2.0 ** 60])
def test_values_of_any_size(factor):
    """Scales of values multiply probabilities, which have to keep their bits then."""
    c = Cache8(7, [1, 50, 300], 2, 64, 16, torch.bfloat16)
    q = normal(np.random.default_rng(8), 3, 4, 1, 64, dtype=torch.bfloat16)
    scales = dict(key_scales=c.k_scales, value_scales=c.v_scales * factor)
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, **scales)
    ref, ref_lse, spread, top, tops = attend8(q, c.keys, [v * factor for v in c.values])
    assert ((out.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -16 + 2.0 ** -20 * (4 + top)) * spread + 2.0 ** -11 * tops).all()


def test_a_scale_that_is_no_number_stays_in_its_request():
    c = Cache8(9, [40, 50], 2, 128, 16, torch.float16)
    c.v_scales[c.table[1, 0].item(), 0, 3] = math.nan
    q = normal(np.random.default_rng(10), 2, 2, 1, 128, dtype=torch.float16)
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, **c.scales)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1, 0]).all() and torch.isfinite(out[1, 1]).all()
    check(out[:1], lse[:1], tuple(x if i == 3 else x[:1] for i, x in enumerate(attend8(q, c.keys, c.values))), torch.float16)


# ---- writing ------------------------------------------------------------------------------------
def empty_pages(n, Hkv, page, D, Dv, token_major=False):
    def one(*size):
        return torch.zeros(*size)

    def laid(t, dtype):
        t = t.to(dtype).cuda()
        return t.transpose(1, 2).contiguous().transpose(1, 2) if token_major else t

    return [laid(one(n, Hkv, page, D) + 77, torch.int8), laid(one(n, Hkv, page, Dv) + 77, torch.int8), laid(one(n, Hkv, page) - 5, torch.float32),
            laid(one(n, Hkv, page) - 5, torch.float32)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,Dv,R,interleaved", [(64, 64, 64, False), (128, 128, 128, False), (128, 64, 64, True), (80, 80, 20, False), (80, 48, 22, True), (256, 256, 256, False),
                                                (20, 12, 6, False), (37, 5, 0, False), (128, 128, 0, False), (24, 24, 24, False)])
@pytest.mark.parametrize("norm,token_major", [(False, False), (True, True)])
def test_what_is_written(dtype, D, Dv, R, interleaved, norm, token_major):
    dt = DTYPES[dtype]
    rng = np.random.default_rng(11)
    T, Hq, Hkv, page, n = 45, 4, 3, 5, 12
    q, k, v = (normal(rng, 1, T, h, d, dtype=dt) for h, d in ((Hq, D), (Hkv, D), (Hkv, Dv)))
    v[0, 3, 1] = 0
    v[0, 4, 1] = 1e-7 if dt == torch.float16 else 1e-43
    slots = torch.from_numpy(rng.permutation(n * page)[:T].copy())
    slots[7] = -1
    weights = [(1 + 0.1 * normal(rng, D)).to(dt).cuda() for _ in range(2)] if norm else [None, None]
    table = fa.rotary_table(100, R, device="cuda") if R else None
    pos = torch.from_numpy(rng.integers(0, 100, (1, T)))
    kp, vp, ks, vs = empty_pages(n, Hkv, page, D, Dv, token_major)
    got_q = fa.rotary_append(q.cuda(), k.cuda(), v.cuda(), kp, vp, slots.cuda(), table, pos.cuda() if R else None, query_weight=weights[0], key_weight=weights[1],
                             interleaved=interleaved, bhln=False, key_scales=ks, value_scales=vs)
    # queries are those of a cache of the tensors' type, and what its keys are in 32 bits, to some roundings, goes into 8
    kp2, vp2 = torch.zeros(n, Hkv, page, D, dtype=dt, device="cuda"), torch.zeros(n, Hkv, page, Dv, dtype=dt, device="cuda")
    args = (slots.cuda(), table, pos.cuda() if R else None)
    same_q = fa.rotary_append(q.cuda(), k.cuda(), v.cuda(), kp2, vp2, *args, query_weight=weights[0], key_weight=weights[1], interleaved=interleaved, bhln=False)
    assert torch.equal(got_q, same_q)
    kp, vp, ks, vs = (t.cpu() for t in (kp, vp, ks, vs))
    y = k.double()
    if norm:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * weights[1].cpu().double()
    if R:
        t = table.cpu().double()[pos]
        c, s = t[..., : R // 2].unsqueeze(-2), t[..., R // 2:].unsqueeze(-2)
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., : R // 2], y[..., R // 2: R])
        p, r = a * c - b * s, b * c + a * s
        y = torch.cat([torch.stack([p, r], -1).flatten(-2) if interleaved else torch.cat([p, r], -1), y[..., R:]], -1)
    whole, scale = eight_bits(v[0])
    exact_k = eight_bits(k[0]) if not norm and not R else None
    written = torch.zeros(n * page, dtype=torch.bool)
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        written[slot] = True
        pg, at = slot // page, slot % page
        assert torch.equal(vp[pg, :, at], whole[i]) and torch.equal(vs[pg, :, at], scale[i])
        if exact_k:
            assert torch.equal(kp[pg, :, at], exact_k[0][i]) and torch.equal(ks[pg, :, at], exact_k[1][i])
        # a scale is off by the roundings of the largest value and its division, a value by half a step and those
        top = y[0, i].abs().amax(-1)
        assert ((ks[pg, :, at].double() * 127 - top).abs() <= 2.0 ** -20 * top).all()
        off = (kp[pg, :, at].double() * ks[pg, :, at].double()[:, None] - y[0, i]).abs()
        assert (off <= (0.5 / 127 + 2.0 ** -19) * top[:, None]).all()
    rest = ~written.view(n, page)
    assert (kp.transpose(1, 2)[rest] == 77).all() and (vp.transpose(1, 2)[rest] == 77).all() and (ks.transpose(1, 2)[rest] == -5).all() and (vs.transpose(1, 2)[rest] == -5).all()
    torch.cuda.synchronize()
    fa.check_status()


@pytest.mark.parametrize("D", [64, 20])
def test_rounding_is_that_of_the_quotient(D):
    """Values that lie on and next to ties: rows whose largest is 127 steps, of halves of steps and their neighbours in fp16."""
    page, Hkv = 16, 2
    rng = np.random.default_rng(12)
    v = torch.from_numpy(rng.integers(-254, 255, (1, 64, Hkv, D)) / 2).to(torch.float16)
    v += torch.from_numpy(rng.integers(-1, 2, v.shape)).half() * torch.finfo(torch.float16).eps * v.abs()
    v[..., 0] = 127 * torch.from_numpy(rng.choice([1, 1, 3, 0.7], v.shape[:-1])).half()
    kp, vp, ks, vs = empty_pages(4, Hkv, page, D, D)
    fa.rotary_append(None, v.cuda(), v.cuda(), kp, vp, torch.arange(64, device="cuda"), bhln=False, key_scales=ks, value_scales=vs)
    whole, scale = eight_bits(v[0])
    for p, s in ((kp, ks), (vp, vs)):
        assert torch.equal(p.cpu().transpose(1, 2).reshape(64, Hkv, D), whole)
        assert torch.equal(s.cpu().transpose(1, 2).reshape(64, Hkv), scale)


@pytest.mark.parametrize("D", [64, 20])
def test_rows_with_no_number(D):
    v = torch.ones(1, 3, 1, D, dtype=torch.bfloat16)
    v[0, 0, 0, 5], v[0, 1, 0, 7] = math.inf, math.nan
    kp, vp, ks, vs = empty_pages(1, 1, 4, D, D)
    fa.rotary_append(None, v.cuda(), v.cuda(), kp, vp, torch.arange(3, device="cuda"), bhln=False, key_scales=ks, value_scales=vs)
    assert torch.isnan(ks[0, 0, :2]).all() and torch.isnan(vs[0, 0, :2]).all() and torch.isfinite(ks[0, 0, 2])
    key, value = fa.read_pages(kp, vp, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), 3,
                               key_scales=ks, value_scales=vs, dtype=torch.float32)
    for t in (key, value):
        assert torch.isnan(t[0, 0, :2]).all() and (t[0, 0, 2] == 1).all()


# ---- reading back -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (80, 48), (20, 7), (256, 8)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("page,token_major,bhln", [(16, False, False), (5, True, True), (1, False, True)])
def test_read(dtype, D, Dv, eight, page, token_major, bhln):
    dt = DTYPES[dtype]
    lengths = [0, 5, 1, 0, 0, 70, 16, 33, 0]
    c = (Cache8 if eight else Cache)(13, lengths, 3, D, page, dt, Dv=Dv, token_major=token_major)
    starts = torch.tensor([0] + lengths).cumsum(0).int() + 3
    n = int(starts[-1]) + 4
    key, value = fa.read_pages(c.k_pages, c.v_pages, c.table, starts.cuda(), n, dtype=dt if eight else None, bhln=bhln, **(c.scales if eight else {}))
    for got, want in ((key, c.keys), (value, c.values)):
        assert got.dtype == dt
        got = (got if bhln else got.transpose(1, 2)).cpu()[0]
        assert (got[:, :3] == 0).all() and (got[:, n - 4:] == 0).all()
        want = torch.cat(want, 1)
        # (8 bits: the product of a whole number and a scale, in fp32 and then in the type)
        assert torch.equal(got[:, 3: n - 4], want.float().to(dt) if eight else want)
    torch.cuda.synchronize()
    fa.check_status()


def test_read_many_requests():
    """More requests than threads look at at once, most of them of no tokens."""
    lengths = [b % 3 if b % 5 == 0 else 0 for b in range(1500)]
    c = Cache(14, lengths, 1, 16, 4, torch.float16)
    starts = torch.tensor([0] + lengths).cumsum(0).int()
    key, value = fa.read_pages(c.k_pages, c.v_pages, c.table, starts.cuda(), int(starts[-1]))
    assert torch.equal(key[0].cpu(), torch.cat(c.keys, 1)) and torch.equal(value[0].cpu(), torch.cat(c.values, 1))


def test_read_of_pages_that_are_none():
    c = Cache(15, [40, 20], 1, 16, 8, torch.float16)
    c.table[0, 1], c.table[1, 0] = -1, 1 << 29
    starts = torch.tensor([0, 40, 70], dtype=torch.int32, device="cuda")  # (the second has no room for 30)
    key, _ = fa.read_pages(c.k_pages, c.v_pages, c.table[:, :5], starts, 70)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError):
        fa.check_status()
    key = key[0].cpu()
    assert torch.equal(key[:, :8], c.keys[0][:, :8]) and (key[:, 8:16] == 0).all() and torch.equal(key[:, 16:40], c.keys[0][:, 16:])
    assert (key[:, 40:48] == 0).all() and torch.equal(key[:, 48:60], c.keys[1][:, 8:])


def test_refusals():
    c = Cache8(16, [20, 30], 2, 64, 16, torch.float16)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.float16, device="cuda")
    call = lambda q=q, **kw: fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, **{**c.scales, **kw})  # noqa: E731
    call()
    with pytest.raises(ValueError, match="both or none"):
        call(key_scales=None)
    with pytest.raises(ValueError, match="dtype of the others"):
        call(key_scales=None, value_scales=None)
    with pytest.raises(NotImplementedError, match="8 bits"):
        call(q=q.float())
    with pytest.raises(ValueError, match="key_scales"):
        call(key_scales=c.k_scales[:, :1])
    with pytest.raises(ValueError, match="value_scales"):
        call(value_scales=c.v_scales.half())
    with pytest.raises(ValueError, match="with scales"):
        fa.paged_attention(q, c.k_pages.half(), c.v_pages.half(), c.table, c.lengths, **c.scales)
    starts = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    read = lambda starts=starts, n=50, **kw: fa.read_pages(c.k_pages, c.v_pages, c.table, starts, n, **{**c.scales, "dtype": torch.float16, **kw})  # noqa: E731
    read()
    with pytest.raises(ValueError, match="need the dtype"):
        read(dtype=None)
    with pytest.raises(TypeError, match="torch.dtype"):
        read(dtype="f16")
    with pytest.raises(ValueError, match="unsupported"):
        read(dtype=torch.float64)
    with pytest.raises(ValueError, match="starts"):
        read(starts=starts.long())
    with pytest.raises(ValueError, match="block_table"):
        read(starts=starts[:2])
    with pytest.raises(ValueError, match="num_tokens"):
        read(n=-1)
    new = torch.zeros(1, 3, 2, 64, dtype=torch.float16, device="cuda")
    slots = torch.arange(3, device="cuda")
    append = lambda x=new, **kw: fa.rotary_append(None, x, x, c.k_pages, c.v_pages, slots, bhln=False, **{**c.scales, **kw})  # noqa: E731
    append()
    with pytest.raises(NotImplementedError, match="8 bits"):
        append(new.float())
    with pytest.raises(ValueError, match="both or none"):
        append(value_scales=None)
    with pytest.raises(ValueError, match="expanded"):
        append(key_scales=c.k_scales[..., :1].expand_as(c.k_scales))
    with pytest.raises(ValueError, match="no gradient"):
        append(key_scales=c.k_scales.clone().requires_grad_())


def test_one_large_scale_leaves_the_others_their_bits():
    """A value of one key that is 2^20 times the others', with a probability of next to nothing: its tile's results are as exact as its share allows."""
    c = Cache8(17, [33, 64], 1, 64, 16, torch.float16)
    q = normal(np.random.default_rng(18), 2, 1, 1, 64, dtype=torch.float16)
    scales = c.v_scales.clone()
    scales[c.table[1, 1].item(), 0, 4] *= 2.0 ** 20
    values = [c.values[0], c.values[1].clone()]
    values[1][0, 20] *= 2.0 ** 20

    def far(score, b, h, q_idx, kv_idx):
        return torch.where(kv_idx == 20, score - 60.0, score)

    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, far, return_lse=True, key_scales=c.k_scales, value_scales=scales)
    check(out, lse, attend8(q, c.keys, values, far), torch.float16)


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1.0, 1e4])
def test_queries_of_any_size(size):
    """Rows of queries in which values differ by much: the largest decides what the others keep."""
    c = Cache8(19, [50, 300], 2, 128, 16, torch.bfloat16)
    q = normal(np.random.default_rng(20), 2, 8, 1, 128) * size
    q[:, 0, :, ::3] *= 1e-4
    q[:, 1] *= torch.logspace(-6, 0, 128)
    q = q.to(torch.bfloat16)
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, sm_scale=0.1 / size, **c.scales)
    check(out, lse, attend8(q, c.keys, c.values, None, None, None, 0.1 / size), torch.bfloat16)


def test_no_numbers_in_queries_and_scales():
    c = Cache8(21, [70, 40], 2, 64, 16, torch.float16)
    q = normal(np.random.default_rng(22), 2, 4, 1, 64, dtype=torch.float16)
    q[0, 1, 0, 5], q[1, 2, 0, 9] = math.inf, math.nan
    out = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, **c.scales)
    gone = torch.zeros(2, 4, dtype=torch.bool)
    gone[0, 1] = gone[1, 2] = True
    assert torch.equal(torch.isnan(out[:, :, 0]).all(-1).cpu(), gone) and torch.isfinite(out.cpu()[:, :, 0][~gone]).all()
    c.k_scales[c.table[0, 1].item(), 1, 3] = math.nan
    out = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, **c.scales)
    gone[0, 2:] = True
    assert torch.equal(torch.isnan(out[:, :, 0]).all(-1).cpu(), gone)


def test_scales_below_zero():
    """What a cache made elsewhere may have."""
    c = Cache8(23, [40, 90], 2, 64, 16, torch.float16)
    q = normal(np.random.default_rng(24), 2, 4, 1, 64, dtype=torch.float16)
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True, key_scales=c.k_scales, value_scales=-c.v_scales)
    check(out, lse, attend8(q, c.keys, [-v for v in c.values]), torch.float16)
