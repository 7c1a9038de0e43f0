"""paged_attention against its definition in 64 bits: types, head layouts, page sizes that tiles do and do not divide, lengths from
none to many tiles, what leaves rows empty, what lies in places that no token holds."""
import math

import pytest
import torch

import flaxattention_b200 as fa
from _pages import Cache, attend, check_attention, normal
from _util import DTYPES

import numpy as np

pytestmark = pytest.mark.gpu


def run(seed, lengths, Hq, Hkv, Sq, D, page, dtype, Dv=None, score=None, mask=None, window=None, token_major=False, bhln=True, scale=None,
        kernel_options=None, on_gpu=None, width=None):
    dt = DTYPES[dtype]
    c = Cache(seed, lengths, Hkv, D, page, dt, Dv=Dv, token_major=token_major, width=width)
    q = normal(np.random.default_rng(seed + 1), len(lengths), Hq, Sq, D, dtype=dt)
    given = q.cuda() if bhln else q.transpose(1, 2).contiguous().cuda()
    gs, gm = (score, mask) if on_gpu is None else on_gpu
    out, lse = fa.paged_attention(given, c.k_pages, c.v_pages, c.table, c.lengths, gs, gm, window=window, sm_scale=scale, bhln=bhln,
                                  return_lse=True, kernel_options=kernel_options)
    assert out.dtype == dt and lse.dtype == torch.float32
    if not bhln:
        out = out.transpose(1, 2)
    check_attention(out, lse, attend(q, c.keys, c.values, score, mask, window, scale), dt)
    torch.cuda.synchronize()
    fa.check_status()
    return out


LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1023]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [1, 8, 12, 16, 64, 128])
def test_lengths_and_pages(dtype, D, page):
    run(1, LENGTHS, 4, 2, 1, D, page, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("D,Dv", [(16, 16), (32, 16), (48, 48), (80, 80), (96, 96), (112, 64), (128, 64), (192, 128), (256, 256), (256, 16)])
def test_head_dims(dtype, D, Dv):
    run(2, [1, 40, 333], 4, 4, 2, D, 16, dtype, Dv=Dv)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(1, 1, 1), (8, 1, 1), (16, 1, 1), (17, 1, 1), (8, 2, 3), (4, 2, 8), (6, 2, 7), (32, 1, 2), (4, 1, 17), (3, 1, 70),
                                       (5, 1, 150)])
def test_rows(dtype, Hq, Hkv, Sq):
    """Rows of one, two and four warps, and of several tiles; requests shorter than their new tokens."""
    for page in (16, 5):
        run(3, [0, 1, Sq, Sq + 1, 200], Hq, Hkv, Sq, 64, page, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("token_major,bhln", [(True, True), (False, False), (True, False)])
def test_layouts(dtype, token_major, bhln):
    run(4, [5, 77, 300], 8, 2, 2, 64, 16, dtype, token_major=token_major, bhln=bhln)
    run(4, [5, 77, 300], 8, 2, 2, 80, 16, dtype, token_major=token_major, bhln=bhln)


@pytest.mark.parametrize("page", [8, 24, 48, 64, 7])
@pytest.mark.parametrize("general", [False, True])
def test_general_kernel(page, general):
    run(5, [1, 100, 700], 8, 2, 1, 128, page, "bf16", kernel_options={"kernels": "general"} if general else None)


def softcap(score, b, h, q_idx, kv_idx):
    return 5.0 * torch.tanh(score / 5.0)


def distance(score, b, h, q_idx, kv_idx):
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


def parity(b, h, q_idx, kv_idx):
    return (q_idx + kv_idx + h) % 2 == 0


def nothing(b, h, q_idx, kv_idx):
    return (kv_idx < 0) & (q_idx < 0)


def no_odd_head(b, h, q_idx, kv_idx):
    return (h % 2 == 0) & (kv_idx >= 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("score", [None, softcap, distance])
@pytest.mark.parametrize("mask", [None, parity, nothing, no_odd_head])
def test_mods(dtype, score, mask):
    run(6, [0, 1, 70, 400], 4, 2, 3, 64, 16, dtype, score=score, mask=mask)
    run(6, [0, 1, 70, 400], 4, 2, 3, 48, 10, dtype, score=score, mask=mask)


@pytest.mark.parametrize("window", [0, 1, 30, 31, 32, 33, 100, 5000, 2 ** 31])
@pytest.mark.parametrize("Sq", [1, 4])
def test_window(window, Sq):
    run(7, [1, 3, 33, 64, 400], 4, 1, Sq, 64, 16, "bf16", window=window)


def test_window_of_row_tiles():
    run(7, [300, 40], 4, 2, 90, 64, 16, "f16", window=50)


@pytest.mark.parametrize("D,page", [(64, 16), (64, 8), (64, 64), (48, 16), (48, 3)])
@pytest.mark.parametrize("Sq", [1, 3])
def test_pages_that_the_window_has_left(D, page, Sq):
    """Their table entries are none any more, and what else lies in front of the window is no number."""
    for dtype in ("f16", "f32"):
        dt, window, lengths = DTYPES[dtype], 70, [1, 71, 72, 75, 130, 333, 1000]
        c = Cache(24, lengths, 2, D, page, dt)
        for b, n in enumerate(lengths):
            first = max(n - Sq - window, 0)  # the first key that any of the queries sees
            for i in range(first // page):
                c.table[b, i] = -1
            p = c.table[b, first // page].long()
            c.k_pages[p, :, : first % page] = math.nan
            c.v_pages[p, :, : first % page] = math.inf
        q = normal(np.random.default_rng(25), len(lengths), 4, Sq, D, dtype=dt)
        for table in (c.table, torch.cat([c.table, torch.full((len(lengths), 6000), -1, dtype=torch.int32, device="cuda")], 1)):  # a CTA per segment, cut segments
            out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, table, c.lengths, window=window, return_lse=True)
            check_attention(out, lse, attend(q, c.keys, c.values, window=window), dt)
        torch.cuda.synchronize()
        fa.check_status()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(4, 2, 1), (12, 2, 2), (6, 2, 7), (8, 1, 5)])
def test_the_same_for_wide_tables(dtype, Hq, Hkv, Sq):
    """Tables with room for much more than there is: the work is cut on the device, with the same results."""
    for D, page, lengths in ((64, 16, [0, 1, 33, 700, 64]), (48, 5, [0, 1, 33, 700, 64]), (128, 64, [3000, 1]), (64, 16, list(range(0, 160)))):
        run(26, lengths, Hq, Hkv, Sq, D, page, dtype, width=20000 // page)
        run(26, lengths, Hq, Hkv, Sq, D, page, dtype, score=distance, mask=parity, window=100, width=20000 // page)


def test_strides_of_single_entries():
    """The stride of a dimension of one entry says nothing."""
    c = Cache(27, [100], 1, 64, 16, torch.float16)
    q = normal(np.random.default_rng(28), 1, 1, 1, 64, dtype=torch.float16).cuda()
    odd = lambda t: t.as_strided(t.shape, [t.stride(i) if n > 1 else 1 for i, n in enumerate(t.shape)])  # noqa: E731
    a = fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths)
    assert torch.equal(a, fa.paged_attention(odd(q), odd(c.k_pages), odd(c.v_pages), c.table, c.lengths))


def test_captured_tensors():
    """Mods over tensors: document ids by position, a bias per head; a tensor on the CPU as well."""
    ids = torch.randint(0, 3, (600,), generator=torch.Generator().manual_seed(0))
    bias = torch.randn(4, generator=torch.Generator().manual_seed(1))
    for dev in ("cuda", "cpu"):
        ids_d, bias_d = ids.to(dev), bias.to(dev)

        def same(b, h, q_idx, kv_idx):
            return ids_d[q_idx] == ids_d[kv_idx]

        def add(score, b, h, q_idx, kv_idx):
            return score + bias_d[h]

        def same_cpu(b, h, q_idx, kv_idx):
            return ids[q_idx.clamp(min=0)] == ids[kv_idx]

        def add_cpu(score, b, h, q_idx, kv_idx):
            return score + bias[h]

        run(8, [1, 20, 600], 4, 2, 2, 64, 16, "f16", score=add_cpu, mask=same_cpu, on_gpu=(add, same))


def test_offsets_of_a_shard():
    """b_offset and h_offset are what the mods see."""
    c = Cache(9, [50, 200, 90], 2, 64, 16, torch.float16)
    q = normal(np.random.default_rng(9), 3, 4, 1, 64, dtype=torch.float16).cuda()
    whole = fa.paged_attention(q, c.k_pages, c.v_pages, c.table, c.lengths, distance, parity)
    part = fa.paged_attention(q[1:, 2:], c.k_pages[:, 1:], c.v_pages[:, 1:], c.table[1:], c.lengths[1:], distance, parity, b_offset=1, h_offset=2)
    assert torch.equal(whole[1:, 2:], part)


@pytest.mark.parametrize("dtype,D,page", [("bf16", 128, 64), ("f16", 64, 16), ("f16", 96, 16), ("f32", 64, 16)])
def test_one_long_request(dtype, D, page):
    """Parts of all workers, and a segment that ends in one."""
    run(10, [20000], 4, 1, 1, D, page, dtype)
    run(10, [3, 20000, 1], 4, 2, 1, D, page, dtype)


@pytest.mark.parametrize("B", [33, 300, 1500])
def test_many_requests(B):
    """More requests than lanes, workers with many segments each."""
    lengths = [int(x) for x in np.random.default_rng(B).integers(0, 90, B)]
    run(11, lengths, 4, 2, 1, 64, 16, "f16")
    run(11, lengths, 4, 2, 1, 48, 16, "f16")


def test_scale_and_same_again():
    a = run(12, [100, 3000, 5], 8, 4, 2, 128, 32, "bf16", scale=0.3)
    b = run(12, [100, 3000, 5], 8, 4, 2, 128, 32, "bf16", scale=0.3)
    assert torch.equal(a, b)  # (no sum depends on which worker is first)


def test_no_requests_and_no_pages():
    c = Cache(13, [4], 2, 64, 16, torch.float16)
    q = torch.zeros(0, 4, 1, 64, dtype=torch.float16, device="cuda")
    out, lse = fa.paged_attention(q, c.k_pages, c.v_pages, c.table[:0], c.lengths[:0], return_lse=True)
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1)
    q = torch.ones(1, 4, 1, 64, dtype=torch.float16, device="cuda")
    out, lse = fa.paged_attention(q, c.k_pages[:0], c.v_pages[:0], c.table[:, :0], torch.zeros_like(c.lengths), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    torch.cuda.synchronize()
    fa.check_status()


@pytest.mark.parametrize("D,page", [(64, 16), (48, 16), (64, 3)])
@pytest.mark.parametrize("bad", ["entry", "negative entry", "length", "negative length"])
def test_bad_entries_are_left_out_and_reported(D, page, bad):
    lengths = [100, 40]
    c = Cache(14, lengths, 2, D, page, torch.float16)
    q = normal(np.random.default_rng(15), 2, 4, 1, D, dtype=torch.float16)
    keys, values = list(c.keys), list(c.values)
    mask = None
    if "entry" in bad:
        c.table[0, 1] = c.k_pages.shape[0] if bad == "entry" else -1

        def mask(b, h, q_idx, kv_idx):
            return (b != 0) | (kv_idx // page != 1)
    elif bad == "length":
        width = c.table.shape[1] - 1
        c.table = c.table[:, :width].contiguous()
        c.lengths[0] = width * page + 5  # is taken for width * page
        more = width * page - 100
        assert more >= 0
        c.k_pages[c.table[0, -1].long()], c.v_pages[c.table[0, -1].long()] = c.k_pages[c.table[0, -1].long()].nan_to_num(0.5), c.v_pages[c.table[0, -1].long()].nan_to_num(0.5)
        keys[0], values[0] = (torch.cat([t, torch.full((2, more, D), 0.5, dtype=t.dtype)], 1) for t in (keys[0], values[0]))
    else:
        c.lengths[0] = -3
        keys[0], values[0] = keys[0][:, :0], values[0][:, :0]
    out, lse = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, return_lse=True)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="0x4"):
        fa.check_status()
    check_attention(out, lse, attend(q, keys, values, mask=mask), torch.float16)


def test_masked_keys_of_any_score():
    """Infinities and NaN of a score_mod in masked places, and a mask of the type's lowest value."""
    low = torch.finfo(torch.float32).min

    def wild(score, b, h, q_idx, kv_idx):
        return torch.where(kv_idx % 3 == 0, score, torch.where(kv_idx % 3 == 1, score / 0.0, score * 0.0 / 0.0))

    def thirds(b, h, q_idx, kv_idx):
        return kv_idx % 3 == 0

    def lowest(score, b, h, q_idx, kv_idx):
        return torch.where(kv_idx % 2 == 0, score, low + score * 0.0)

    def all_lowest(score, b, h, q_idx, kv_idx):
        return score * 0.0 + low

    run(16, [0, 1, 100], 4, 2, 2, 64, 16, "f16", score=wild, mask=thirds)
    run(16, [1, 100], 4, 2, 1, 64, 16, "f16", score=lowest)
    # every score the lowest: the mean of the values (the lse is beyond the range of log2 units, and not looked at)
    c = Cache(17, [50], 2, 64, 16, torch.float16)
    q = normal(np.random.default_rng(17), 1, 4, 1, 64, dtype=torch.float16)
    out = fa.paged_attention(q.cuda(), c.k_pages, c.v_pages, c.table, c.lengths, lambda s, b, h, i, j: s * 0.0 - 1e38)
    ref = c.values[0].double().mean(1).repeat_interleave(2, 0)
    assert (out[0, :, 0].cpu().double() - ref).abs().max() <= 2.0 ** -10


def test_another_stream_and_a_graph():
    """The call works on the current stream, and a captured one follows lengths and tables that change behind its back."""
    a, b = Cache(18, [100, 900], 2, 64, 16, torch.float16, width=80), Cache(19, [1000, 7], 2, 64, 16, torch.float16, width=80)
    n = max(a.k_pages.shape[0], b.k_pages.shape[0])
    q = normal(np.random.default_rng(20), 2, 4, 1, 64, dtype=torch.float16)
    kp, vp = (torch.zeros(n, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    table, lengths = torch.zeros_like(a.table), torch.zeros_like(a.lengths)

    def put(c):
        kp[:c.k_pages.shape[0]].copy_(c.k_pages)
        vp[:c.v_pages.shape[0]].copy_(c.v_pages)
        table.copy_(c.table)
        lengths.copy_(c.lengths)

    qd = q.cuda()
    put(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = fa.paged_attention(qd, kp, vp, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    check_attention(out, None, attend(q, a.keys, a.values), torch.float16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = fa.paged_attention(qd, kp, vp, table, lengths, return_lse=True)
    for c in (a, b, a):
        put(c)
        g.replay()
        check_attention(out, lse, attend(q, c.keys, c.values), torch.float16)


@pytest.mark.parametrize("D,page", [(64, 16), (48, 16)])
def test_offsets_beyond_32_bits(D, page):
    """Pages whose place in memory passes 2^32 bytes and 2^31 values."""
    n = (1 << 31) // (page * D) + 40
    pool = torch.empty(n, 1, page, D, dtype=torch.float16, device="cuda")
    c = Cache(21, [100], 1, D, page, torch.float16)
    used = c.table[0, : -(-100 // page)].long()
    far = n - 1 - torch.arange(len(used), device="cuda")
    pool[far] = c.k_pages[used]
    near = far - 20
    pool[near] = c.v_pages[used]
    q = normal(np.random.default_rng(22), 1, 1, 1, D, dtype=torch.float16)
    # (values 20 pages in front of the keys, in the same tensor)
    out = fa.paged_attention(q.cuda(), pool[20:], pool[:-20], (far - 20)[None].int().contiguous(), c.lengths)
    check_attention(out, None, attend(q, c.keys, c.values), torch.float16)


def test_refusals():
    c = Cache(23, [20], 2, 64, 16, torch.float16)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device="cuda")
    call = lambda **kw: fa.paged_attention(**{**dict(query=q, key_pages=c.k_pages, value_pages=c.v_pages, block_table=c.table, lengths=c.lengths), **kw})  # noqa: E731
    call()
    for kw, err in ((dict(query=q.float()), ValueError), (dict(query=q.double(), key_pages=c.k_pages.double(), value_pages=c.v_pages.double()), ValueError),
                    (dict(query=q[0]), ValueError), (dict(query=q[:, :3]), ValueError), (dict(query=q[..., :48]), ValueError),
                    (dict(query=torch.zeros(2, 4, 1, 64, dtype=torch.float16, device="cuda")), ValueError),
                    (dict(block_table=c.table.long()), ValueError), (dict(lengths=c.lengths.long()), ValueError),
                    (dict(lengths=torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError), (dict(window=-1), ValueError),
                    (dict(value_pages=c.v_pages[:-1]), ValueError), (dict(key_pages=c.k_pages.transpose(2, 3)), ValueError),
                    (dict(query=q.cpu()), RuntimeError), (dict(lengths=c.lengths.cpu()), RuntimeError), (dict(query=[1]), TypeError),
                    (dict(query=q.clone().requires_grad_()), ValueError), (dict(block_table=c.table.t()), ValueError),
                    (dict(key_pages=c.k_pages[..., :8], value_pages=c.v_pages[..., :8], query=q[..., :8]), fa._cabi.FlaxAttnError)):
        with pytest.raises(err):
            call(**kw)
    with torch.no_grad():
        call(query=q.clone().requires_grad_())
    torch.cuda.synchronize()
    fa.check_status()
