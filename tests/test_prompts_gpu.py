"""prompt_attention against its definition in 64 bits: types, head layouts, lengths around tiles, pieces of prompts, windows and mods, rows of no request."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import Prompts, check_attention, with_slope
from _util import DTYPES

pytestmark = pytest.mark.gpu


def run(seed, lengths, Hq, Hkv, D, dtype, score=None, mask=None, window=None, scale=None, kernels=None, **kw):
    p = Prompts(seed, lengths, Hq, Hkv, D, DTYPES[dtype], **kw)
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, score, mask, key_starts=p.key_starts if p.past else None, window=window, sm_scale=scale, bhln=p.bhln,
                                   return_lse=True, kernel_options={"kernels": kernels} if kernels else None)
    assert out.dtype == p.dtype and lse.dtype == torch.float32
    p.check(out, lse, with_slope(p.want(score, mask, window, scale), 2.0 ** -0.5 if score is distance else 0.0))
    torch.cuda.synchronize()
    fa.check_status()
    return out


LENGTHS = [5, 0, 1, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (4, 1), (6, 2)])
def test_lengths_and_heads(kernels, dtype, D, Hq, Hkv):
    run(1, LENGTHS, Hq, Hkv, D, dtype, kernels=kernels, pad=(3, 7))


@pytest.mark.parametrize("dtype,D,Dv", [*(("f16", *x) for x in ((16, 16), (48, 48), (80, 80), (96, 32), (112, 64), (128, 64), (192, 128), (256, 256))),
                                        *(("f32", *x) for x in ((16, 16), (96, 96), (256, 256), (256, 16)))])
def test_head_dims(dtype, D, Dv):
    run(2, [1, 40, 333], 4, 2, D, dtype, Dv=Dv)


@pytest.mark.parametrize("G", [1, 3, 5, 7, 8, 12, 32, 130])
def test_groups(G):
    run(3, [1, 33, 140], G, 1, 64, "bf16")


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("bhln", [True, False])
def test_pieces(kernels, D, bhln):
    """Queries behind keys that were there before; also fewer keys than queries, whose first then see nothing."""
    run(4, [1, 2, 130, 64, 7], 4, 2, D, "bf16", past=[500, 0, 126, 64, 3], bhln=bhln, kernels=kernels)
    p = Prompts(5, [40, 9], 4, 2, D, torch.float16, bhln=bhln)
    short = torch.tensor([0, 15, 20], dtype=torch.int32, device="cuda")
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, key_starts=short, bhln=bhln, return_lse=True)
    full_k, full_v = (torch.cat(x, 1) for x in (p.keys, p.values))
    p.keys, p.values = ([x[:, :15], x[:, 15:20]] for x in (full_k, full_v))
    p.check(out, lse, p.want())
    assert torch.isneginf(lse[0, :, :25]).all() and torch.isfinite(lse[0, :, 25:40]).all()


def softcap(score, b, h, q_idx, kv_idx):
    return 5.0 * torch.tanh(score / 5.0)


def distance(score, b, h, q_idx, kv_idx):
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


def of_request(score, b, h, q_idx, kv_idx):
    return score * (b + 1) * 0.5


def parity(b, h, q_idx, kv_idx):
    return (q_idx + kv_idx + h + b) % 2 == 0


def nothing(b, h, q_idx, kv_idx):
    return (kv_idx < 0) & (q_idx < 0)


def no_odd_head(b, h, q_idx, kv_idx):
    return (h % 2 == 0) & (kv_idx >= 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("score,mask", [(softcap, None), (of_request, parity), (None, nothing), (distance, no_odd_head)])
def test_mods(dtype, score, mask):
    run(6, [1, 70, 400, 200], 4, 2, 64, dtype, score=score, mask=mask)
    run(6, [1, 70, 400], 4, 2, 128, dtype, score=score, mask=mask, past=[3, 200, 0])


@pytest.mark.parametrize("kernels", [None, "general"])
@pytest.mark.parametrize("window", [0, 1, 63, 64, 127, 128, 129, 300, 5000, 2 ** 31])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(kernels, window, D):
    run(7, [1, 3, 129, 700], 4, 1, D, "bf16", window=window, kernels=kernels)
    run(8, [40, 200], 2, 2, D, "f16", window=window, kernels=kernels, past=[300, 100], score=distance)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(D, scale):
    run(9, [100, 30], 2, 1, D, "f16", scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_other_requests_may_hold_anything(dtype, D):
    p = Prompts(10, [130, 100, 50], 2, 2, D, DTYPES[dtype])
    a, b = 130, 230
    p.k[:, :, a:b], p.v[:, :, a:b], p.q[:, :, a:b] = math.nan, math.inf, -math.inf
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, return_lse=True)
    want = p.want()
    keep = torch.cat([torch.arange(a), torch.arange(b, 280)])
    check_attention(out.cpu()[:, :, keep], lse.cpu()[:, :, keep], (*(x[:, :, keep] for x in want[:3]), want[3]), p.dtype)


def test_many_requests():
    """More requests than a warp keeps, most of them of no tokens."""
    rng = np.random.default_rng(11)
    lengths = [int(rng.integers(0, 40)) if b % 3 == 0 else 0 for b in range(700)]
    lengths[500] = 600
    run(12, lengths, 2, 1, 64, "bf16")
    run(12, lengths, 2, 1, 128, "f32")


def test_nothing_there():
    q = torch.zeros(1, 2, 0, 64, device="cuda", dtype=torch.float16)
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert fa.prompt_attention(q, q, q, starts).shape == (1, 2, 0, 64)
    # tokens, but no requests, or none with tokens; queries without keys
    q = torch.full((1, 2, 300, 64), math.nan, device="cuda", dtype=torch.float16)
    for s in (torch.zeros(1, dtype=torch.int32, device="cuda"), starts, starts + 7):
        out, lse = fa.prompt_attention(q, q, q, s, return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
    out, lse = fa.prompt_attention(q, q[:, :, :0], q[:, :, :0], torch.tensor([0, 300], dtype=torch.int32, device="cuda"), key_starts=starts[:2], return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    torch.cuda.synchronize()
    fa.check_status()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("starts", [[0, 50, 20, 100], [0, 30, 500, 100], [-5, 30, 60, 100], [70, 10, 2 ** 31 - 1, -2 ** 31]])
def test_broken_starts(dtype, starts):
    """Cut to what is there, and reported."""
    p = Prompts(13, [100], 2, 1, 64, DTYPES[dtype])
    fa.prompt_attention(p.q, p.k, p.v, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="starts"):
        fa.check_status()


@pytest.mark.parametrize("D", [64, 128])
def test_strides(D):
    """Parts of one projection, read by their strides; rows of 16 bytes beside each other and not."""
    lengths = [100, 30, 61]
    p = Prompts(14, lengths, 4, 2, D, torch.bfloat16, bhln=False)
    qkv = torch.cat([p.q, p.k, p.v], 2)
    q, k, v = qkv.split([4, 2, 2], 2)
    out, lse = fa.prompt_attention(q, k, v, p.starts, bhln=False, return_lse=True)
    p.check(out, lse, p.want())
    wide = torch.zeros(1, 191, 2, 2 * D + 8, dtype=torch.bfloat16, device="cuda")
    wide[..., 8: D + 8], wide[..., D + 8:] = p.k, p.v
    out2, _ = fa.prompt_attention(q, wide[..., 8: D + 8], wide[..., D + 8:], p.starts, bhln=False, return_lse=True)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("D", [64, 128])
def test_one_long_prompt(D):
    run(15, [3000], 2, 1, D, "bf16")


def test_offsets_and_captured_tensors():
    """b and h as the mods see them, and a mod over a tensor."""
    bias = torch.randn(8, 4, generator=torch.Generator().manual_seed(0))
    on_gpu = bias.cuda()

    def by_table(score, b, h, q_idx, kv_idx):
        return score + on_gpu[b, h]

    p = Prompts(16, [70, 150], 2, 1, 64, torch.float16)
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, by_table, return_lse=True, b_offset=5, h_offset=2)
    p.check(out, lse, p.want(lambda x, b, h, i, j: x + bias[b + 5, h + 2]))


def test_graph_and_stream():
    """Captured once, replayed over other lengths; on another stream than the current one's."""
    p = Prompts(17, [200, 90, 40], 4, 2, 128, torch.bfloat16)
    fa.prompt_attention(p.q, p.k, p.v, p.starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, return_lse=True)
        graph.replay()
    side.synchronize()
    p.check(out, lse, p.want())
    p.lengths = [10, 300, 20]
    cut = torch.tensor(p.lengths).cumsum(0)[:-1]
    p.queries, p.keys, p.values = ([x.contiguous() for x in torch.cat(t, 1).tensor_split(cut, 1)] for t in (p.queries, p.keys, p.values))
    p.starts.copy_(torch.tensor([0, 10, 310, 330], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    p.check(out, lse, p.want())


def test_refusals():
    p = Prompts(18, [20, 30], 4, 2, 64, torch.float16)
    call = lambda **kw: fa.prompt_attention(*({"query": p.q, "key": p.k, "value": p.v, "starts": p.starts} | kw).values()) if "key_starts" not in kw else None  # noqa: E731
    call()
    for kw, match in ((dict(query=torch.cat([p.q, p.q])), "batch dimension"), (dict(query=p.q[..., :48]), "embedding"), (dict(key=p.k[:, :, :40], value=p.v[:, :, :40]), "key_starts"),
                      (dict(value=p.v[:, :, :40]), "same heads and sequence"), (dict(starts=p.starts.long()), "starts"), (dict(starts=p.starts[::2]), "starts"),
                      (dict(starts=p.starts[:0]), "starts"), (dict(query=p.q[:, :3]), "multiple"), (dict(key=p.k.float()), "dtype"), (dict(query=p.q.clone().requires_grad_()), "no gradient")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    with pytest.raises(ValueError, match="window"):
        fa.prompt_attention(p.q, p.k, p.v, p.starts, window=-1)
    with pytest.raises(ValueError, match="key_starts"):
        fa.prompt_attention(p.q, p.k, p.v, p.starts, key_starts=p.key_starts[:2])
    with pytest.raises(fa._cabi.FlaxAttnError, match="16"):
        fa.prompt_attention(p.q[..., :60], p.k[..., :60], p.v[..., :60], p.starts)


@pytest.mark.parametrize("D", [96, 128])
def test_two_query_tiles(D):
    """Long prompts at wide heads take two tiles per CTA: rows of one end in the first, between, in the second."""
    run(19, [2300, 1900, 2101], 8, 1, D, "bf16")
    run(20, [700, 660, 600], 24, 1, D, "f16", past=[1700, 2000, 1500], score=distance, window=1900)


@pytest.mark.parametrize("D,Dv", [(64, 64), (96, 48), (128, 128)])
@pytest.mark.parametrize("score,window", [(None, None), (distance, 1500), (None, 600)])
def test_few_rows_over_many_keys(D, Dv, score, window):
    """Keys in parts: requests that have some of the parts only, no keys, no tokens; rows of no request; what lies behind a request is no number."""
    p = Prompts(21, [16, 1, 0, 30], 4, 1, D, torch.bfloat16, Dv=Dv, past=[3000, 4100, 100, 0], pad=(2, 3))
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, score, key_starts=p.key_starts, window=window, return_lse=True)
    p.check(out, lse, with_slope(p.want(score, None, window), 2.0 ** -0.5 if score else 0.0))
    again, _ = fa.prompt_attention(p.q, p.k, p.v, p.starts, score, key_starts=p.key_starts, window=window, return_lse=True)
    assert torch.equal(out, again)


def test_one_row_over_many_keys():
    run(22, [1], 1, 1, 64, "f16", past=[20000])
    run(23, [5], 8, 2, 128, "bf16", past=[9000], mask=parity, score=softcap)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("low", [-3.4028234663852886e38, -math.inf])
def test_scores_that_take_keys_out(D, dtype, low):
    """The lowest value and minus infinity as scores: what they leave of a row, or nothing."""
    def lowest(score, b, h, q_idx, kv_idx):
        return torch.where((kv_idx < 130) | (kv_idx % 3 == 1), low, score)

    p = Prompts(24, [140, 300], 2, 1, D, DTYPES[dtype])
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, lowest, return_lse=True)
    p.check(out, lse, p.want(None, lambda b, h, i, j: (j >= 130) & (j % 3 != 1)))
    assert torch.isneginf(lse[0, :, :131]).all()  # (130 % 3 == 1)


def test_scores_far_below_zero_are_no_mask():
    """A penalty of 1e4 for all keys of the first tiles: the rows that have no others are softmaxes of those, the others do not see them."""
    def far(score, b, h, q_idx, kv_idx):
        return torch.where(kv_idx < 200, score - 1e4, score)

    p = Prompts(25, [330], 2, 2, 64, torch.float16)
    out, lse = fa.prompt_attention(p.q, p.k, p.v, p.starts, far, return_lse=True)
    out, lse = out.cpu().double(), lse.cpu().double()
    ref, ref_lse, spread, _ = p.want(far)
    # (fp32 scores near 1e4 have steps of 2^-10, in log2 units: probabilities are off by as much in proportion)
    off = torch.where(torch.arange(330) < 200, 2.0 ** -9, 2.0 ** -16)
    assert ((out - ref).abs() <= 2.0 ** -11 * ref.abs() + (2.0 ** -11 + off)[:, None] * spread + 2.0 ** -24).all()
    assert ((lse - ref_lse).abs() <= off + 2.0 ** -22 * ref_lse.abs()).all()


@pytest.mark.parametrize("pad", [(0, 0), (50, 700)])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "f16"), (32, "f32")])
def test_hundreds_of_requests(pad, D, dtype):
    """257 and more are found in another way: none with tokens, one, several tiles; rows of no request in front and behind, of several items."""
    rng = np.random.default_rng(26)
    lengths = [int(rng.integers(0, 30)) for _ in range(300)]
    lengths[0], lengths[17], lengths[299] = 0, 400, 129
    run(27, lengths, 6, 2, D, dtype, pad=pad)
    run(28, [0] * 256 + [1], 2, 1, D, dtype, pad=pad)


def test_broken_starts_of_hundreds_of_requests():
    p = Prompts(29, [300], 2, 1, 64, torch.float16)
    starts = torch.randint(-2 ** 31, 2 ** 31 - 1, (400,), generator=torch.Generator().manual_seed(0)).int().cuda()
    fa.prompt_attention(p.q, p.k, p.v, starts)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="starts"):
        fa.check_status()


@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16"), (32, "f16"), (256, "bf16")])
@pytest.mark.parametrize("general", [False, True])
def test_capped_scores_over_the_whole_range(D, dtype, general):
    """Rows that see one key each (a window of 0): the logsumexp is the capped score itself.

    A score here is one product, exact in fp32, and a scale of 1.  Roundings, in proportion: tanh 4e-7 (3.3e-7 of its form and roundings, a reciprocal off
    by 2^-23), its argument's two (2^-24 each), the cap's, the way to log2 units and back (4 more): 4e-7 + 7 * 2^-24 < 1e-6.  And the exponential of 0,
    which is the sum: 1 to within 2.7e-6."""
    torch_type = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    q = torch.zeros(1, 2048, 1, D, dtype=torch_type, device="cuda")
    k, v = torch.zeros_like(q), torch.ones_like(q)
    values = torch.cat([torch.linspace(-300, 300, 1024), torch.logspace(-12, 15.9, 512, base=2), -torch.logspace(-12, 15.9, 512, base=2)]).to(torch_type)
    q[0, :, 0, 3] = values.cuda()
    k[0, :, 0, 3] = 1.0
    starts = torch.tensor([0, 2048], dtype=torch.int32, device="cuda")
    options = {"kernels": "general"} if general else None
    for score, want in ((lambda s, b, h, qi, ki: 30.0 * torch.tanh(s / 30.0), 30 * torch.tanh(values.double() / 30)),
                        (lambda s, b, h, qi, ki: 5.0 - torch.tanh(s * 0.5) * (-2.0) + (qi - ki) * 0.25, 5 + 2 * torch.tanh(values.double() * 0.5))):
        out, lse = fa.prompt_attention(q, k, v, starts, score, window=0, sm_scale=1.0, bhln=False, return_lse=True, kernel_options=options)
        size = want.abs() + (0 if want[0] < 0 else 10)  # (of the second, the sum's parts)
        assert ((lse.reshape(-1).double().cpu() - want).abs() <= 1e-6 * size + 2.7e-6).all()
        assert (out == 1).all()
    q[0, 5, 0, 3] = float("nan")
    out, lse = fa.prompt_attention(q, k, v, starts, lambda s, b, h, qi, ki: 30.0 * torch.tanh(s / 30.0), window=0, sm_scale=1.0, bhln=False, return_lse=True, kernel_options=options)
    assert lse.reshape(-1)[5].isnan() and out[0, 5].isnan().all() and not lse.reshape(-1)[6:].isnan().any()
