"""The operators of serving together, as a server runs them: prompts in pieces, caches of both kinds, a shared prefix, steps in a CUDA graph."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import attend, check_attention, eight_bits, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits8,prefix", [(False, 40), (True, 0), (True, 200)])
def test_example(bits8, prefix):
    """The example, against layers without a cache.  In 8 bits a key or value is kept to 1 / 254 of its row's largest, at most 4 in size for rows of 64 normed values, a hundredth of what
    their mean size makes of it; two layers of sums over them stay within 1 / 16 of the largest output."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decoding.py")
    spec = importlib.util.spec_from_file_location("paged_decoding", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(steps=5, prompts=(5, 33, 1, 70), check=True, bits8=bits8, prefix=prefix)
    assert r["lengths"] == [10, 38, 6, 75]
    assert r["worst"] <= (2.0 ** -4 if bits8 else 2.0 ** -5)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompts_in_pieces_then_steps(dtype, eight):
    """Prompts of all lengths go in in two pieces, then tokens one by one, replayed as a graph; every output against the definition over what the cache stands for."""
    dt, rng = DTYPES[dtype], np.random.default_rng(0)
    B, Hq, Hkv, D, P, steps = 4, 8, 2, 64, 16, 4
    pieces = [[37, 1, 0, 90], [20, 150, 7, 1]]
    total = [sum(x) + steps for x in zip(*pieces)]
    width = -(-max(total) // P)
    pages = B * width
    q, k, v = ([normal(rng, h, n, D, dtype=dt) for n in total] for h in (Hq, Hkv, Hkv))
    kp, vp = (torch.zeros(pages, Hkv, P, D, dtype=torch.int8 if eight else dt, device="cuda") for _ in range(2))
    scales = dict(key_scales=torch.zeros(pages, Hkv, P, device="cuda"), value_scales=torch.zeros(pages, Hkv, P, device="cuda")) if eight else {}
    kept = []  # what the cache stands for: no rotation and no norm, so that it is known to the bit
    for t in (k, v):
        kept.append([(lambda w, s: w.double() * s.double()[..., None])(*eight_bits(x)) if eight else x for x in t])
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    free = torch.from_numpy(rng.permutation(pages)).int().cuda()
    lengths, taken = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    at = [0] * B

    def rows(t, n):  # the next n[b] tokens of each request, [1, tokens, heads, D]
        return torch.cat([x[:, a: a + m] for x, a, m in zip(t, at, n)], 1).transpose(0, 1)[None].contiguous().cuda()

    for n in pieces:
        s = fa.page_step(lengths, torch.tensor(n, dtype=torch.int32, device="cuda"), table, free, P, sum(n), taken=taken)
        q1 = fa.rotary_append(rows(q, n), rows(k, n), rows(v, n), kp, vp, s.slots, bhln=False, **scales)
        ends = [a + m for a, m in zip(at, n)]
        key_starts = torch.nn.functional.pad(s.lengths.cumsum(0), (1, 0)).int()
        k1, v1 = fa.read_pages(kp, vp, table, key_starts, sum(ends), bhln=False, dtype=dt, **scales)
        out, lse = fa.prompt_attention(q1, k1, v1, s.starts, key_starts=key_starts, bhln=False, return_lse=True)
        first = 0
        for b in range(B):
            if n[b]:
                # (read_pages rounds what the cache stands for to the dtype)
                want = attend(q[b][None, :, at[b]: ends[b]], [kept[0][b][:, : ends[b]].to(dt)], [kept[1][b][:, : ends[b]].to(dt)])
                check_attention(out[:, first: first + n[b]].transpose(1, 2), lse[:, :, first: first + n[b]], want, dt)
            first += n[b]
        at = ends
        lengths, taken = s.lengths.clone(), s.taken.clone()

    one = torch.ones(B, dtype=torch.int32, device="cuda")
    given = [torch.empty(1, B, h, D, dtype=dt, device="cuda") for h in (Hq, Hkv, Hkv)]

    def step():
        s = fa.page_step(lengths, one, table, free, P, B, taken=taken)
        q1 = fa.rotary_append(*given, kp, vp, s.slots, bhln=False, **scales)
        out, lse = fa.paged_attention(q1.view(B, 1, Hq, D), kp, vp, table, s.lengths, bhln=False, return_lse=True, **scales)
        lengths.copy_(s.lengths)
        taken.copy_(s.taken)
        return out, lse

    graph = None
    for i in range(steps):
        for g, t in zip(given, (q, k, v)):
            g.copy_(rows(t, [1] * B))
        at = [a + 1 for a in at]
        if i == 0:
            out, lse = step()
        elif graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out, lse = step()
        if graph is not None:
            graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            want = attend(q[b][None, :, at[b] - 1: at[b]], [kept[0][b][:, : at[b]]], [kept[1][b][:, : at[b]]])
            if not eight:
                check_attention(out[b: b + 1].transpose(1, 2), lse[b: b + 1], want, dt)
            else:  # (probabilities times scales: 32 * 2^-16 of the mean of the rows' largest values, see test_eight_bits_gpu.py; the largest of normal values is below 8)
                err = (out[b: b + 1].transpose(1, 2).cpu().double() - want[0]).abs()
                assert (err <= (2.0 ** -11 if dt == torch.float16 else 2.0 ** -8) * want[0].abs() + 2.0 ** -11 * 8 + 2.0 ** -15 * want[2]).all()
                assert ((lse[b: b + 1].cpu().double() - want[1]).abs() <= 2.0 ** -17).all()
    fa.check_status()


def test_a_step_behind_a_prefix_sees_what_the_step_before_wrote():
    """The pages' kernel runs beside the prefix's: what rotary_append writes in front of both has to be there, over and over."""
    rng = np.random.default_rng(1)
    B, Hq, Hkv, D, P, T = 16, 8, 2, 128, 64, 400
    kp, vp = (torch.zeros(B * 8, Hkv, P, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(B * 8, dtype=torch.int32, device="cuda").view(B, 8)
    pre = [normal(rng, 1, Hkv, 2000, D, dtype=torch.bfloat16).cuda() for _ in range(2)]
    rows = [normal(rng, T, 1, B, h, D, dtype=torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv)]
    lengths = torch.arange(1, T + 1, dtype=torch.int32, device="cuda")[:, None].expand(T, B).contiguous()
    slots = [(table[:, t // P].long() * P + t % P)[None] for t in range(T)]
    outs = {}
    for waits in (True, False):
        kp.zero_(), vp.zero_()
        got = []
        for t in range(T):
            q = fa.rotary_append(*(x[t] for x in rows), kp, vp, slots[t], bhln=False)
            if waits:
                torch.cuda.synchronize()
            got.append(fa.paged_attention(q.view(B, 1, Hq, D), kp, vp, table, lengths[t], bhln=False, prefix=(pre[0].transpose(1, 2), pre[1].transpose(1, 2))))
            if waits:
                torch.cuda.synchronize()
        outs[waits] = torch.stack(got)
    assert torch.equal(outs[True], outs[False])


def test_calls_at_once_on_two_streams():
    """Calls of every operator on two streams, each over tensors of its own: nothing is shared between them."""
    rng = np.random.default_rng(2)
    B, Hq, Hkv, D, P = 8, 8, 2, 128, 16
    lens = torch.tensor([100 + 7 * b for b in range(B)], dtype=torch.int32, device="cuda")
    table = torch.arange(B * 10, dtype=torch.int32, device="cuda").view(B, 10)
    starts = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).int()
    n = int(starts[-1])

    def setup(i):
        x = [normal(rng, 1, n, h, D, dtype=torch.float16).cuda() for h in (Hq, Hkv, Hkv)]
        pre = [normal(rng, 1, Hkv, 1500, D, dtype=torch.float16).cuda() for _ in range(2)]
        pages = [torch.zeros(B * 10, Hkv, P, D, dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = [torch.zeros(B * 10, Hkv, P, device="cuda") for _ in range(2)]
        return x, pre, pages, scales

    token = torch.arange(n, device="cuda")
    b = torch.searchsorted(starts[1:].long(), token, right=True)
    j = token - starts[b]
    slots = table[b, j // P].long() * P + j % P

    def run(state):
        (q, k, v), pre, pages, scales = state
        sc = dict(key_scales=scales[0], value_scales=scales[1])
        q1 = fa.rotary_append(q, k, v, *pages, slots, bhln=False, **sc)
        k1, v1 = fa.read_pages(*pages, table, starts, n, dtype=torch.float16, bhln=False, **sc)
        o1 = fa.prompt_attention(q1, k1, v1, starts, bhln=False)
        last = q1[0, starts[1:].long() - 1][:, :, None]
        o2 = fa.paged_attention(last, *pages, table, lens, prefix=(pre[0], pre[1]), **sc)
        o3 = fa.paged_attention(last, *pages, table, lens, **sc)
        return o1, o2, o3

    states = [setup(i) for i in range(2)]
    want = [run(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(states[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(r, want[i]))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    q = torch.randn(1, 2, 100, 64, device="cuda:1", dtype=torch.float16)
    out = fa.prompt_attention(q, q, q, torch.tensor([0, 100], dtype=torch.int32, device="cuda:1"))
    assert out.device == q.device and torch.isfinite(out).all()
