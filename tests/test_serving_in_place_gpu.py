"""Steps behind a shared prefix, as a serving loop makes them: lengths, block table, scales and a tensor that the score_mod reads are rewritten in place in front of every call."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight,kernels,B,prefix", [(False, None, 16, 2000), (False, "general", 16, 300), (True, None, 16, 2000), (True, "general", 40, 2000), (True, None, 3, 40)])
def test_what_is_rewritten_in_place_is_seen(eight, kernels, B, prefix):
    """Every call with a wait for the GPU around it, without any, and all calls as one graph: the same to the bit."""
    rng = np.random.default_rng(1)
    Hq, Hkv, D, P, T = 8, 2, 128, 16, 64
    width = T // P
    pages = 2 * B * width  # twice the batch's: the table changes from one half to the other, whose values differ
    kp, vp = (torch.zeros(pages, Hkv, P, D, dtype=torch.int8 if eight else torch.bfloat16, device="cuda") for _ in range(2))
    scales = [torch.zeros(pages, Hkv, P, device="cuda") for _ in range(2)]
    kw = dict(key_scales=scales[0], value_scales=scales[1]) if eight else {}
    tables = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).int().view(2, B, width).cuda()
    table, lengths = torch.zeros_like(tables[0]), torch.zeros(B, dtype=torch.int32, device="cuda")
    biases = normal(rng, 3, Hq, prefix + T).cuda()
    bias = torch.zeros_like(biases[0])
    pre = [normal(rng, 1, prefix, Hkv, D, dtype=torch.bfloat16).cuda() for _ in range(2)]
    rows = [normal(rng, T, 2, 1, B, h, D, dtype=torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv)]
    slots = [[(t[:, i // P].long() * P + i % P)[None] for t in tables] for i in range(T)]

    def near(score, b, h, q_idx, kv_idx):
        return score + bias[h, kv_idx]

    def steps(wait):
        got = []
        lengths.zero_()
        for t in (kp, vp, *scales):
            t.zero_()
        for i in range(T):
            lengths.add_(1)
            table.copy_(tables[i % 2])
            bias.copy_(biases[i % 3])
            for half in (1 - i % 2, i % 2):
                q = fa.rotary_append(*(x[i, half] for x in rows), kp, vp, slots[i][half], bhln=False, **kw)
            wait()
            got.append(fa.paged_attention(q.view(B, 1, Hq, D), kp, vp, table, lengths, near, bhln=False, prefix=pre, kernel_options={"kernels": kernels} if kernels else None, **kw))
            wait()
        return torch.stack(got)

    want = steps(torch.cuda.synchronize)
    assert torch.isfinite(want).all() and not torch.equal(want[0], want[1])
    assert torch.equal(steps(lambda: None), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps(lambda: None)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    fa.check_status()
