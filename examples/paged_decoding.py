"""Serving with a paged key / value cache: prompts of different lengths, then tokens one by one.

A few layers of grouped-query attention (random weights) over a batch of requests.  The prompts go in at once, laid end to end: their
queries and keys are normed and rotated by ``rotary_append``, which also writes keys and values into the cache, and attend through
``prompt_attention`` over what ``read_pages`` lays end to end of them.  After that every step is ``page_step`` once and, per layer, ``rotary_append`` and
``paged_attention`` (here with a capped score).  Nothing in a step waits for the GPU or depends on a length on the host, so that the steps run
as one CUDA graph.

    python examples/paged_decoding.py [--steps N] [--check] [--bits8] [--prefix N]

``--bits8``: the cache holds 8-bit integers with a scale for each token and head.  ``--prefix N``: all requests begin with the same ``N`` tokens, whose keys and
values are worked out once and attended to once for all requests in every step.  ``--check`` computes every step again without a cache and compares.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import flaxattention_b200 as fa  # noqa: E402

LAYERS, WIDTH, HEADS, KV_HEADS, DIM, PAGE = 2, 256, 8, 2, 64, 16
CAP = 20.0


def softcap(score, b, h, q_idx, kv_idx):
    return CAP * torch.tanh(score / CAP)


class Layer:
    def __init__(self, g, pages, bits8):
        def weight(*shape):
            return (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to("cuda", torch.bfloat16)

        self.qkv, self.out = weight(WIDTH, (HEADS + 2 * KV_HEADS) * DIM), weight(HEADS * DIM, WIDTH)
        self.wq, self.wk = (torch.ones(DIM, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.keys, self.values = (torch.zeros(pages, KV_HEADS, PAGE, DIM, device="cuda", dtype=torch.int8 if bits8 else torch.bfloat16) for _ in range(2))
        scales = [torch.zeros(pages, KV_HEADS, PAGE, device="cuda") if bits8 else None for _ in range(2)]
        self.scales = dict(key_scales=scales[0], value_scales=scales[1])
        self.prefix = None  # keys and values that all requests begin with

    def split(self, x):
        """[1, tokens, heads, DIM] of queries, keys and values: parts of one product, read by their strides."""
        return (x @ self.qkv).view(1, len(x), -1, DIM).split([HEADS, KV_HEADS, KV_HEADS], 2)


def plain(layers, table, x, starts):
    """All tokens of all requests (x, laid end to end) through the layers, without a cache."""
    pos = torch.cat([torch.arange(b - a) for a, b in zip(starts, starts[1:])]).cuda()
    ids = torch.cat([torch.full((b - a,), i) for i, (a, b) in enumerate(zip(starts, starts[1:]))]).cuda()

    def same_request(b, h, q_idx, kv_idx):
        return (ids[q_idx] == ids[kv_idx]) & (q_idx >= kv_idx)

    for layer in layers:
        q, k, v = layer.split(x)
        q, k = fa.rotary_embedding(q, k, table, pos[None], query_weight=layer.wq, key_weight=layer.wk, bhln=False)
        o = fa.flax_attention_pallas(q, k, v, score_mod=softcap, mask_mod=same_request, bhln=False, enable_gqa=True)
        x = x + o.reshape(len(x), -1) @ layer.out
    return x


@torch.no_grad()
def main(steps=8, prompts=(5, 33, 1, 70), check=False, bits8=False, prefix=0):
    B, longest = len(prompts), max(prompts) + steps
    width = -(-longest // PAGE)
    g = torch.Generator().manual_seed(0)
    layers = [Layer(g, B * width, bits8) for _ in range(LAYERS)]
    table = fa.rotary_table(prefix + longest, DIM, device="cuda")
    block_table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    free = torch.randperm(B * width, generator=g).int().cuda()
    tokens = (torch.randn(sum(prompts) + steps * B, WIDTH, generator=g)).to("cuda", torch.bfloat16)  # (in place of an embedding)
    common = (torch.randn(prefix, WIDTH, generator=g)).to("cuda", torch.bfloat16)

    # ---- what all requests begin with: one prompt, whose keys and values every layer keeps
    x = common
    for layer in layers if prefix else ():
        q, k, v = layer.split(x)
        q, k = fa.rotary_embedding(q, k, table, query_weight=layer.wq, key_weight=layer.wk, bhln=False)
        o = fa.prompt_attention(q, k, v, torch.tensor([0, prefix], dtype=torch.int32, device="cuda"), softcap, bhln=False)
        layer.prefix = (k, v)
        x = x + o.reshape(prefix, -1) @ layer.out

    # ---- the prompts
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    new = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    step = fa.page_step(lengths, new, block_table, free, PAGE, sum(prompts))
    n, positions = sum(prompts), prefix + step.positions[None]
    # (with a prefix every prompt has its keys in front: the rows of both go to their places among all)
    mine = torch.arange(n, device="cuda") + (step.requests + 1) * prefix
    key_starts = step.starts + torch.arange(B + 1, dtype=torch.int32, device="cuda") * prefix
    x = tokens[:n]
    for layer in layers:
        q, k, v = layer.split(x)
        q2 = fa.rotary_append(q, k, v, layer.keys, layer.values, step.slots, table, positions, query_weight=layer.wq, key_weight=layer.wk, bhln=False, **layer.scales)
        # (the keys and values as attention is to have them, here and in the steps to come, are the ones in the cache)
        kv = fa.read_pages(layer.keys, layer.values, block_table, step.starts, n, bhln=False, dtype=x.dtype, **layer.scales)
        if prefix:
            whole = [t.new_empty(1, n + B * prefix, KV_HEADS, DIM) for t in kv]
            for to, t, p in zip(whole, kv, layer.prefix):
                for b in range(B):
                    to[:, sum(prompts[:b]) + b * prefix:][:, :prefix] = p
                to[:, mine] = t
            kv = whole
        o = fa.prompt_attention(q2, *kv, step.starts, softcap, key_starts=key_starts, bhln=False)
        x = x + o.reshape(len(x), -1) @ layer.out
    outputs = [x]

    # ---- one token per request and step
    lengths, taken = step.lengths.clone(), step.taken.clone()
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    given = torch.empty(B, WIDTH, device="cuda", dtype=torch.bfloat16)

    def decode():
        s = fa.page_step(lengths, one, block_table, free, PAGE, B, taken=taken)
        x = given
        for layer in layers:
            q, k, v = layer.split(x)
            q = fa.rotary_append(q, k, v, layer.keys, layer.values, s.slots, table, prefix + s.positions[None], query_weight=layer.wq, key_weight=layer.wk, bhln=False,
                                 **layer.scales)
            o = fa.paged_attention(q.view(B, 1, HEADS, DIM), layer.keys, layer.values, block_table, s.lengths, softcap, bhln=False, prefix=layer.prefix, **layer.scales)
            x = x + o.reshape(B, -1) @ layer.out
        lengths.copy_(s.lengths)
        taken.copy_(s.taken)
        return x

    graph, result = None, None
    for i in range(steps):
        given.copy_(tokens[sum(prompts) + i * B: sum(prompts) + (i + 1) * B])
        if i == 0:
            result = decode()  # (the first step compiles and loads the kernels)
        elif graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                result = decode()
        if graph is not None:
            graph.replay()
        outputs.append(result.clone())
    torch.cuda.synchronize()
    fa.check_status()

    worst = None
    if check:
        # the same tokens, request by request, through the layers without a cache
        n = [prefix + p + steps for p in prompts]
        starts = [sum(n[:i]) for i in range(B + 1)]
        at = [sum(prompts[:i]) for i in range(B)]
        rows = torch.cat([torch.cat([common, tokens[at[b]: at[b] + prompts[b]], tokens[sum(prompts) + b:: B]]) for b in range(B)])
        want = plain(layers, table, rows, starts)
        want = torch.cat([want[starts[b] + prefix: starts[b + 1]] for b in range(B)])
        got = torch.cat([torch.cat([outputs[0][at[b]: at[b] + prompts[b]], *(o[b: b + 1] for o in outputs[1:])]) for b in range(B)])
        worst = ((got.float() - want.float()).abs().max() / want.float().abs().max()).item()
    return {"lengths": lengths.tolist(), "pages": int(taken), "worst": worst}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--check", action="store_true")
    ap.add_argument("--bits8", action="store_true")
    ap.add_argument("--prefix", type=int, default=0)
    a = ap.parse_args()
    print(main(a.steps, check=a.check, bits8=a.bits8, prefix=a.prefix))
