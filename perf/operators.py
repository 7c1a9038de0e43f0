"""The operators around attention over a paged key / value cache, as cases that can be timed and compared:

"rotary"   training: queries and keys get an optional RMS norm per head and the rotary position embedding; the pass
           is forward and backward (gradients of queries, keys and norm weights)
"append"   serving: the same for new tokens, whose keys and values go straight into their places in the cache's pages
"step"     pages for the new tokens of a batch of requests: block tables, slots and positions, from the lengths
"attend"   attention of the newest tokens of each request over its pages

A case is a dict of plain values.  With ``own`` false ``run`` computes the plain form: elementary torch operations in
32 bits, rounded once at the end.  With ``own`` true it makes the calls a user makes of flaxattention_b200.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CAP = 30.0
EPS = 1e-6


# ---- score_mods of the attention cases (written once for tensors and for tracing) --------------------------------
def softcap(score, b, h, q_idx, kv_idx):
    """Scores held between -CAP and CAP."""
    return CAP * torch.tanh(score / CAP)


def distance(score, b, h, q_idx, kv_idx):
    """A penalty per position of distance, smaller for every further head."""
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


SCORE_MODS = {"": None, "softcap": softcap, "distance": distance}


# ---- the cases ---------------------------------------------------------------------------------------------------
def _rotary(name, B, Hq, Hkv, S, D, R, dtype, norm=False, interleaved=False, bhln=True):
    return dict(name=name, op="rotary", B=B, Hq=Hq, Hkv=Hkv, S=S, D=D, R=R, dtype=dtype, norm=norm, interleaved=interleaved, bhln=bhln)


def _append(name, T, Hq, Hkv, D, R, dtype, page, norm=False, interleaved=False):
    return dict(name=name, op="append", T=T, Hq=Hq, Hkv=Hkv, D=D, R=R, dtype=dtype, page=page, norm=norm, interleaved=interleaved)


def _step(name, B, T, page, longest):
    return dict(name=name, op="step", B=B, T=T, page=page, longest=longest)


def _attend(name, B, Hq, Hkv, Sq, L, D, dtype, page, mod="", window=0, ragged=True, lse=False):
    return dict(name=name, op="attend", B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, L=L, D=D, dtype=dtype, page=page, mod=mod, window=window,
                ragged=ragged, lse=lse)


def listed():
    return [
        # a layer of a small model in full precision, trained on short sequences: launches and the call itself count
        _rotary("rotary_small_f32", 2, 4, 4, 256, 64, 64, "f32"),
        # a layer of a grouped-query model with normalised queries and keys, trained on whole sequences
        _rotary("rotary_normed_gqa", 4, 32, 8, 4096, 128, 128, "bf16", norm=True),
        # neighbouring values as pairs, part of the head rotated, token-major tensors, no round length
        _rotary("rotary_part_of_head", 3, 16, 4, 1553, 80, 32, "f16", interleaved=True, bhln=False),
        # one new token for each of 32 requests, small pages
        _append("append_one_token", 32, 32, 8, 128, 128, "bf16", 16, norm=True),
        # the prompts of a batch, laid end to end
        _append("append_prompts", 16384, 32, 8, 128, 128, "bf16", 64),
        # the start of a decoding step: one new token each for 64 running requests
        _step("step_one_token", 64, 64, 16, 2048),
        # admission of many prompts at once
        _step("step_prompts", 512, 524288, 64, 4096),
        # short conversations, one new token each: a few microseconds per layer
        _attend("attend_short", 8, 8, 8, 1, 500, 64, "f16", 16, lse=True),
        # the serving batch: requests of all lengths, grouped-query heads
        _attend("attend_ragged_gqa", 32, 32, 8, 1, 16384, 128, "bf16", 64),
        # one request with a long document: everything has to come from the split over its length
        _attend("attend_one_long", 1, 32, 8, 1, 131072, 128, "bf16", 128),
        # five drafted tokens to be checked at once, capped scores
        _attend("attend_drafts_softcap", 16, 16, 4, 5, 4097, 128, "f16", 32, mod="softcap", ragged=False),
        # a layer with a sliding window and a distance penalty, head dim and page size of no power of two
        _attend("attend_window_odd", 24, 8, 8, 1, 3001, 96, "bf16", 12, mod="distance", window=1024, lse=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "step", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    G = rng.choice([1, 1, 2, 4, 8])
    while Hkv * G > 32:
        G //= 2
    if op == "rotary":
        B, R = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([D, D, D, D // 2, 2 * rng.randint(1, D // 2)])
        S = _log(rng, 1, 8192)
        while B * S * Hkv * (G + 1) * D > 60_000_000:
            S = (S + 1) // 2
        c = _rotary("", B, Hkv * G, Hkv, S, D, R, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    elif op == "append":
        R = rng.choice([D, D, D, D // 2, 2 * rng.randint(1, D // 2)])
        T = _log(rng, 1, 16384)
        while T * Hkv * (G + 2) * D > 60_000_000:
            T = (T + 1) // 2
        c = _append("", T, Hkv * G, Hkv, D, R, dtype, rng.choice([1, 8, 12, 16, 16, 32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5)
    elif op == "step":
        B = _log(rng, 1, 2048)
        c = _step("", B, min(524288, B * _log(rng, 1, 1024) + rng.randint(0, B)), rng.choice([1, 8, 12, 16, 16, 32, 64, 128]), _log(rng, 16, 4096))
    else:
        B, L = _log(rng, 1, 64), _log(rng, 1, 131072)
        while B * L * Hkv * D > 110_000_000:
            B, L = ((B + 1) // 2, L) if B > 1 and rng.random() < 0.5 else (B, (L + 1) // 2)
        c = _attend("", B, Hkv * G, Hkv, rng.choice([1, 1, 1, 2, 4, 7]), L, D, dtype, rng.choice([1, 8, 12, 16, 16, 32, 64, 128]),
                    rng.choice(["", "", "softcap", "distance"]), rng.choice([0, 0, 0, 127, 1000]), rng.random() < 0.7, rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of each request: all L, or spread between a tenth of L and L (some shorter than their new tokens)."""
    if not case["ragged"]:
        return [case["L"]] * case["B"]
    return [max(1, int(case["L"] * (0.1 + 0.9 * ((1 + 0.6180339887 * b) % 1.0 or 1.0)))) for b in range(case["B"])]


def _angles(length, R, device):
    """cos | sin of position times frequency, [length, R], worked out in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
    a = torch.arange(length, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def _laid(bhln, *sizes):
    B, H, S, D = sizes
    return (B, H, S, D) if bhln else (B, S, H, D)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=DTYPES.get(case.get("dtype"))):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    s = {"case": case}
    op = case["op"]
    if op == "rotary":
        B, Hq, Hkv, S, D, n = (case[k] for k in ("B", "Hq", "Hkv", "S", "D", "bhln"))
        s["q"], s["k"] = normal(*_laid(n, B, Hq, S, D)).requires_grad_(), normal(*_laid(n, B, Hkv, S, D)).requires_grad_()
        s["dq"], s["dk"] = normal(*_laid(n, B, Hq, S, D)), normal(*_laid(n, B, Hkv, S, D))
        s["table"] = _angles(S, case["R"], "cuda")
    elif op == "append":
        T, Hq, Hkv, D, P = (case[k] for k in ("T", "Hq", "Hkv", "D", "page"))
        s["q"], s["k"], s["v"] = normal(1, T, Hq, D), normal(1, T, Hkv, D), normal(1, T, Hkv, D)
        pages = -(-T // P) + 64
        s["k_pages"], s["v_pages"] = normal(pages, Hkv, P, D), normal(pages, Hkv, P, D)
        s["slots"] = torch.randperm(pages * P, device="cuda", generator=g)[:T].view(1, T)
        s["positions"] = torch.randint(0, 32768, (1, T), device="cuda", generator=g, dtype=torch.int32)
        s["table"] = _angles(32768, case["R"], "cuda")
    elif op == "step":
        B, T, P, longest = (case[k] for k in ("B", "T", "page", "longest"))
        s["lengths"] = torch.randint(0, longest + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        share = torch.rand(B, device="cuda", generator=g, dtype=torch.float64) + 0.1
        ends = (share.cumsum(0) / share.sum() * T).round().long()
        ends[-1] = T
        s["new"] = torch.diff(ends, prepend=ends.new_zeros(1)).int() if T != B else torch.ones(B, device="cuda", dtype=torch.int32)
        had = (s["lengths"] + P - 1) // P
        need = (s["lengths"] + s["new"] + P - 1) // P
        n_had, n_all = int(had.sum()), int(need.sum())
        width = -(-(longest + (1 if T == B else min(T, 11 * T // B + 1))) // P) + 3  # (no share is above 11 / B)
        pool = torch.randperm(n_all + 100, device="cuda", generator=g).int()
        col = torch.arange(width, device="cuda")
        at = had.cumsum(0) - had
        s["block_table"] = torch.where(col < had[:, None], pool[(at[:, None] + col).clamp(max=n_had)], -1).int().contiguous()
        s["free"] = pool[n_had:].contiguous()
        s["taken"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    else:
        B, Hq, Hkv, Sq, D, P = (case[k] for k in ("B", "Hq", "Hkv", "Sq", "D", "page"))
        order = torch.randperm(B, device="cuda", generator=g)
        s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order]
        width = -(-case["L"] // P)
        n = (s["lengths"] + P - 1) // P
        total = int(n.sum())
        pool = torch.randperm(total + 7, device="cuda", generator=g).int()
        col = torch.arange(width, device="cuda")
        s["block_table"] = torch.where(col < n[:, None], pool[((n.cumsum(0) - n)[:, None] + col).clamp(max=total)], 0).int().contiguous()
        s["q"] = normal(B, Hq, Sq, D)
        s["k_pages"], s["v_pages"] = normal(total + 7, Hkv, P, D), normal(total + 7, Hkv, P, D)
    if case.get("norm"):
        s["wq"], s["wk"] = 1 + 0.1 * normal(case["D"]), 1 + 0.1 * normal(case["D"])
        if op == "rotary":
            s["wq"].requires_grad_(), s["wk"].requires_grad_()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, R, interleaved, back=False):
    """The pairs of x's first R values turned by their angles (back: the transposed map)."""
    if back:
        sin = -sin
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2: R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _normed(x, w):
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * inv, inv, x * inv * w


def _angle_of(table, positions, R, bhln):
    """cos and sin of positions [.., S], shaped to broadcast over heads."""
    t = table[positions]
    t = t.unsqueeze(-3) if bhln else t.unsqueeze(-2)
    return t[..., : R // 2], t[..., R // 2:]


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angle_of(s["table"], torch.arange(c["S"], device="cuda"), c["R"], c["bhln"])
    out, grads, weights = [], [], []
    for x, d, w in ((s["q"], s["dq"], s.get("wq")), (s["k"], s["dk"], s.get("wk"))):
        xf = x.detach().float()
        g = _rotate(d.float(), cos, sin, c["R"], c["interleaved"], back=True)
        if w is None:
            y = xf
        else:
            wf = w.detach().float()
            unit, inv, y = _normed(xf, wf)
            weights.append((g * unit).flatten(0, 2).sum(0).to(x.dtype))
            g = g * wf
            g = inv * (g - unit * (g * unit).mean(-1, keepdim=True))
        out.append(_rotate(y, cos, sin, c["R"], c["interleaved"]).to(x.dtype))
        grads.append(g.to(x.dtype))
    return out + grads + weights


def _plain_append(s):
    c = s["case"]
    cos, sin = _angle_of(s["table"], s["positions"].long(), c["R"], False)
    out = []
    for x, w in ((s["q"], s.get("wq")), (s["k"], s.get("wk"))):
        y = x.float() if w is None else _normed(x.float(), w.float())[2]
        out.append(_rotate(y, cos, sin, c["R"], c["interleaved"]).to(x.dtype))
    page, at = s["slots"][0] // c["page"], s["slots"][0] % c["page"]
    s["k_pages"][page, :, at] = out[1][0]
    s["v_pages"][page, :, at] = s["v"][0]
    return [out[0], s["k_pages"], s["v_pages"]]


def _plain_step(s):
    c = s["case"]
    P, old, new, table = c["page"], s["lengths"], s["new"], s["block_table"]
    had, need = (old + P - 1) // P, (old + new + P - 1) // P
    starts = torch.nn.functional.pad(new.cumsum(0), (1, 0)).int()
    first = (need - had).cumsum(0) - (need - had) + s["taken"]  # of a request's new pages, in the free list
    col = torch.arange(table.shape[1], device="cuda")
    nth = first[:, None] + col - had[:, None]
    fresh = (col >= had[:, None]) & (col < need[:, None])
    table.copy_(torch.where(fresh, s["free"][nth.clamp(0, s["free"].numel() - 1)], table))
    t = torch.arange(c["T"], device="cuda")
    r = torch.searchsorted(starts[1:].long(), t, right=True)
    pos = old[r] + (t - starts[r])
    slots = table[r, pos // P].long() * P + pos % P
    taken = s["taken"] + (need - had).sum().int()
    return [old + new, pos.int(), slots, r.int(), starts, taken.int(), table]


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, Sq, D, P = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "D", "page"))
    L = c["L"]
    k, v = (p[s["block_table"]].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2).float() for p in (s["k_pages"], s["v_pages"]))
    q = s["q"].float().view(B, Hkv, Hq // Hkv * Sq, D)
    x = (q @ k.transpose(-1, -2) * D ** -0.5).view(B, Hq, Sq, L)
    qi = (s["lengths"][:, None] - Sq + torch.arange(Sq, device="cuda"))[:, None, :, None]
    ki = torch.arange(L, device="cuda")
    if c["mod"]:
        x = SCORE_MODS[c["mod"]](x, torch.arange(B, device="cuda")[:, None, None, None], torch.arange(Hq, device="cuda")[:, None, None], qi, ki)
    keep = ki <= qi
    if c["window"]:
        keep = keep & (qi - ki <= c["window"])
    x = x.masked_fill(~keep, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    o = (e / total.clamp(min=1e-30)).view(B, Hkv, Hq // Hkv * Sq, L) @ v
    o = o.view(B, Hq, Sq, D).to(s["q"].dtype)
    return [o, (top + total.log())[..., 0]] if c["lse"] else [o]


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "step": _plain_step, "attend": _plain_attend}


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _own_rotary(s):
    import flaxattention_b200 as fa

    c = s["case"]
    w = [s["wq"], s["wk"]] if c["norm"] else []
    out = fa.rotary_embedding(s["q"], s["k"], s["table"], query_weight=s.get("wq"), key_weight=s.get("wk"), eps=EPS,
                              interleaved=c["interleaved"], bhln=c["bhln"])
    return [*(t.detach() for t in out), *torch.autograd.grad(out, [s["q"], s["k"], *w], (s["dq"], s["dk"]))]


def _own_append(s):
    import flaxattention_b200 as fa

    c = s["case"]
    q = fa.rotary_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], s["table"], s["positions"],
                         query_weight=s.get("wq"), key_weight=s.get("wk"), eps=EPS, interleaved=c["interleaved"], bhln=False)
    return [q, s["k_pages"], s["v_pages"]]


def _own_step(s):
    import flaxattention_b200 as fa

    c = s["case"]
    r = fa.page_step(s["lengths"], s["new"], s["block_table"], s["free"], c["page"], c["T"], taken=s["taken"])
    return [r.lengths, r.positions, r.slots, r.requests, r.starts, r.taken, s["block_table"]]


def _own_attend(s):
    import flaxattention_b200 as fa

    c = s["case"]
    r = fa.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], SCORE_MODS[c["mod"]],
                           window=c["window"] or None, return_lse=c["lse"])
    return list(r) if c["lse"] else [r]


OWN = {"rotary": _own_rotary, "append": _own_append, "step": _own_step, "attend": _own_attend}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    es = 4 if case.get("dtype") == "f32" else 2
    if op == "rotary":
        n = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * case["D"]
        # read and write forward; gradients read and written backward, and with a norm the inputs read again
        return {"bytes": n * es * (5 if case["norm"] else 4) + case["S"] * case["R"] * 4,
                "flops": n * (20 if case["norm"] else 6)}
    if op == "append":
        n = case["T"] * case["D"] * (case["Hq"] + 2 * case["Hkv"])
        return {"bytes": 2 * n * es + case["T"] * (case["R"] * 4 + 12), "flops": n * (8 if case["norm"] else 3)}
    if op == "step":
        return {"bytes": 16 * case["T"] + 16 * case["B"] + 8 * (case["T"] // case["page"] + case["B"]), "flops": 4 * case["T"]}
    w, Sq = case["window"], case["Sq"]
    keys = sum(min(n, w + Sq) if w else n for n in _lengths(case))
    rows = case["B"] * case["Hq"] * Sq
    return {"bytes": keys * case["Hkv"] * case["D"] * 2 * es + rows * case["D"] * 2 * es + keys // case["page"] * 4,
            "flops": 4 * keys * case["Hq"] * Sq * case["D"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _turned(x, angle, R, interleaved):
    """x's first R values as complex numbers, multiplied by cos + i sin."""
    z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) if interleaved else torch.complex(x[..., : R // 2], x[..., R // 2: R])
    z = z * angle
    head = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., R:]], -1)


def exact(case, seed):
    op = case["op"]
    if op == "step":
        return None
    s = prepare(case, seed)
    if op == "attend":
        outs, lses = [], []
        for b in range(case["B"]):
            n, G = int(s["lengths"][b]), case["Hq"] // case["Hkv"]
            ids = s["block_table"][b, : -(-n // case["page"])].long()
            k, v = (p[ids].double().permute(1, 0, 2, 3).reshape(case["Hkv"], -1, case["D"])[:, :n].repeat_interleave(G, 0)
                    for p in (s["k_pages"], s["v_pages"]))
            x = torch.einsum("hid,hjd->hij", s["q"][b].double(), k) / math.sqrt(case["D"])
            qi = torch.arange(n - case["Sq"], n, device="cuda", dtype=torch.float64)[:, None]
            ki = torch.arange(n, device="cuda", dtype=torch.float64)
            h = torch.arange(case["Hq"], device="cuda", dtype=torch.float64)[:, None, None]
            if case["mod"] == "softcap":
                x = CAP * torch.tanh(x / CAP)
            elif case["mod"] == "distance":
                x = x - (qi - ki) * 2.0 ** (-(h + 1) / 2)
            x = torch.where((ki > qi) | ((qi - ki > case["window"]) & (case["window"] > 0)), -math.inf, x)
            lse = torch.logsumexp(x, -1)
            outs.append(torch.exp(x - lse.clamp(min=-1e300)[..., None]) @ v)
            lses.append(lse)
        return [torch.stack(outs), torch.stack(lses)] if case["lse"] else [torch.stack(outs)]
    R, bhln = case["R"], case.get("bhln", False)
    t = s["table"].double()
    t = torch.complex(t[:, : R // 2], t[:, R // 2:])
    t = t[s["positions"].long()] if op == "append" else t[None]
    t = t.unsqueeze(1) if bhln else t.unsqueeze(2)

    def forward(x, w):
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w
        return _turned(x, t, R, case["interleaved"])

    if op == "append":
        w = [s[n].double() if n in s else None for n in ("wq", "wk")]
        pages = []
        for p, x in ((s["k_pages"], forward(s["k"].double(), w[1])), (s["v_pages"], s["v"].double())):
            flat = p.double().transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
            flat[s["slots"][0]] = x[0]
            pages.append(flat.view(-1, case["page"], case["Hkv"], case["D"]).transpose(1, 2))
        return [forward(s["q"].double(), w[0]), *pages]
    out, grads, weights = [], [], []
    for x, d, w in (("q", "dq", "wq"), ("k", "dk", "wk")):
        leaf = [s[n].detach().double().requires_grad_() for n in (x, w) if n in s]
        y = forward(leaf[0], leaf[1] if len(leaf) > 1 else None)
        got = torch.autograd.grad(y, leaf, s[d].double())
        out.append(y.detach())
        grads.append(got[0])
        weights += got[1:]
    return out + grads + weights
