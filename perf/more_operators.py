"""Operators of serving that read long prompts, shared ones and caches of 8 bits, as cases that can be timed and compared:

"cache"    new tokens of a batch go into pages of 8-bit integers with a scale for each token and head (rotary positions and an
           optional norm in front), and all tokens of the requests are read back, as the next piece of a prompt needs them
"attend8"  attention of the newest tokens of each request over such pages
"prompt"   causal attention of whole prompts, or of pieces of them, laid end to end
"prefix"   attention of the newest tokens of requests that begin with the same long prompt: over that, computed once for
           all, and over the pages of each

A case is a dict of plain values.  With ``own`` false ``run`` computes the plain form: elementary torch operations in
32 bits, rounded once at the end.  With ``own`` true it makes the calls a user makes of flaxattention_b200.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CAP = 30.0
EPS = 1e-6


# ---- score_mods (written once for tensors and for tracing) --------------------------------------------------------
def softcap(score, b, h, q_idx, kv_idx):
    """Scores held between -CAP and CAP."""
    return CAP * torch.tanh(score / CAP)


def distance(score, b, h, q_idx, kv_idx):
    """A penalty per position of distance, smaller for every further head."""
    return score - (q_idx - kv_idx) * torch.exp2((h + 1) * -0.5)


SCORE_MODS = {"": None, "softcap": softcap, "distance": distance}


# ---- the cases ---------------------------------------------------------------------------------------------------
def _cache(name, B, past, new, Hq, Hkv, D, R, dtype, page, norm=False):
    return dict(name=name, op="cache", B=B, past=past, new=new, Hq=Hq, Hkv=Hkv, D=D, R=R, dtype=dtype, page=page, norm=norm)


def _attend8(name, B, Hq, Hkv, Sq, L, D, dtype, page, mod="", window=0, ragged=True, lse=False):
    return dict(name=name, op="attend8", B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, L=L, D=D, dtype=dtype, page=page, mod=mod, window=window,
                ragged=ragged, lse=lse)


def _prompt(name, B, Hq, Hkv, L, D, dtype, past=0, mod="", window=0, ragged=True, lse=False):
    return dict(name=name, op="prompt", B=B, Hq=Hq, Hkv=Hkv, L=L, D=D, dtype=dtype, past=past, mod=mod, window=window, ragged=ragged, lse=lse)


def _prefix(name, B, Hq, Hkv, Sq, P, L, D, dtype, page, bits8=False, mod="", window=0, lse=False):
    return dict(name=name, op="prefix", B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, P=P, L=L, D=D, dtype=dtype, page=page, bits8=bits8, mod=mod, window=window,
                ragged=True, lse=lse)


def listed():
    return [
        # the first tokens of a few short conversations: launches and the calls themselves count
        _cache("cache_short", 8, 40, 3, 8, 8, 64, 64, "f16", 16),
        # a piece of 1000 tokens for each of 8 long prompts, whose earlier pieces are in the cache
        _cache("cache_pieces", 8, 8000, 1000, 32, 8, 128, 128, "bf16", 64, norm=True),
        # short conversations, one new token each: a few microseconds per layer
        _attend8("attend8_short", 8, 8, 8, 1, 500, 64, "f16", 16, lse=True),
        # the serving batch: requests of all lengths, grouped-query heads
        _attend8("attend8_ragged_gqa", 32, 32, 8, 1, 16384, 128, "bf16", 64),
        # five drafted tokens to be checked at once, capped scores, small pages
        _attend8("attend8_drafts_softcap", 16, 16, 4, 5, 4097, 128, "f16", 32, mod="softcap", ragged=False),
        # a handful of short questions
        _prompt("prompt_short", 7, 8, 8, 60, 64, "f16", lse=True),
        # the prompts of a batch, of all lengths, grouped-query heads
        _prompt("prompt_ragged_gqa", 8, 32, 8, 4096, 128, "bf16"),
        # one long document, head dim 64, local layers
        _prompt("prompt_long_window", 1, 16, 4, 16384, 64, "bf16", window=4096, ragged=False),
        # pieces of prompts that continue what the cache holds, head dim of no power of two, capped scores
        _prompt("prompt_pieces_odd", 5, 12, 4, 777, 80, "f16", past=3001, mod="softcap", lse=True),
        # a short instruction in front of everything
        _prefix("prefix_short", 8, 8, 8, 1, 500, 200, 64, "f16", 16, lse=True),
        # the serving batch behind a long system prompt
        _prefix("prefix_long_gqa", 64, 32, 8, 1, 8192, 1000, 128, "bf16", 64),
        # drafted tokens behind a document of no round length, the requests' own tokens in 8 bits
        _prefix("prefix_drafts_8bit", 24, 16, 4, 3, 5001, 700, 128, "f16", 32, bits8=True, mod="distance"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend8", "attend8", "prompt", "prompt", "prefix"])
    dtype = rng.choice(["bf16", "f16"])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    G = rng.choice([1, 1, 2, 3, 4, 8])
    while Hkv * G > 32:
        G //= 2
    page = rng.choice([1, 8, 12, 16, 16, 32, 64, 128])
    mod = rng.choice(["", "", "softcap", "distance"])
    lse = rng.random() < 0.5
    window = rng.choice([0, 0, 0, 127, 1000])
    if op == "cache":
        B, past, new = _log(rng, 1, 32), _log(rng, 1, 8000), _log(rng, 1, 1000)
        while B * ((past + new) * Hkv + new * Hkv * G) * D > 100_000_000:
            B, past, new = (B + 1) // 2, (past + 1) // 2, (new + 1) // 2
        c = _cache("", B, past, new, Hkv * G, Hkv, D, rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), dtype, page, rng.random() < 0.5)
    elif op == "attend8":
        B, L = _log(rng, 1, 64), _log(rng, 1, 131072)
        while B * L * Hkv * D > 110_000_000:
            B, L = ((B + 1) // 2, L) if B > 1 and rng.random() < 0.5 else (B, (L + 1) // 2)
        c = _attend8("", B, Hkv * G, Hkv, rng.choice([1, 1, 1, 2, 4, 7]), L, D, dtype, page, mod, window, rng.random() < 0.7, lse)
    elif op == "prompt":
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        B, L, past = _log(rng, 1, 64), _log(rng, 1, 8192), rng.choice([0, 0, 0, _log(rng, 1, 8192)])
        most = 100_000_000 if dtype == "f32" or D > 128 else 1_000_000_000
        while B * Hkv * G * L * (L + past) > most:
            B, L, past = ((B + 1) // 2, L, past) if B > 1 and rng.random() < 0.5 else (B, (L + 1) // 2, past // 2)
        c = _prompt("", B, Hkv * G, Hkv, L, D, dtype, past, mod, window, rng.random() < 0.7, lse)
    else:
        B, P, L = _log(rng, 1, 64), _log(rng, 1, 16384), _log(rng, 1, 2000)
        while P * Hkv * D > 16_000_000 or B * L * Hkv * D > 60_000_000:
            P, L = (P + 1) // 2, (L + 1) // 2
        c = _prefix("", B, Hkv * G, Hkv, rng.choice([1, 1, 1, 2, 4, 7]), P, L, D, dtype, page, rng.random() < 0.5, mod, window, lse)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------
def _spread(B, most, ragged=True):
    """B lengths: all `most`, or spread between a tenth of it and all."""
    return [most if not ragged else max(1, int(most * (0.1 + 0.9 * ((1 + 0.6180339887 * b) % 1.0 or 1.0)))) for b in range(B)]


def _angles(length, R, device):
    """cos | sin of position times frequency, [length, R], worked out in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
    a = torch.arange(length, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def _eight_bits(x):
    """Whole numbers from -127 to 127 and the scales of the rows (last dimension) that make x of them again, nearly."""
    x = x.float()
    scale = x.abs().amax(-1) / 127
    whole = torch.where(scale[..., None] > 0, (x / scale[..., None]).round().clamp(-127, 127), 0.0)
    return whole.to(torch.int8), scale


def _ends(lengths):
    return torch.nn.functional.pad(lengths.cumsum(0), (1, 0)).int()


def _block_table(lengths, page, width, pool):
    n = (lengths + page - 1) // page
    col = torch.arange(width, device="cuda")
    return torch.where(col < n[:, None], pool[((n.cumsum(0) - n)[:, None] + col).clamp(max=pool.numel() - 1)], 0).int().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    def pages(n, bits8):
        k, v = (normal(n, case["Hkv"], case["page"], case["D"]) for _ in range(2))
        if not bits8:
            return {"k_pages": k, "v_pages": v}
        (k, ks), (v, vs) = _eight_bits(k), _eight_bits(v)
        return {"k_pages": k, "v_pages": v, "k_scales": ks, "v_scales": vs}

    s = {"case": case}
    op, B, Hq, Hkv, D = (case[k] for k in ("op", "B", "Hq", "Hkv", "D"))
    if op == "prompt":
        order = torch.randperm(B, device="cuda", generator=g)
        n = torch.tensor(_spread(B, case["L"], case["ragged"]), device="cuda")[order]
        had = torch.tensor(_spread(B, case["past"]) if case["past"] else [0] * B, device="cuda")
        s["starts"], s["key_starts"] = _ends(n), _ends(n + had)
        T = sum(_spread(B, case["L"], case["ragged"]))
        Tk = T + (sum(_spread(B, case["past"])) if case["past"] else 0)
        s["q"], s["k"], s["v"] = normal(1, T, Hq, D), normal(1, Tk, Hkv, D), normal(1, Tk, Hkv, D)
        return s
    P = case["page"]
    if op == "cache":
        had = torch.tensor(_spread(B, case["past"]), device="cuda")[torch.randperm(B, device="cuda", generator=g)]
        n = had + case["new"]
        T = B * case["new"]
        s["q"], s["k"], s["v"] = normal(1, T, Hq, D), normal(1, T, Hkv, D), normal(1, T, Hkv, D)
        total = int(((n + P - 1) // P).sum())
        s["block_table"] = _block_table(n, P, -(-(case["past"] + case["new"]) // P), torch.randperm(total + 7, device="cuda", generator=g).int())
        s |= pages(total + 7, True)
        at = had[:, None] + torch.arange(case["new"], device="cuda")
        s["positions"] = at.view(1, T).int()
        s["slots"] = (s["block_table"].gather(1, at // P).long() * P + at % P).view(1, T)
        s["starts"], s["tokens"] = _ends(n), sum(_spread(B, case["past"])) + T
        s["table"] = _angles(case["past"] + case["new"], case["R"], "cuda")
        if case["norm"]:
            s["wq"], s["wk"] = 1 + 0.1 * normal(D), 1 + 0.1 * normal(D)
        return s
    s["lengths"] = torch.tensor(_spread(B, case["L"], case["ragged"]), device="cuda", dtype=torch.int32)[torch.randperm(B, device="cuda", generator=g)]
    total = int(((s["lengths"] + P - 1) // P).sum())
    s["block_table"] = _block_table(s["lengths"], P, -(-case["L"] // P), torch.randperm(total + 7, device="cuda", generator=g).int())
    s["q"] = normal(B, Hq, case["Sq"], D)
    s |= pages(total + 7, op == "attend8" or case["bits8"])
    if op == "prefix":
        s["k_prefix"], s["v_prefix"] = normal(1, Hkv, case["P"], D), normal(1, Hkv, case["P"], D)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------
def _rotated(x, w, cos, sin, R):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x[..., : R // 2], x[..., R // 2: R]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], -1)


def _plain_cache(s):
    c = s["case"]
    P, R = c["page"], c["R"]
    t = s["table"][s["positions"].long()].unsqueeze(-2)
    q, k = (_rotated(x, w, t[..., : R // 2], t[..., R // 2:], R) for x, w in ((s["q"], s.get("wq")), (s["k"], s.get("wk"))))
    page, at = s["slots"][0] // P, s["slots"][0] % P
    for x, n in ((k, "k"), (s["v"], "v")):
        s[n + "_pages"][page, :, at], s[n + "_scales"][page, :, at] = _eight_bits(x[0])
    token = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), token, right=True)
    j = token - s["starts"][b]
    page, at = s["block_table"][b, j // P].long(), j % P
    out = [(s[n + "_pages"][page, :, at].float() * s[n + "_scales"][page, :, at, None])[None].to(s["q"].dtype) for n in ("k", "v")]
    return [q.to(s["q"].dtype), *out]


def _gathered(s, n, L):
    """The pages of all requests as [B, Hkv, L, D] in 32 bits."""
    x = s[n + "_pages"][s["block_table"]].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2).float()
    if n + "_scales" in s:
        x = x * s[n + "_scales"][s["block_table"]].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2)[..., None]
    return x


def _softmax(x, keep):
    x = x.masked_fill_(~keep, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    return x.div_(total.clamp(min=1e-30)), (top + total.log())[..., 0]


def _scored(c, q, k, qi, ki):
    """Scores [B, Hq, Sq, L] of queries [B, Hq, Sq, D] and keys [B or 1, Hkv, L, D], and which keys are seen."""
    B, Hq, Sq, D = q.shape
    x = (q.view(B, c["Hkv"], -1, D) @ k.transpose(-1, -2)).view(B, Hq, Sq, -1).mul_(D ** -0.5)
    if c["mod"]:
        x = SCORE_MODS[c["mod"]](x, None, torch.arange(Hq, device="cuda")[:, None, None], qi, ki)
    keep = ki <= qi
    return x, keep & (qi - ki <= c["window"]) if c["window"] else keep


def _weighed(c, p, v):
    B, Hq, Sq, L = p.shape
    return (p.view(B, c["Hkv"], -1, L) @ v).view(B, Hq, Sq, -1)


def _plain_attend8(s):
    c = s["case"]
    qi = (s["lengths"][:, None] - c["Sq"] + torch.arange(c["Sq"], device="cuda"))[:, None, :, None]
    x, keep = _scored(c, s["q"].float(), _gathered(s, "k", c["L"]), qi, torch.arange(c["L"], device="cuda"))
    p, lse = _softmax(x, keep)
    o = _weighed(c, p, _gathered(s, "v", c["L"])).to(s["q"].dtype)
    return [o, lse] if c["lse"] else [o]


def _plain_prompt(s):
    c = s["case"]
    L, Lk = c["L"], c["L"] + c["past"]
    T, Tk = s["q"].shape[1], s["k"].shape[1]
    n, nk = torch.diff(s["starts"].long())[:, None], torch.diff(s["key_starts"].long())[:, None]
    at, col = torch.arange(L, device="cuda"), torch.arange(Lk, device="cuda")
    rows, keys = (s["starts"][:-1, None] + at).clamp(max=T - 1), (s["key_starts"][:-1, None] + col).clamp(max=Tk - 1)
    q = s["q"][0][rows].transpose(1, 2).float().contiguous()
    k, v = (t[0][keys].transpose(1, 2).float() for t in (s["k"], s["v"]))
    x, keep = _scored(c, q, k, (nk - n + at)[:, None, :, None], col)
    p, lse = _softmax(x, keep)
    o = _weighed(c, p, v)
    to = torch.where(at < n, rows, T).flatten()  # (rows that pad a prompt go behind the last)
    out = o.new_empty(T + 1, c["Hq"], c["D"])
    out[to] = o.transpose(1, 2).flatten(0, 1)
    res = [out[None, :T].to(s["q"].dtype)]
    if c["lse"]:
        out = lse.new_empty(T + 1, c["Hq"])
        out[to] = lse.transpose(1, 2).flatten(0, 1)
        res.append(out[:T].t()[None].contiguous())
    return res


def _plain_prefix(s):
    c = s["case"]
    L, P = c["L"], c["P"]
    own_q = (s["lengths"][:, None] - c["Sq"] + torch.arange(c["Sq"], device="cuda"))[:, None, :, None]
    ki = torch.arange(P + L, device="cuda")
    q = s["q"].float()
    xs = [_scored(c, q, s["k_prefix"].float(), own_q + P, ki[:P]), _scored(c, q, _gathered(s, "k", L), own_q + P, ki[P:])]
    p, lse = _softmax(torch.cat([x for x, _ in xs], -1), torch.cat([keep for _, keep in xs], -1) & (own_q >= 0))
    o = (_weighed(c, p[..., :P].contiguous(), s["v_prefix"].float()) + _weighed(c, p[..., P:].contiguous(), _gathered(s, "v", L))).to(s["q"].dtype)
    return [o, lse] if c["lse"] else [o]


PLAIN = {"cache": _plain_cache, "attend8": _plain_attend8, "prompt": _plain_prompt, "prefix": _plain_prefix}


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _own_cache(s):
    import flaxattention_b200 as fa

    q = fa.rotary_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], s["table"], s["positions"], query_weight=s.get("wq"),
                         key_weight=s.get("wk"), eps=EPS, bhln=False, key_scales=s["k_scales"], value_scales=s["v_scales"])
    k, v = fa.read_pages(s["k_pages"], s["v_pages"], s["block_table"], s["starts"], s["tokens"], key_scales=s["k_scales"],
                         value_scales=s["v_scales"], dtype=s["q"].dtype, bhln=False)
    return [q, k, v]


def _own_paged(s):
    import flaxattention_b200 as fa

    c = s["case"]
    r = fa.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], SCORE_MODS[c["mod"]], window=c["window"] or None,
                           return_lse=c["lse"], key_scales=s.get("k_scales"), value_scales=s.get("v_scales"),
                           prefix=(s["k_prefix"], s["v_prefix"]) if c["op"] == "prefix" else None)
    return list(r) if c["lse"] else [r]


def _own_prompt(s):
    import flaxattention_b200 as fa

    c = s["case"]
    r = fa.prompt_attention(s["q"], s["k"], s["v"], s["starts"], SCORE_MODS[c["mod"]], key_starts=s["key_starts"] if c["past"] else None,
                            window=c["window"] or None, return_lse=c["lse"], bhln=False)
    return list(r) if c["lse"] else [r]


OWN = {"cache": _own_cache, "attend8": _own_paged, "prompt": _own_prompt, "prefix": _own_paged}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def _pairs(n, had, window):
    """How many (query, key) pairs a causal prompt of n tokens behind `had` others has, at most `window` apart."""
    whole = n * had + n * (n + 1) // 2
    if not window:
        return whole
    beyond = max(0, had + n - 1 - window)  # of the last query; of the one before it one fewer, ..
    few = min(n, beyond)
    return whole - (beyond * (beyond + 1) // 2 - (beyond - few) * (beyond - few + 1) // 2)


def work(case):
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "cache":
        T, all_tokens = B * case["new"], sum(_spread(B, case["past"])) + B * case["new"]
        n = T * (2 * Hq + 2 * Hkv) * D
        kv = 2 * all_tokens * Hkv
        # queries read and written, new keys and values read; all 8-bit rows with their scales: the old read, the new written; all of it written
        return {"bytes": n * es + kv * (D + 4) + kv * D * es + T * (case["R"] * 4 + 12), "flops": n * 6 + kv * D}
    if case["op"] == "prompt":
        n, had = _spread(B, case["L"], case["ragged"]), _spread(B, case["past"]) if case["past"] else [0] * B
        T, Tk = sum(n), sum(n) + sum(had)
        # (which length goes with which past is up to the seed: of each query the mean)
        pairs = sum(_pairs(a, sum(had) // B, case["window"]) for a in n)
        return {"bytes": (2 * T * Hq + 2 * Tk * Hkv) * D * es + (T * Hq * 4 if case["lse"] else 0), "flops": 4 * pairs * Hq * D}
    w, Sq = case["window"], case["Sq"]
    lengths = _spread(B, case["L"], case["ragged"])
    keys = sum(min(n, w + Sq) if w else n for n in lengths)
    bits8 = case["op"] == "attend8" or case["bits8"]
    size = keys * Hkv * 2 * (D + 4 if bits8 else D * es) + 2 * B * Hq * Sq * D * es + keys // case["page"] * 4
    pairs = keys
    if case["op"] == "prefix":
        seen = [min(case["P"], max(0, w + Sq - n)) if w else case["P"] for n in lengths]
        size += max(seen) * Hkv * 2 * D * es
        pairs += sum(seen)
    return {"bytes": size, "flops": 4 * pairs * Hq * Sq * D}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _attention64(case, q, k, v, first):
    """Queries [Hq, n, D] whose first one is token `first`, keys and values [Hkv, m, D]: (output, lse), a head at a time."""
    outs, lses = [], []
    ki = torch.arange(k.shape[1], device="cuda", dtype=torch.float64)
    qi = torch.arange(first, first + q.shape[1], device="cuda", dtype=torch.float64)[:, None]
    for h in range(case["Hq"]):
        hk = h // (case["Hq"] // case["Hkv"])
        x = q[h] @ k[hk].T / math.sqrt(case["D"])
        if case["mod"] == "softcap":
            x = CAP * torch.tanh(x / CAP)
        elif case["mod"] == "distance":
            x = x - (qi - ki) * 2.0 ** (-(h + 1) / 2)
        x[(ki > qi) | ((qi - ki > case["window"]) & (case["window"] > 0))] = -math.inf
        lses.append(torch.logsumexp(x, -1))
        outs.append(torch.exp(x - lses[-1].clamp(min=-1e300)[:, None]) @ v[hk])
    return torch.stack(outs), torch.stack(lses)


def _pages64(s, b, n):
    """Keys and values [Hkv, n, D] of request b."""
    ids = s["block_table"][b, : -(-n // s["case"]["page"])].long()
    out = []
    for name in ("k", "v"):
        x = s[name + "_pages"][ids].double()
        if name + "_scales" in s:
            x = x * s[name + "_scales"][ids].double()[..., None]
        out.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    if case["op"] == "cache":
        R = case["R"]
        t = s["table"].double()[s["positions"].long()][:, :, None]
        turn = torch.complex(t[..., : R // 2], t[..., R // 2:])

        def forward(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * turn
            return torch.cat([z.real, z.imag, x[..., R:]], -1)

        out = [forward(s["q"], s.get("wq"))]
        new = case["new"]
        for name, x in (("k", forward(s["k"], s.get("wk"))), ("v", s["v"].double())):
            top = x.abs().amax(-1, keepdim=True) / 127
            x = (torch.round(x / top.clamp(min=1e-300)) * top)[0].view(B, new, Hkv, D)
            parts = []
            for b in range(B):
                n = int(s["starts"][b + 1] - s["starts"][b])
                parts += [_pages64(s, b, n)[0 if name == "k" else 1].transpose(0, 1)[: n - new], x[b]]
            out.append(torch.cat(parts)[None])
        return out
    outs, lses = [], []
    if case["op"] == "prompt":
        starts, key_starts = s["starts"].tolist(), s["key_starts"].tolist()
    for b in range(B):
        if case["op"] == "prompt":
            n, m = starts[b + 1] - starts[b], key_starts[b + 1] - key_starts[b]
            q = s["q"][0, starts[b]: starts[b + 1]].double().transpose(0, 1)
            k, v = (x[0, key_starts[b]: key_starts[b + 1]].double().transpose(0, 1) for x in (s["k"], s["v"]))
            o, lse = _attention64(case, q, k, v, m - n)
        else:
            n, P = int(s["lengths"][b]), case.get("P", 0)
            k, v = _pages64(s, b, n)
            if P:
                k, v = torch.cat([s["k_prefix"][0].double(), k], 1), torch.cat([s["v_prefix"][0].double(), v], 1)
            o, lse = _attention64(case, s["q"][b].double(), k, v, P + n - case["Sq"])
            none = max(0, case["Sq"] - n)  # queries in front of the request's first token
            o[:, :none], lse[:, :none] = 0, -math.inf
        outs.append(o)
        lses.append(lse)
    if case["op"] == "prompt":
        o, lse = torch.cat(outs, 1).transpose(0, 1)[None], torch.cat(lses, 1)[None]
    else:
        o, lse = torch.stack(outs), torch.stack(lses)
    return [o, lse] if case["lse"] else [o]
