"""Caches in pages for the tests, and the definitions of the operators on them in 64 bits (on the CPU, request by request)."""
import math

import numpy as np
import torch

# unit roundoff of a value rounded to the type (f32: far below the noise of sums in another order, which the bounds add)
ROUNDOFF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def normal(rng, *shape, dtype=torch.float32):
    return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to(dtype)


class Cache:
    """Pages with the keys and values of requests of `lengths`, in random order.  What holds no token is NaN, table entries
    behind a request's last page are no pages."""

    def __init__(self, seed, lengths, Hkv, D, page, dtype, Dv=None, token_major=False, spare=2, width=None, device="cuda"):
        rng = np.random.default_rng(seed)
        Dv = D if Dv is None else Dv
        n = [-(-max(x, 0) // page) for x in lengths]
        total = sum(n) + spare
        self.page, self.dtype = page, dtype
        self.keys = [normal(rng, Hkv, x, D, dtype=dtype) for x in lengths]
        self.values = [normal(rng, Hkv, x, Dv, dtype=dtype) for x in lengths]
        width = max(n + [0]) + 1 if width is None else width
        table = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32)
        table[:, ::2] = -7
        k_pages = torch.full((total, Hkv, page, D), math.nan, dtype=dtype)
        v_pages = torch.full((total, Hkv, page, Dv), math.nan, dtype=dtype)
        order, at = rng.permutation(total), 0
        for b, x in enumerate(lengths):
            for i in range(n[b]):
                table[b, i] = p = int(order[at])
                at += 1
                m = min(page, x - i * page)
                k_pages[p, :, :m] = self.keys[b][:, i * page: i * page + m]
                v_pages[p, :, :m] = self.values[b][:, i * page: i * page + m]
        if token_major:  # [pages, page_size, heads, D] seen the other way round
            k_pages, v_pages = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (k_pages, v_pages))
        self.k_pages, self.v_pages = k_pages.to(device), v_pages.to(device)
        self.table = table.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.free = torch.tensor(order[at:].copy(), dtype=torch.int32, device=device)


def attend(q, keys, values, score=None, mask=None, window=None, scale=None):
    """(out, lse, spread) of queries [B, Hq, Sq, D] over lists of keys and values: the definition in 64 bits.  spread: the sums of p |v|,
    and the largest |score|, which the rounding of results goes by."""
    B, Hq, Sq, D = q.shape
    outs, lses, spreads, top = [], [], [], 1.0
    for b in range(B):
        k, v = keys[b].double(), values[b].double()
        G, n = Hq // k.shape[0], k.shape[1]
        k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        x = torch.einsum("hid,hjd->hij", q[b].double(), k) * (1 / math.sqrt(D) if scale is None else scale)
        h = torch.arange(Hq)[:, None, None]
        qi, ki = torch.arange(n - Sq, n)[:, None], torch.arange(n)
        if score is not None and n > 0:
            x = score(x, torch.tensor(b), h, qi, ki).double()
        keep = (ki <= qi) & (ki < n)
        if window is not None:
            keep = keep & (qi - ki <= window)
        if mask is not None and n > 0:
            keep = keep & mask(torch.tensor(b), h, qi, ki)
        keep = keep.expand(x.shape)
        seen = keep & (x > -1e30)  # (a mask's lowest value is no score)
        if seen.any():
            top = max(top, x[seen].abs().max().item())
        x = torch.where(keep, x, -math.inf)
        lse = torch.logsumexp(x, -1) if n > 0 else torch.full((Hq, Sq), -math.inf, dtype=torch.float64)
        p = torch.exp(x - lse.clamp(min=-1e300)[..., None])
        outs.append(p @ v)
        spreads.append(p @ v.abs())
        lses.append(lse)
    return torch.stack(outs), torch.stack(lses), torch.stack(spreads), top


def check_attention(out, lse, want, dtype):
    """Bounds: the output is rounded once (u |o|), each probability once for the product (u sum p |v|, not in fp32); a score is off by some
    fp32 roundings of the largest (2^-21 top, of D products and the mod), which changes probabilities by as much in proportion."""
    ref, ref_lse, spread, top = want
    u = ROUNDOFF[dtype]
    bound = u * ref.abs() + (u + 2.0 ** -20 * (4 + top)) * spread + 2.0 ** -24
    got = out.detach().cpu().double()
    assert got.shape == ref.shape and torch.isfinite(got).all()
    assert ((got - ref).abs() <= bound).all(), ((got - ref).abs() / bound).max().item()
    if lse is not None:
        lse = lse.cpu().double()
        empty = torch.isneginf(ref_lse)
        assert torch.equal(torch.isneginf(lse), empty)
        assert ((lse - ref_lse)[~empty].abs() <= 2.0 ** -20 * (4 + top) + 2.0 ** -22 * ref_lse[~empty].abs()).all()
        assert (got[empty] == 0).all()
