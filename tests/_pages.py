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


def eight_bits(x):
    """The whole numbers and scales that rows of x (last dimension) have in a cache of 8 bits: the definition, in fp32 divisions."""
    x = x.float()
    scale = torch.where(torch.isfinite(x).all(-1), x.abs().amax(-1) / 127, math.nan)
    whole = torch.where(scale[..., None] > 0, (x / scale[..., None]).round().clamp(-127, 127), torch.zeros(()))
    return whole.nan_to_num(0.0).to(torch.int8), scale


class Cache8(Cache):
    """The same in 8 bits: `keys` and `values` are what the pages stand for, in 64 bits.  Scales of what holds no token are NaN."""

    def __init__(self, seed, lengths, Hkv, D, page, dtype, *args, token_major=False, **kw):
        super().__init__(seed, lengths, Hkv, D, page, dtype, *args, token_major=token_major, **kw)
        device = self.k_pages.device
        for n in ("k", "v"):
            whole, scale = eight_bits(getattr(self, n + "_pages").cpu())
            empty = torch.isnan(scale)
            whole[empty] = torch.randint(-128, 128, whole[empty].shape, generator=torch.Generator().manual_seed(seed)).to(torch.int8)
            if token_major:
                whole, scale = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (whole, scale))
            setattr(self, n + "_pages", whole.to(device))
            setattr(self, n + "_scales", scale.to(device))
        for n in ("keys", "values"):
            got = []
            for x in getattr(self, n):
                whole, scale = eight_bits(x)
                got.append(whole.double() * scale.double()[..., None])
            setattr(self, n, got)

    @property
    def scales(self):
        return dict(key_scales=self.k_scales, value_scales=self.v_scales)


def with_slope(want, slope):
    """The tcgen05 kernels take a bias that is linear over the keys from that of the first key of a tile of 128, which the sums of up to 128 slopes are added to:
    three roundings of 128 slopes at most, 3 * 2^-24 * 128 |slope|, written as 2^-20 of a larger `top`."""
    return (*want[:3], want[3] + 3 * 2.0 ** -24 * 128 * slope / 2.0 ** -20)


class Prompts:
    """Requests of `lengths` new tokens behind `past` others, laid end to end; rows of no request (`pad` in front and behind) are NaN."""

    def __init__(self, seed, lengths, Hq, Hkv, D, dtype, Dv=None, past=None, pad=(0, 0), bhln=True, device="cuda"):
        rng = np.random.default_rng(seed)
        Dv = D if Dv is None else Dv
        self.lengths, self.dtype, self.pad, self.bhln = lengths, dtype, pad, bhln
        total = [n + p for n, p in zip(lengths, past or [0] * len(lengths))]
        self.queries = [normal(rng, Hq, n, D, dtype=dtype) for n in lengths]
        self.keys = [normal(rng, Hkv, n, D, dtype=dtype) for n in total]
        self.values = [normal(rng, Hkv, n, Dv, dtype=dtype) for n in total]
        self.starts, self.key_starts = (torch.tensor([pad[0]] + [int(x) for x in pad[0] + np.cumsum(n)], dtype=torch.int32, device=device) for n in (lengths, total))
        self.q, self.k, self.v = (self.laid(x, device) for x in (self.queries, self.keys, self.values))
        self.past = past is not None

    def laid(self, parts, device):
        front, back = (torch.full((parts[0].shape[0], n, parts[0].shape[2]), math.nan, dtype=self.dtype) for n in self.pad)
        x = torch.cat([front, *parts, back], 1)[None]
        return (x if self.bhln else x.transpose(1, 2).contiguous()).to(device)

    def want(self, score=None, mask=None, window=None, scale=None):
        """The definition in 64 bits: (out, lse, spread, top) of all requests' rows."""
        outs, top = [], 1.0
        for b, (q, k, v) in enumerate(zip(self.queries, self.keys, self.values)):
            f = None if score is None else lambda x, _, h, i, j: score(x, torch.tensor(b), h, i, j)  # noqa: B023
            g = None if mask is None else lambda _, h, i, j: mask(torch.tensor(b), h, i, j)  # noqa: B023
            *r, t = attend(q[None], [k], [v], f, g, window, scale)
            outs.append([x[0] for x in r])
            top = max(top, t)
        return (*(torch.cat([o[i] for o in outs], 1)[None] for i in range(3)), top)

    def check(self, out, lse, want):
        front, back = self.pad
        if not self.bhln:
            out = out.transpose(1, 2)
        n = sum(self.lengths)
        for t, nothing in ((out, 0.0), (lse[..., None], -math.inf)):
            assert (t[:, :, :front] == nothing).all() and (t[:, :, front + n:] == nothing).all()
        check_attention(out[:, :, front: front + n], lse[:, :, front: front + n], want, self.dtype)
