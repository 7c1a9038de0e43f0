"""rotary_embedding and rotary_append against their definition in 64 bits, gradients against the formula's and against differences."""
import math

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import ROUNDOFF, normal
from _util import DTYPES

pytestmark = pytest.mark.gpu
EPS = 1e-5


def definition(x, w, angle, R, interleaved):
    """x [.., S, D] in 64 bits; angle complex [.., S, R / 2] or None"""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if R == 0:
        return x
    z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) if interleaved else torch.complex(x[..., : R // 2], x[..., R // 2: R])
    z = z * angle
    turned = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([turned, x[..., R:]], -1)


def check(got, ref, dtype, terms=1.0):
    """One rounding of the result, and some fp32 roundings of what it is made of (as large as the largest value of the row; of sums of `terms`
    values: as many as these add up to)."""
    got, size = got.detach().cpu().double(), ref.abs().amax(-1, keepdim=True)
    assert got.shape == ref.shape
    bound = ROUNDOFF[dtype] * ref.abs() + 2.0 ** -20 * size * terms + 2.0 ** -24
    assert ((got - ref).abs() <= bound).all(), ((got - ref).abs() / bound).max().item()


def case(seed, B, Hq, Hkv, S, D, dtype, norm, wdtype=None):
    rng = np.random.default_rng(seed)
    dt = DTYPES[dtype]
    q, k = normal(rng, B, Hq, S, D, dtype=dt), normal(rng, B, Hkv, S, D, dtype=dt)
    dq, dk = normal(rng, B, Hq, S, D, dtype=dt), normal(rng, B, Hkv, S, D, dtype=dt)
    w = [(1 + 0.2 * normal(rng, D)).to(dt if wdtype is None else wdtype) if norm else None for _ in range(2)]
    return q, k, dq, dk, w


def run(B, Hq, Hkv, S, D, R, dtype, norm=False, interleaved=False, bhln=True, positions=None, seed=0, wdtype=None, which=(0, 1), table=None, lay=None):
    q, k, dq, dk, w = case(seed, B, Hq, Hkv, S, D, dtype, norm, wdtype)
    if norm and which != (0, 1):
        w = [x if i in which else None for i, x in enumerate(w)]
    dt = DTYPES[dtype]
    table = fa.rotary_table(max(S, 300), R, 1000.0) if table is None else table
    t = table.double()
    pos = torch.arange(S) if positions is None else positions
    angle = torch.complex(t[:, : R // 2], t[:, R // 2:])[pos.long()] if R else None
    if angle is not None and angle.ndim == 3:
        angle = angle[:, None]
    lay = lay or ((lambda x: x) if bhln else (lambda x: x.transpose(1, 2).contiguous()))
    gq, gk = lay(q).cuda().requires_grad_(), lay(k).cuda().requires_grad_()
    gw = [None if x is None else x.cuda().requires_grad_() for x in w]
    oq, ok = fa.rotary_embedding(gq, gk, table.cuda() if R else None, None if positions is None else positions.cuda(), query_weight=gw[0], key_weight=gw[1],
                                 eps=EPS, interleaved=interleaved, bhln=bhln)
    assert oq.dtype == dt and oq.shape == gq.shape and ok.shape == gk.shape
    torch.autograd.backward((oq, ok), (lay(dq).cuda(), lay(dk).cuda()))
    torch.cuda.synchronize()
    fa.check_status()
    back = (lambda x: x) if bhln else (lambda x: x.transpose(1, 2))
    for x, d, o, g, i in ((q, dq, oq, gq.grad, 0), (k, dk, ok, gk.grad, 1)):
        leaf = x.double().requires_grad_()
        wl = None if w[i] is None else w[i].double().requires_grad_()
        y = definition(leaf, wl, angle, R, interleaved)
        y.backward(d.double())
        check(back(o), y.detach(), dt, 4)
        check(back(g), leaf.grad, dt, 8 + D ** 0.5)
        if wl is not None:
            got, ref = gw[i].grad.cpu().double(), wl.grad
            assert got.dtype == torch.float64 and gw[i].grad.dtype == w[i].dtype
            rows = x.numel() // D
            # (sums over the rows of products of two values of N(0, 1): each off by some fp32 roundings, the sum by as many of its partial sums)
            bound = ROUNDOFF[w[i].dtype] * ref.abs() + 2.0 ** -20 * (8 + 4 * rows ** 0.5)
            assert ((got - ref).abs() <= bound).all(), ((got - ref).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,R", [(64, 64), (64, 32), (64, 16), (64, 10), (64, 0), (128, 128), (80, 80), (80, 48), (96, 64), (256, 256), (16, 16), (48, 6), (20, 20), (33, 8), (1, 0)])
def test_head_dims(dtype, interleaved, norm, D, R):
    run(2, 3, 1, 37, D, R, dtype, norm, interleaved)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bhln", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,S", [(1, 1, 1, 1), (1, 32, 8, 1), (3, 9, 3, 5), (1, 4, 4, 1000), (2, 17, 1, 130), (5, 8, 2, 63)])
def test_shapes(dtype, bhln, B, Hq, Hkv, S):
    for norm in (False, True):
        run(B, Hq, Hkv, S, 64, 64, dtype, norm, bhln=bhln, seed=1)
        run(B, Hq, Hkv, S, 24, 10, dtype, norm, bhln=bhln, seed=1)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("per_request", [False, True])
def test_positions(kind, per_request):
    pos = torch.randint(0, 300, (3, 41) if per_request else (41,), dtype=kind, generator=torch.Generator().manual_seed(3))
    run(3, 4, 2, 41, 64, 64, "f16", True, positions=pos)
    run(3, 4, 2, 41, 30, 20, "f16", False, True, positions=pos)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 6e4])
def test_values_that_stay_are_copied(interleaved, value):
    """What lies behind the rotated part is passed on bit by bit, whatever it is, and does not touch what is rotated."""
    for D, R in ((64, 20), (64, 22), (64, 32), (24, 6), (20, 6), (128, 128 - 2)):
        q, k, *_ = case(4, 1, 2, 1, 5, D, "f16", False)
        q[..., R:] = value
        q[..., R] = 1.0
        oq, _ = fa.rotary_embedding(q.cuda(), k.cuda(), fa.rotary_table(5, R).cuda(), interleaved=interleaved)
        assert torch.equal(oq[..., R:].cpu().view(torch.int16), q[..., R:].view(torch.int16))
        assert torch.isfinite(oq[..., :R]).all()


def test_weights_in_fp32_and_of_one_side():
    run(2, 4, 2, 50, 128, 64, "bf16", True, wdtype=torch.float32)
    for which in ((0,), (1,)):
        run(2, 4, 2, 50, 64, 64, "f16", True, which=which)
        run(2, 4, 2, 50, 20, 20, "f16", True, which=which)


def test_strides():
    """Parts of a joined projection, expanded gradients and heads out of order, with and without 16-byte alignment."""
    for pad, D in ((0, 64), (8, 64), (3, 64)):
        def lay(x):
            big = torch.empty(x.shape[0], x.shape[2], x.shape[1], D + pad, dtype=x.dtype)
            big[..., :D] = x.transpose(1, 2)
            return big.cuda()[..., :D].transpose(1, 2).detach()
        q, k, dq, dk, w = case(5, 2, 6, 2, 33, D, "bf16", True)
        table = fa.rotary_table(33, D).cuda()
        a = [lay(q).requires_grad_(), lay(k).requires_grad_()]
        b = [q.cuda().requires_grad_(), k.cuda().requires_grad_()]
        wd = [x.cuda() for x in w]
        oa, ob = (fa.rotary_embedding(*x, table, query_weight=wd[0], key_weight=wd[1], eps=EPS) for x in (a, b))
        for x, y in zip(oa, ob):
            assert (x.float() - y.float()).abs().max() <= 2 * ROUNDOFF[torch.bfloat16] * y.float().abs().max()
        # (one value expanded: its gradient has strides of 0)
        (oa[0].sum() + oa[1].sum()).backward()
        (ob[0].sum() + ob[1].sum()).backward()
        for x, y in zip(a, b):
            assert (x.grad.float() - y.grad.float()).abs().max() <= 2 * ROUNDOFF[torch.bfloat16] * y.grad.float().abs().max() + 1e-5


def test_gradient_against_differences():
    """In fp32, along random directions: (f(x + h u) - f(x - h u)) / 2 h.  With h = 2^-6 the differences' error of third order is h^2 / 6 times
    third derivatives (below 40 times a step's size: unit rows, weights near 1), and the fp32 outputs give 2^-22 / h."""
    q, k, dq, dk, w = case(6, 1, 2, 1, 9, 32, "f32", True)
    table = fa.rotary_table(9, 16).cuda()
    x = [t.cuda() for t in (q, k, *w)]
    g = [t.cuda() for t in (dq, dk)]

    def f(ts):
        out = fa.rotary_embedding(ts[0], ts[1], table, query_weight=ts[2], key_weight=ts[3], eps=EPS)
        return sum((o.double() * d.double()).sum() for o, d in zip(out, g))

    leaves = [t.clone().requires_grad_() for t in x]
    out = fa.rotary_embedding(leaves[0], leaves[1], table, query_weight=leaves[2], key_weight=leaves[3], eps=EPS)
    grads = torch.autograd.grad(out, leaves, g)
    h = 2.0 ** -6
    for i in range(4):
        u = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        up, down = ([t + s * h * u if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        diff = (f(up) - f(down)) / (2 * h)
        exact = (grads[i].double() * u.double()).sum()
        size = (grads[i].double() * u.double()).abs().sum() + 1
        assert (diff - exact).abs() <= (h * h * 40 / 6 + 2.0 ** -22 / h) * size


def test_what_needs_a_gradient():
    """Only what is asked for; an output that is not used; once, not twice; outputs that are changed."""
    q, k, dq, dk, w = case(7, 2, 4, 2, 20, 64, "f32", True)
    table = fa.rotary_table(20, 64).cuda()
    full = [t.cuda().requires_grad_() for t in (q, k, *w)]
    all_ = torch.autograd.grad(fa.rotary_embedding(full[0], full[1], table, query_weight=full[2], key_weight=full[3]), full, (dq.cuda(), dk.cuda()))
    for i in range(4):
        ts = [t.cuda().requires_grad_(j == i) for j, t in enumerate((q, k, *w))]
        out = fa.rotary_embedding(ts[0], ts[1], table, query_weight=ts[2], key_weight=ts[3])
        got, = torch.autograd.grad(out, [ts[i]], (dq.cuda(), dk.cuda()))
        assert torch.equal(got, all_[i])
    a = q.cuda().requires_grad_()
    only_k = fa.rotary_embedding(a, k.cuda().requires_grad_(), table)[1]
    only_k.sum().backward()
    assert (a.grad == 0).all()
    out = fa.rotary_embedding(a, k.cuda(), table)
    first, = torch.autograd.grad(out[0].square().sum(), [a], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward()
    with torch.no_grad():
        assert not fa.rotary_embedding(a, k.cuda(), table)[0].requires_grad
    x = q.cuda().requires_grad_()
    y = (x * 1.0)
    out = fa.rotary_embedding(y, k.cuda(), table, query_weight=w[0].cuda(), key_weight=w[1].cuda())
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        out[0].sum().backward()


def test_same_again():
    """The weights' gradients are the same every time, and do not depend on the number of tokens in flight."""
    q, k, dq, dk, w = case(8, 3, 16, 4, 700, 128, "bf16", True)
    table = fa.rotary_table(700, 128).cuda()
    runs = []
    for _ in range(2):
        ts = [t.cuda().requires_grad_() for t in (q, k, *w)]
        runs.append(torch.autograd.grad(fa.rotary_embedding(ts[0], ts[1], table, query_weight=ts[2], key_weight=ts[3]), ts, (dq.cuda(), dk.cuda())))
    assert all(torch.equal(x, y) for x, y in zip(*runs))


def test_positions_beyond_the_table():
    q, k, *_ = case(9, 1, 2, 1, 4, 64, "f16", False)
    table = fa.rotary_table(8, 32).cuda()
    pos = torch.tensor([0, 8, -1, 7], device="cuda")
    oq, ok = fa.rotary_embedding(q.cuda(), k.cuda(), table, pos)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="0x8"):
        fa.check_status()
    assert (oq[:, :, 1:3, :32] == 0).all() and torch.equal(oq[..., 32:].cpu(), q[..., 32:])
    good, _ = fa.rotary_embedding(q.cuda(), k.cuda(), table, pos.clamp(0, 7))
    assert torch.equal(oq[:, :, ::3], good[:, :, ::3])


def test_empty_and_refusals():
    q, k, *_ = (t.cuda() if isinstance(t, torch.Tensor) else t for t in case(10, 2, 4, 2, 8, 64, "f16", False))
    table = fa.rotary_table(8, 64).cuda()
    oq, ok = fa.rotary_embedding(q[:, :, :0].clone().requires_grad_(), k[:, :, :0], table)
    assert oq.shape == (2, 4, 0, 64)
    w = torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True)
    e = q[:, :, :0].clone().requires_grad_()
    fa.rotary_embedding(e, k[:, :, :0], table, query_weight=w)[0].sum().backward()
    assert (w.grad == 0).all()
    for args, kw, err in (((q.double(), k.double(), table), {}, ValueError), ((q, k.float(), table), {}, ValueError), ((q[0], k[0], table), {}, ValueError),
                          ((q, k[:, :, :4], table), {}, ValueError), ((q, k[..., :32], table), {}, ValueError), ((q, k, table.half()), {}, ValueError),
                          ((q, k, table[:4]), {}, ValueError), ((q, k, table[:, :33]), {}, ValueError), ((q, k, fa.rotary_table(8, 66).cuda()), {}, ValueError),
                          ((q, k, table, torch.zeros(2, 9, dtype=torch.int64, device="cuda")), {}, ValueError),
                          ((q, k, table, torch.zeros(8, device="cuda")), {}, ValueError), ((q, k, table), dict(query_weight=w[:32]), ValueError),
                          ((q, k, table), dict(query_weight=w.double()), ValueError), ((q, k, table), dict(eps=-1.0), ValueError),
                          ((q, k, table), dict(query_weight=w, key_weight=w.float()), ValueError), ((q.transpose(2, 3), k.transpose(2, 3), table), {}, ValueError),
                          ((q.cpu(), k, table), {}, RuntimeError), ((q, k, table.cpu()), {}, RuntimeError), ((q, k, 3), {}, TypeError),
                          ((q, k, table.clone().requires_grad_()), {}, ValueError),
                          ((torch.zeros(1, 1, 1, 300, device="cuda"),) * 2 + (None,), {}, fa._cabi.FlaxAttnError)):
        with pytest.raises(err):
            fa.rotary_embedding(*args, **kw)
    for kw in (dict(length=4, rotary_dim=3), dict(length=-1, rotary_dim=4), dict(length=4, rotary_dim=4, scaling="other"),
               dict(length=4, rotary_dim=4, scaling="by_parts"), dict(length=4, rotary_dim=2, scaling="ntk"), dict(length=4, rotary_dim=4, factor=0.0)):
        with pytest.raises(ValueError):
            fa.rotary_table(**kw)


# ---- rotary_append ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,Dv,R,page,norm,interleaved,bhln,token_major", [
    (32, 1, 32, 8, 128, 128, 128, 16, True, False, True, False), (1, 77, 8, 2, 64, 64, 64, 8, False, True, False, True),
    (3, 5, 4, 4, 96, 64, 32, 12, True, False, True, True), (2, 9, 3, 1, 20, 12, 10, 1, True, True, False, False),
    (1, 1, 1, 1, 64, 32, 0, 3, False, False, True, False), (1, 513, 4, 2, 64, 64, 48, 128, True, False, False, False)])
def test_append(dtype, B, S, Hq, Hkv, D, Dv, R, page, norm, interleaved, bhln, token_major):
    dt = DTYPES[dtype]
    q, k, _, _, w = case(11, B, Hq, Hkv, S, D, dtype, norm)
    v = normal(np.random.default_rng(12), B, Hkv, S, Dv, dtype=dt)
    pages = -(-B * S // page) + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[: B * S].view(B, S)
    slots[0, 0] = -1  # goes nowhere
    pos = torch.randint(0, 300, (B, S), dtype=torch.int32, generator=torch.Generator().manual_seed(2))
    table = fa.rotary_table(300, R, 1000.0)
    shape = lambda d: (pages, page, Hkv, d) if token_major else (pages, Hkv, page, d)  # noqa: E731
    kp, vp = (torch.full(shape(d), 7.0, dtype=dt, device="cuda") for d in (D, Dv))
    if token_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    lay = (lambda x: x.cuda()) if bhln else (lambda x: x.transpose(1, 2).contiguous().cuda())
    out = fa.rotary_append(lay(q), lay(k), lay(v), kp, vp, slots.cuda() if B > 1 else slots.cuda().view(-1), table.cuda() if R else None, pos.cuda(),
                           query_weight=None if not norm else w[0].cuda(), key_weight=None if not norm else w[1].cuda(), eps=EPS, interleaved=interleaved, bhln=bhln)
    out = out if bhln else out.transpose(1, 2)
    t = table.double()
    angle = torch.complex(t[:, : R // 2], t[:, R // 2:])[pos.long()][:, None] if R else None
    check(out, definition(q.double(), None if w[0] is None else w[0].double(), angle, R, interleaved), dt, 4)
    kd = definition(k.double(), None if w[1] is None else w[1].double(), angle, R, interleaved)
    want_k, want_v = torch.full((pages * page, Hkv, D), 7.0, dtype=torch.float64), torch.full((pages * page, Hkv, Dv), 7.0, dtype=dt)
    keep = slots.view(-1) >= 0
    want_k[slots.view(-1)[keep]] = kd.transpose(1, 2).reshape(B * S, Hkv, D)[keep]
    want_v[slots.view(-1)[keep]] = v.transpose(1, 2).reshape(B * S, Hkv, Dv)[keep]
    check(kp.transpose(1, 2).reshape(-1, Hkv, D), want_k, dt, 4)
    assert torch.equal(vp.transpose(1, 2).reshape(-1, Hkv, Dv).cpu(), want_v)
    torch.cuda.synchronize()
    fa.check_status()
    # the same as rotary_embedding gives, bit by bit; without queries
    same = fa.rotary_embedding(lay(q), lay(k), table.cuda() if R else None, pos.cuda(), query_weight=None if not norm else w[0].cuda(),
                               key_weight=None if not norm else w[1].cuda(), eps=EPS, interleaved=interleaved, bhln=bhln)
    assert torch.equal(out, same[0] if bhln else same[0].transpose(1, 2))
    before = kp.clone()
    assert fa.rotary_append(None, lay(k), lay(v), kp, vp, slots.cuda(), table.cuda() if R else None, pos.cuda(), key_weight=None if not norm else w[1].cuda(), eps=EPS,
                            interleaved=interleaved, bhln=bhln) is None
    assert torch.equal(before, kp)


def test_append_far_slots_and_bad_ones():
    """Slots whose place passes 2^31 values; one beyond the pages is left out and reported."""
    page, D = 64, 64
    n = (1 << 31) // (page * D) + 20
    pool = torch.zeros(n, 1, page, D, dtype=torch.float16, device="cuda")
    k = normal(np.random.default_rng(13), 1, 1, 3, D, dtype=torch.float16).cuda()
    v = normal(np.random.default_rng(14), 1, 1, 3, D, dtype=torch.float16).cuda()
    slots = torch.tensor([n * page - 1, 5, n * page], device="cuda")
    fa.rotary_append(None, k, v, pool[10:], pool[:-10], slots - 10 * page)
    torch.cuda.synchronize()
    with pytest.raises(fa._cabi.FlaxAttnError, match="0x10"):
        fa.check_status()
    # (key pages are the pool from page 10 on, value pages the pool up to 10 pages before its end)
    assert torch.equal(pool[n - 1, 0, page - 1], k[0, 0, 0]) and torch.equal(pool[n - 11, 0, page - 1], v[0, 0, 0])
    assert int((pool[n - 12:] != 0).any(-1).sum()) == 2


def test_append_refusals():
    q, k, *_ = (t.cuda() if isinstance(t, torch.Tensor) else t for t in case(15, 1, 4, 2, 8, 64, "f16", False))
    kp, vp = (torch.zeros(3, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.arange(8, device="cuda")
    call = lambda **kw: fa.rotary_append(**{**dict(query=q, key=k, value=k, key_pages=kp, value_pages=vp, slots=slots), **kw})  # noqa: E731
    version = kp._version
    call()
    assert kp._version > version  # (a change that autograd sees)
    for kw, err in ((dict(slots=slots.int()), ValueError), (dict(slots=slots[:7]), ValueError), (dict(value=k[:, :1]), ValueError), (dict(value=k.float()), ValueError),
                    (dict(key_pages=kp[:, :1], value_pages=vp[:, :1]), ValueError), (dict(value_pages=vp[:2]), ValueError), (dict(key_pages=kp.float()), ValueError),
                    (dict(query=q[:, :, :7]), ValueError), (dict(key=k.clone().requires_grad_()), ValueError), (dict(key_pages=kp[:1].expand(3, 2, 16, 64)), ValueError),
                    (dict(slots=slots.cpu()), RuntimeError), (dict(value=None), TypeError)):
        with pytest.raises(err):
            call(**kw)
    call(query=q[:, :, :0], key=k[:, :, :0], value=k[:, :, :0], slots=slots[:0])
    torch.cuda.synchronize()
    fa.check_status()


# ---- the table ----------------------------------------------------------------------------------------------------
def test_table():
    base, R, n = 500.0, 16, 5000
    freq = [base ** (-2 * i / R) for i in range(R // 2)]
    ntk = [(base * 4.0 ** (R / (R - 2))) ** (-2 * i / R) for i in range(R // 2)]
    parts = []
    for f in freq:
        turns = 1000 * f / (2 * math.pi)
        stay = min(max((turns - 1.0) / (4.0 - 1.0), 0.0), 1.0)
        parts.append(f * stay + f / 4.0 * (1 - stay))
    for kw, fs in ((dict(), freq), (dict(scaling="linear", factor=4.0), [f / 4 for f in freq]), (dict(scaling="ntk", factor=4.0), ntk),
                   (dict(scaling="by_parts", factor=4.0, original_length=1000, low=1.0, high=4.0), parts)):
        t = fa.rotary_table(n, R, base, magnitude=1.25, device="cuda", **kw)
        assert t.shape == (n, R) and t.dtype == torch.float32 and t.is_cuda
        for pos in (0, 1, 777, n - 1):
            want = [1.25 * math.cos(pos * f) for f in fs] + [1.25 * math.sin(pos * f) for f in fs]
            assert (t[pos].cpu().double() - torch.tensor(want, dtype=torch.float64)).abs().max() <= 2.0 ** -22
