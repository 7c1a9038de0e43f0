"""rotary_embedding where rows, norms and saved tensors are out of the ordinary."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import ROUNDOFF, normal
from _util import DTYPES
from test_rotary_gpu import run

pytestmark = pytest.mark.gpu


def definition(x, w, angle, eps):
    """x [.., S, D] in 64 bits with a norm, all of it rotated in halves; angle complex [S, D / 2]"""
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    z = torch.complex(x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]) * angle
    return torch.cat([z.real, z.imag], -1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,D", [(1, 128), (33, 128), (37, 64), (37, 80), (129, 256), (5, 20)])
def test_norm_without_eps(dtype, S, D):
    """eps 0, and numbers of tokens that no block divides: what lies beyond the last token takes no part in the weights' gradients."""
    rng, dt = np.random.default_rng(S + D), DTYPES[dtype]
    q, k, dq, dk = (normal(rng, 1, H, S, D, dtype=dt) for H in (3, 1, 3, 1))
    w = [(1 + 0.2 * normal(rng, D)).to(dt) for _ in range(2)]
    table = fa.rotary_table(S, D)
    t = table.double()
    angle = torch.complex(t[:, : D // 2], t[:, D // 2:])
    leaves = [x.cuda().requires_grad_() for x in (q, k, *w)]
    out = fa.rotary_embedding(leaves[0], leaves[1], table.cuda(), query_weight=leaves[2], key_weight=leaves[3], eps=0.0)
    got = torch.autograd.grad(out, leaves, (dq.cuda(), dk.cuda()))
    for i, (x, d) in enumerate(((q, dq), (k, dk))):
        ref = [x.double().requires_grad_(), w[i].double().requires_grad_()]
        want = torch.autograd.grad(definition(*ref, angle, 0.0), ref, d.double())
        # (the bounds of the tests with an eps: some fp32 roundings of the row's largest, or of as many as the sums' partial sums are)
        for g, r, bound in ((got[i], want[0], 2.0 ** -20 * (8 + D ** 0.5) * want[0].abs().amax(-1, keepdim=True)),
                            (got[2 + i], want[1], 2.0 ** -20 * (8 + 4 * (x.numel() // D) ** 0.5))):
            assert ((g.cpu().double() - r).abs() <= ROUNDOFF[dt] * r.abs() + bound + 2.0 ** -24).all()


@pytest.mark.parametrize("seed", [66, 67, 68])
def test_gradients_that_nearly_cancel(seed):
    """Two values in a row under a norm: their gradient is what two terms leave, of some rows next to nothing."""
    run(4, 33, 3, 64, 2, 2, "f32", norm=True, interleaved=True, bhln=False, seed=seed, which=(0,))
    run(4, 33, 3, 64, 2, 2, "f32", norm=True, seed=seed)
