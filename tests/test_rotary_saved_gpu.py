"""rotary_embedding's backward on tensors that saved-tensor hooks have moved."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from _pages import normal

pytestmark = pytest.mark.gpu


def test_tensors_that_saved_tensor_hooks_give_back():
    """Moved to the host and back, the table and the positions lie in memory in another way than before; what is no longer the same is refused."""
    rng = np.random.default_rng(3)
    q, k, dq, dk = (normal(rng, 2, H, 33, 64).cuda() for H in (4, 2, 4, 2))
    w = [(1 + 0.2 * normal(rng, 64)).cuda() for _ in range(2)]
    wide = torch.full((50, 160), float("nan"), device="cuda")
    wide[:, 96:128] = fa.rotary_table(50, 32).cuda()
    table = wide[:, 96:128]
    every = torch.full((2, 33, 3), 10 ** 6, dtype=torch.int32, device="cuda")
    every[:, :, 1] = torch.randint(0, 50, (2, 33), generator=torch.Generator().manual_seed(1)).int().cuda()
    for positions in (None, every[:, :, 1], every[0, :, 1], every[:1, :, 1].expand(2, 33)):
        for weights in ((None, None), w):
            leaves = [t.clone().requires_grad_() for t in (q, k, *(x for x in weights if x is not None))]

            def grads(pack, unpack):
                with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                    out = fa.rotary_embedding(leaves[0], leaves[1], table, positions, query_weight=leaves[2] if len(leaves) > 2 else None,
                                              key_weight=leaves[3] if len(leaves) > 2 else None)
                return torch.autograd.grad(out, leaves, (dq, dk))

            want = grads(lambda t: t, lambda t: t)
            for unpack in (lambda t: t.cuda(), lambda t: t.contiguous().cuda()):
                got = grads(lambda t: t.cpu(), unpack)
                assert all(torch.equal(x, y) for x, y in zip(want, got))
            with torch.autograd.graph.save_on_cpu():
                out = fa.rotary_embedding(leaves[0], leaves[1], table, positions)
            plain = torch.autograd.grad(out, leaves[:2], (dq, dk))
            again = torch.autograd.grad(fa.rotary_embedding(leaves[0], leaves[1], table, positions), leaves[:2], (dq, dk))
            assert all(torch.equal(x, y) for x, y in zip(plain, again))
            for spoil in (lambda t: t.cpu(), lambda t: t[..., :-1], lambda t: t.double()):
                with pytest.raises(RuntimeError, match="another shape, type or device"):
                    grads(lambda t: t, spoil)
    torch.cuda.synchronize()
    fa.check_status()
