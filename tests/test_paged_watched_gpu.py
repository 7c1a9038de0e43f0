"""The operators around a paged cache work on tensors' memory behind torch's back: what would look on is told so, instead of seeing nothing."""
import pytest
import torch

import flaxattention_b200 as fa

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def calls():
    """name -> (call of one tensor, that tensor)"""
    x = torch.randn(1, 2, 4, 64, device="cuda", dtype=torch.float16)
    kp, vp = (torch.zeros(3, 2, 16, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    table = ints(0, 1)[None]
    return {"rotary_embedding": (lambda t: fa.rotary_embedding(t, x, None)[0], x),
            "rotary_append": (lambda t: fa.rotary_append(t, x, x, kp, vp, torch.arange(4, device="cuda")), x),
            "page_step": (lambda t: fa.page_step(t, ints(1), table, ints(2), 16, 1).lengths, ints(3)),
            "paged_attention": (lambda t: fa.paged_attention(t, kp, vp, table, ints(4)), x)}




def mode(f, t):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Mode():
        f(t)


def looking_on(f, t):
    class Logged(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            return super().__torch_function__(func, types, args, kwargs or {})

    f(t.as_subclass(Logged))


def fake(f, t):
    from torch._subclasses.fake_tensor import FakeTensorMode

    other = FakeTensorMode().from_tensor(t)
    f(other)


def dual(f, t):
    import torch.autograd.forward_ad as ad

    if not t.is_floating_point():
        raise NotImplementedError
    with ad.dual_level():
        f(ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("name", ["rotary_embedding", "rotary_append", "page_step", "paged_attention"])
@pytest.mark.parametrize("where", [mode, looking_on, fake, dual, lambda f, t: torch.jit.trace(f, (t,), check_trace=False), lambda f, t: torch.func.vmap(f)(t[None])],
                         ids=["mode", "subclass", "fake", "dual", "jit", "vmap"])
@pytest.mark.filterwarnings("ignore")
def test_refused(name, where):
    f, t = calls()[name]
    with torch.no_grad():
        f(t)
        seen = []

        def told(x):
            try:
                return f(x)
            except NotImplementedError as e:
                seen.append(e)
                raise

        with pytest.raises(Exception):
            where(told, t)
        assert seen or (where is dual and name == "page_step")


@pytest.mark.parametrize("name", ["rotary_embedding", "rotary_append", "page_step", "paged_attention"])
def test_taken(name):
    """Parameters, subclasses that change nothing, a default device, the profiler."""
    class Named(torch.Tensor):
        pass

    f, t = calls()[name]
    with torch.no_grad():
        want = f(t)
        if t.is_floating_point():
            assert torch.equal(f(torch.nn.Parameter(t)), want)
        assert torch.equal(f(t.as_subclass(Named)), want)
        with torch.device("cuda"):
            assert torch.equal(f(t), want)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
            assert torch.equal(f(t), want)
