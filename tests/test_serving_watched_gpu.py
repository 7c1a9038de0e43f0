"""read_pages, prompt_attention, and the scales and prefixes of the other calls: what would look on at a tensor is told so, instead of seeing nothing."""
import pytest
import torch

import flaxattention_b200 as fa
from test_paged_watched_gpu import dual, fake, ints, looking_on, mode

pytestmark = pytest.mark.gpu


def calls():
    """name -> (call of one tensor, that tensor)"""
    x = torch.randn(1, 2, 4, 64, device="cuda", dtype=torch.float16)
    kp, vp = (torch.zeros(3, 2, 16, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    k8, v8 = (torch.ones(3, 2, 16, 64, device="cuda", dtype=torch.int8) for _ in range(2))
    s = torch.ones(3, 2, 16, device="cuda")
    table, starts = ints(0, 1)[None], ints(0, 4)
    pre = torch.randn(1, 2, 40, 64, device="cuda", dtype=torch.float16)
    read = lambda k=k8, v=v8, t=table, b=starts, ks=s, vs=s: fa.read_pages(k, v, t, b, 4, key_scales=ks, value_scales=vs, dtype=torch.float16)[0]  # noqa: E731
    prompt = lambda q=x, k=x, v=x, b=starts, kb=starts: fa.prompt_attention(q, k, v, b, key_starts=kb)  # noqa: E731
    paged = lambda ks=s, vs=s, pk=pre, pv=pre: fa.paged_attention(x, k8, v8, table, ints(4), key_scales=ks, value_scales=vs, prefix=(pk, pv))  # noqa: E731
    append = lambda ks, vs=torch.ones_like(s): fa.rotary_append(x, x, x, k8.clone(), v8.clone(), torch.arange(4, device="cuda"), key_scales=ks, value_scales=vs)  # noqa: E731
    return {"read_pages-pages": (lambda t: fa.read_pages(t, vp, table, starts, 4)[0], kp), "read_pages-value_pages": (lambda t: read(v=t), v8), "read_pages-table": (lambda t: read(t=t), table),
            "read_pages-starts": (lambda t: read(b=t), starts), "read_pages-scales": (lambda t: read(ks=t), s), "read_pages-value_scales": (lambda t: read(vs=t), s),
            "prompt_attention-query": (lambda t: prompt(q=t), x), "prompt_attention-key": (lambda t: prompt(k=t), x), "prompt_attention-value": (lambda t: prompt(v=t), x),
            "prompt_attention-starts": (lambda t: prompt(b=t), starts), "prompt_attention-key_starts": (lambda t: prompt(kb=t), starts),
            "paged_attention-scales": (lambda t: paged(ks=t), s), "paged_attention-value_scales": (lambda t: paged(vs=t), s),
            "paged_attention-prefix": (lambda t: paged(pk=t), pre), "paged_attention-prefix_values": (lambda t: paged(pv=t), pre),
            "rotary_append-scales": (append, s.clone()), "rotary_append-value_scales": (lambda t: append(torch.ones_like(s), t), s.clone())}


NAMES = ["read_pages-pages", "read_pages-value_pages", "read_pages-table", "read_pages-starts", "read_pages-scales", "read_pages-value_scales", "prompt_attention-query", "prompt_attention-key",
         "prompt_attention-value", "prompt_attention-starts", "prompt_attention-key_starts", "paged_attention-scales", "paged_attention-value_scales", "paged_attention-prefix",
         "paged_attention-prefix_values", "rotary_append-scales", "rotary_append-value_scales"]


@pytest.mark.parametrize("name", NAMES)
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
        assert seen or (where is dual and not t.is_floating_point())


@pytest.mark.parametrize("name", NAMES)
def test_taken(name):
    """Parameters, subclasses that change nothing, a default device, the profiler."""
    class Named(torch.Tensor):
        pass

    f, t = calls()[name]
    with torch.no_grad():
        want = f(t)
        assert torch.isfinite(want).all()
        assert torch.equal(f(t.as_subclass(Named)), want)
        if t.is_floating_point() and not name.startswith("rotary_append"):  # (scales that are written take no gradient)
            assert torch.equal(f(torch.nn.Parameter(t)), want)
        with torch.device("cuda"):
            assert torch.equal(f(t), want)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
            assert torch.equal(f(t), want)
