"""Host-side checks of the entry points for prompts, prefixes and 8-bit pages that need no GPU: arguments are refused before CUDA is touched, workspaces are as large as
said, and the kernels compile."""
import ctypes as C

import numpy as np
import pytest
import torch

import flaxattention_b200 as fa
from flaxattention_b200 import _cabi, modtrace


def tensor(ptr=0x1000, b=1 << 20, h=1 << 12, s=64):
    return _cabi.FaTensor(ptr, b, h, s)


def prompt(**kw):
    p = _cabi.FaPromptParams()
    p.dtype, p.B, p.Hq, p.Hkv, p.D, p.Dv, p.tokens, p.keys, p.scale, p.window = 0, 2, 4, 2, 64, 64, 100, 100, 0.125, -1
    p.q, p.k, p.v, p.o = tensor(), tensor(), tensor(), tensor()
    p.starts = 0x2000
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -1), (dict(B=-1), -1), (dict(Hq=0), -1), (dict(Hkv=3), -1), (dict(tokens=-1), -1), (dict(keys=-1), -1), (dict(D=60), -4), (dict(D=272, Dv=16), -4), (dict(Dv=80), -1),
    (dict(tokens=1 << 31), -4), (dict(B=(1 << 30) + 1), -4), (dict(tokens=1 << 30, Hq=8), -4), (dict(keys=1 << 31), -4), (dict(starts=None), -1), (dict(q=tensor(0x1008)), -1), (dict(o=tensor(None)), -1),
    (dict(k=tensor(s=63)), -1), (dict(v=tensor(None)), -1)])
def test_prompt_arguments(kw, code):
    L, m = _cabi.lib(), _cabi.Module(None)
    assert L.fa_prompt(m.handle, C.byref(prompt(**kw)), 0x8000, 1 << 40, None) == code, L.fa_last_error()


def test_prompt_nothing_to_do_and_workspace():
    L, m = _cabi.lib(), _cabi.Module(None)
    assert L.fa_prompt(m.handle, C.byref(prompt(tokens=0)), None, 0, None) == 0
    assert L.fa_prompt(None, C.byref(prompt()), None, 0, None) == L.fa_prompt(m.handle, None, None, 0, None) == -1
    assert L.fa_prompt(m.handle, C.byref(prompt()), 0x8004, 1 << 40, None) == -1
    assert L.fa_prompt_workspace_bytes(C.byref(prompt())) == L.fa_prompt_workspace_bytes(None) == 0
    # few rows over many keys are split: float32 sums of every row and part
    few = prompt(B=1, tokens=16, keys=40000)
    need = L.fa_prompt_workspace_bytes(C.byref(few))
    assert need % (16 * 4 * (64 + 2) * 4) == 0 and need > 0
    assert L.fa_prompt_workspace_bytes(C.byref(prompt(B=1, tokens=16, keys=40000, flags=16))) == 0
    assert L.fa_prompt_workspace_bytes(C.byref(prompt(B=1, tokens=16, keys=40000, window=100))) == 0


def read(**kw):
    p = _cabi.FaReadParams()
    p.dtype, p.B, p.Hkv, p.D, p.Dv, p.num_tokens, p.num_pages, p.page_size, p.table_width, p.block_table_stride = 0, 2, 2, 64, 64, 50, 8, 16, 4, 4
    p.k_pages, p.v_pages, p.k, p.v = tensor(), tensor(), tensor(), tensor()
    p.block_table, p.starts = 0x2000, 0x3000
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -1), (dict(B=-1), -1), (dict(D=0), -1), (dict(D=257), -4), (dict(Hkv=65536), -4), (dict(num_tokens=-1), -1), (dict(num_tokens=1 << 31), -4), (dict(num_pages=1 << 31), -4),
    (dict(page_size=0), -1), (dict(table_width=-1), -1), (dict(k_scales=tensor()), -1), (dict(k=tensor(None)), -1), (dict(v_pages=tensor(None)), -1), (dict(starts=None), -1),
    (dict(block_table=None), -1), (dict(num_tokens=0), 0), (dict(Hkv=0), 0)])
def test_read_arguments(kw, code):
    assert _cabi.lib().fa_read_pages(C.byref(read(**kw)), None) == code, _cabi.lib().fa_last_error()
    assert _cabi.lib().fa_read_pages(None, None) == -1


def paged(**kw):
    p = _cabi.FaPagedParams()
    p.dtype, p.B, p.Hq, p.Hkv, p.Sq, p.D, p.Dv, p.scale = 0, 2, 4, 2, 1, 64, 64, 0.125
    p.q, p.o, p.k_pages, p.v_pages = tensor(), tensor(), tensor(), tensor()
    p.num_pages, p.page_size, p.block_table, p.block_table_stride, p.table_width, p.lengths, p.window = 8, 16, 0x2000, 4, 4, 0x3000, -1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(k_scales=tensor()), -1), (dict(k_scales=tensor(), v_scales=tensor(), dtype=2), -4), (dict(k_scales=tensor(), v_scales=tensor(), k_pages=tensor(s=72)), -1),
    (dict(prefix_length=-1), -1), (dict(prefix_length=10), -1), (dict(prefix_length=10, k_prefix=tensor(), v_prefix=tensor(0x1004)), -1),
    (dict(prefix_length=(1 << 23) + 1, k_prefix=tensor(), v_prefix=tensor()), -4)])
def test_paged_arguments(kw, code):
    L, m = _cabi.lib(), _cabi.Module(None)
    assert L.fa_paged(m.handle, C.byref(paged(**kw)), 0x8000, 1 << 40, None) == code, L.fa_last_error()


def test_prefix_workspace():
    """The sums of every part, and of the pages."""
    L, m = _cabi.lib(), _cabi.Module(None)
    kw = dict(k_prefix=tensor(), v_prefix=tensor())
    own, with_prefix = (L.fa_paged_workspace_bytes(C.byref(paged(prefix_length=n, **kw))) for n in (0, 5000))
    assert with_prefix > own + 2 * 2 * 4 * 64 * 4
    assert L.fa_paged(m.handle, C.byref(paged(prefix_length=5000, **kw)), 0x8000, 100, None) == -5


def test_workspace_of_impossible_heads():
    """Fewer query heads than kv heads: refused by the call, and nothing is divided by their quotient before."""
    p = paged(Hq=2, Hkv=4, prefix_length=500, k_prefix=tensor(), v_prefix=tensor())
    assert _cabi.lib().fa_paged_workspace_bytes(C.byref(p)) >= 0
    m = _cabi.Module(None)
    assert _cabi.lib().fa_paged(m.handle, C.byref(p), None, 0, None) == -1


@pytest.mark.parametrize("D,Sq", [(64, 1), (128, 1), (256, 1), (128, 5), (64, 9), (96, 20), (80, 2)])
@pytest.mark.parametrize("prefix", [0, 500])
def test_eight_bit_kernels_with_capped_scores_compile(D, Sq, prefix):
    m = _cabi.Module(modtrace.lower_mods(lambda s, b, h, q, k: 30.0 * torch.tanh(s / 30.0), None).source)
    p = paged(D=D, Dv=D, Sq=Sq, page_size=16, k_scales=tensor(), v_scales=tensor(), prefix_length=prefix, k_prefix=tensor(), v_prefix=tensor())
    _cabi.check(_cabi.lib().fa_paged_prepare(m.handle, C.byref(p)))


def test_append_arguments():
    p = _cabi.FaRotaryParams()
    p.B, p.S, p.Hq, p.Hkv, p.D, p.Dv, p.eps = 1, 4, 2, 2, 64, 64, 1e-6
    for n in ("q", "k", "q_out", "k_out", "v", "k_pages", "v_pages"):
        setattr(p, n, tensor())
    p.slots, p.num_pages, p.page_size = 0x3000, 4, 16
    p.k_scales = tensor()
    assert _cabi.lib().fa_rotary_append(C.byref(p), None) == -1
    p.v_scales, p.dtype, p.weight_dtype = tensor(), 2, 2
    assert _cabi.lib().fa_rotary_append(C.byref(p), None) == -4


@pytest.mark.parametrize("dtype,D,Dv", [(0, 64, 64), (1, 128, 128), (1, 80, 48), (2, 64, 64), (0, 256, 256), (2, 256, 16)])
def test_prompt_kernels_compile(dtype, D, Dv):
    m = _cabi.Module(None)
    _cabi.check(_cabi.lib().fa_prompt_prepare(m.handle, C.byref(prompt(dtype=dtype, D=D, Dv=Dv))))


@pytest.mark.parametrize("D,Sq,page,prefix", [(64, 1, 16, 0), (128, 6, 16, 0), (96, 9, 6, 0), (256, 1, 16, 0), (64, 1, 16, 5000), (128, 1, 16, 50)])
def test_eight_bit_kernels_compile(D, Sq, page, prefix):
    p = paged(D=D, Dv=D, Sq=Sq, page_size=page, k_scales=tensor(), v_scales=tensor(), prefix_length=prefix, k_prefix=tensor(), v_prefix=tensor())
    m = _cabi.Module(None)
    _cabi.check(_cabi.lib().fa_paged_prepare(m.handle, C.byref(p)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="says what happens without a GPU")
@pytest.mark.parametrize("dtype,D", [(0, 64), (1, 128), (1, 256), (2, 64)])
def test_capped_scores_with_a_tensor_compile(dtype, D):
    """What stands in front of the mods must not keep the kernels from seeing that these read a tensor (the mods' text says so to the compiler)."""
    bias = torch.zeros(8, 4)
    mods = modtrace.lower_mods(lambda s, b, h, qi, ki: 30.0 * torch.tanh(s / 30.0) + bias[b, h], None)
    assert "FA_SCORE_PAIRS" in mods.source
    m = _cabi.Module(mods.source)
    _cabi.check(_cabi.lib().fa_prompt_prepare(m.handle, C.byref(prompt(dtype=dtype, D=D, Dv=D))))


def test_scores_of_two_keys_at_once():
    """Only where a tanh of the score is between sums and products; nothing that decides."""
    def pairs(f):
        return "FA_SCORE_PAIRS" in modtrace.lower_mods(f, None).source

    assert pairs(lambda s, b, h, q, k: 30.0 * torch.tanh(s / 30.0))
    assert pairs(lambda s, b, h, q, k: -torch.tanh(s) * 3.0 + (q - k) * 0.5)
    assert not pairs(lambda s, b, h, q, k: s * 2.0)
    assert not pairs(lambda s, b, h, q, k: s + (q - k) * 0.5)
    assert not pairs(lambda s, b, h, q, k: torch.where(q > k, 30.0 * torch.tanh(s / 30.0), s))
    assert not pairs(lambda s, b, h, q, k: torch.exp(torch.tanh(s)))
    assert not pairs(lambda s, b, h, q, k: torch.tanh(s / (h + 1)))


def test_there_is_no_cpu_path():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    starts = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fa.prompt_attention(q, q, q, starts)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fa.read_pages(q, q, starts[None], starts, 4)


def test_quotients_are_those_of_a_division():
    """What rotary_append does for a quotient (the product with the rounded reciprocal, and once more with what that left), in numpy, against fp32 divisions: scales of any size, values on
    and next to ties of their whole numbers."""
    rng = np.random.default_rng(0)
    n = 400_000
    scale = np.exp(rng.uniform(np.log(1e-30), np.log(1e30), n)).astype(np.float32)
    y = (rng.uniform(-127.4, 127.4, n) * scale.astype(np.float64)).astype(np.float32)
    half = n // 2
    y[:half] = ((rng.integers(-127, 127, half) + 0.5) * scale[:half].astype(np.float64)).astype(np.float32)
    y[: half // 2] = np.nextafter(y[: half // 2], np.float32(0))

    def fma(a, b, c):  # (a product of two fp32 is exact in 80 bits, and sums of what cancels nearly are too)
        return (np.longdouble(a) * np.longdouble(b) + np.longdouble(c)).astype(np.float32)

    r = np.float32(1) / scale
    q = y * r
    got = fma(fma(-scale, q, y), r, q)
    assert (got == y / scale).all()
    top = np.exp(rng.uniform(np.log(8e-31), np.log(3e38), n)).astype(np.float32)
    r = np.float32(1) / np.float32(127)
    q = top * r
    assert (fma(fma(np.full_like(top, -127), q, top), np.full_like(top, r), q) == top / np.float32(127)).all()
