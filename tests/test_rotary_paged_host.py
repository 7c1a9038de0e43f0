"""Host-side checks of the rotary and page entry points that need no GPU: arguments are refused before CUDA is touched, workspaces
are as large as said, and the kernels compile."""
import ctypes as C

import pytest
import torch

import flaxattention_b200 as fa
from flaxattention_b200 import _cabi


def tensor(ptr=0x1000, b=1 << 20, h=1 << 12, s=64):
    return _cabi.FaTensor(ptr, b, h, s)


def rotary(**kw):
    p = _cabi.FaRotaryParams()
    p.B, p.S, p.Hq, p.Hkv, p.D, p.Dv, p.rotary_dim, p.eps = 1, 4, 2, 2, 64, 64, 64, 1e-6
    for n in ("q", "k", "q_out", "k_out", "v", "k_pages", "v_pages"):
        setattr(p, n, tensor())
    p.table, p.table_length, p.table_stride = 0x2000, 4, 64
    p.slots, p.num_pages, p.page_size = 0x3000, 4, 16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=5), -1, "dtype"), (dict(weight_dtype=1), -1, "weights"), (dict(B=-1), -1, "negative"), (dict(B=1 << 20, S=1 << 12), -4, "2^31"),
    (dict(Hq=65535), -4, "65535"), (dict(D=257, rotary_dim=0), -4, "256"), (dict(rotary_dim=3), -1, "even"), (dict(rotary_dim=66), -1, "even"),
    (dict(table=None), -1, "table"), (dict(table_length=0), -1, "table"), (dict(table_stride=32), -1, "table"),
    (dict(positions=0x10, position_bits=16), -1, "positions"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"), (dict(k=tensor(None)), -1, "null")])
def test_rotary_arguments(kw, code, frag):
    L = _cabi.lib()
    p = rotary(**kw)
    t = tensor()
    calls = [lambda: L.fa_rotary(C.byref(p), None), lambda: L.fa_rotary_append(C.byref(p), None)]
    if "k" not in kw:
        calls.append(lambda: L.fa_rotary_bwd(C.byref(p), *([C.byref(t)] * 4), None, None, None, 0, None))
    for call in calls:
        assert call() == code
        assert frag in L.fa_last_error().decode()


def test_rotary_backward_and_append_arguments():
    L = _cabi.lib()
    t = tensor()
    p = rotary(q_weight=0x5000)
    assert L.fa_rotary_bwd_workspace_bytes(C.byref(rotary())) == 0
    need = L.fa_rotary_bwd_workspace_bytes(C.byref(p))
    assert need >= 64 * 4
    assert L.fa_rotary_bwd(C.byref(p), *([C.byref(t)] * 4), None, None, 0x6000, need - 1, None) == -5
    assert L.fa_rotary_bwd(C.byref(p), *([C.byref(t)] * 4), None, None, 0x6004, need, None) == -1
    assert L.fa_rotary_bwd(C.byref(p), *([C.byref(t)] * 4), None, 0x7000, 0x6000, need, None) == -1  # no key weight to have a gradient
    assert L.fa_rotary_bwd(C.byref(p), None, *([C.byref(t)] * 3), None, None, 0x6000, need, None) == -1
    for kw in (dict(page_size=0), dict(num_pages=-1), dict(num_pages=1 << 62), dict(slots=None), dict(v=tensor(None)), dict(k_pages=tensor(None)), dict(q_out=tensor(None))):
        assert L.fa_rotary_append(C.byref(rotary(**kw)), None) == -1, kw
    assert L.fa_rotary_append(C.byref(rotary(Dv=0)), None) == -4
    assert L.fa_rotary(None, None) == L.fa_rotary_append(None, None) == -1


def paged(**kw):
    p = _cabi.FaPagedParams()
    p.dtype, p.B, p.Hq, p.Hkv, p.Sq, p.D, p.Dv, p.scale = 0, 2, 4, 2, 1, 64, 64, 0.125
    p.q, p.o, p.k_pages, p.v_pages = tensor(), tensor(), tensor(), tensor()
    p.num_pages, p.page_size, p.block_table, p.block_table_stride, p.table_width, p.lengths, p.window = 8, 16, 0x2000, 4, 4, 0x3000, -1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -1), (dict(B=0), -1), (dict(Hkv=3), -1), (dict(D=60), -4), (dict(D=272, Dv=16), -4), (dict(Dv=80), -1), (dict(Sq=(1 << 20) + 1), -4), (dict(page_size=0), -1),
    (dict(num_pages=-1), -1), (dict(num_pages=1 << 31), -4), (dict(lengths=None), -1), (dict(block_table=None), -1), (dict(q=tensor(0x1008)), -1), (dict(o=tensor(None)), -1),
    (dict(k_pages=tensor(s=63)), -1), (dict(v_pages=tensor(None)), -1), (dict(B=1 << 16, Hq=1 << 15, Hkv=1 << 15), -4), (dict(table_width=1 << 27, B=1 << 10), -4)])
def test_paged_arguments(kw, code):
    L = _cabi.lib()
    m = _cabi.Module(None)
    assert L.fa_paged(m.handle, C.byref(paged(**kw)), 0x8000, 1 << 40, None) == code, L.fa_last_error()


def test_paged_workspace_and_module():
    L = _cabi.lib()
    m = _cabi.Module(None)
    p = paged(table_width=4096)
    need = L.fa_paged_workspace_bytes(C.byref(p))
    assert need >= 148 * 2 * 16 * (64 + 2) * 4 + 3 * 4
    assert L.fa_paged(m.handle, C.byref(p), 0x8000, need - 1, None) == -5
    assert L.fa_paged(m.handle, C.byref(p), None, need, None) == -5
    assert L.fa_paged(m.handle, C.byref(p), 0x8008, need, None) == -1
    assert L.fa_paged(None, C.byref(p), 0x8000, need, None) == L.fa_paged(m.handle, None, 0x8000, need, None) == -1


@pytest.mark.parametrize("dtype,D,Dv,Sq,page", [(0, 64, 64, 1, 16), (1, 128, 128, 4, 12), (2, 80, 16, 1, 1), (1, 256, 256, 40, 64)])
def test_paged_kernels_compile(dtype, D, Dv, Sq, page):
    from flaxattention_b200.modtrace import lower_mods
    L = _cabi.lib()
    m = _cabi.Module(lower_mods(lambda s, b, h, q, kv: s - (q - kv) * 0.5, lambda b, h, q, kv: (q + kv) % 2 == 0).source)
    _cabi.check(L.fa_paged_prepare(m.handle, C.byref(paged(dtype=dtype, D=D, Dv=Dv, Sq=Sq, page_size=page))))
    assert L.fa_paged_prepare(m.handle, C.byref(paged(D=20))) == -1


def test_page_step_arguments():
    L = _cabi.lib()
    good = dict(lengths=1, new=1, B=2, table=1, stride=4, width=4, free=1, num_free=3, taken=None, page=16, tokens=2, out=1, pos=1, slots=1, req=1, starts=1, out_taken=1)

    def call(**kw):
        return L.fa_page_step(*{**good, **kw}.values(), None)

    for kw in (dict(B=-1), dict(width=-1), dict(num_free=-1), dict(tokens=-1), dict(page=0), dict(lengths=None), dict(new=None), dict(out=None), dict(starts=None),
               dict(out_taken=None), dict(pos=None), dict(slots=None), dict(req=None), dict(table=None), dict(free=None)):
        assert call(**kw) == -1, kw
    assert call(tokens=1 << 31) == -4


@pytest.mark.skipif(torch.cuda.is_available(), reason="without a GPU")
def test_fails_loudly_without_cuda():
    x, i = torch.zeros(1, 2, 4, 64), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: fa.rotary_embedding(x, x, None), lambda: fa.rotary_append(x, x, x, x, x, torch.zeros(4, dtype=torch.int64)),
                 lambda: fa.page_step(i, i, i[None], i, 16, 2), lambda: fa.paged_attention(x, x, x, i[None], i)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_table_needs_no_gpu():
    t = fa.rotary_table(10, 8)
    assert t.shape == (10, 8) and t.dtype == torch.float32 and (t[0, :4] == 1).all() and (t[0, 4:] == 0).all()
