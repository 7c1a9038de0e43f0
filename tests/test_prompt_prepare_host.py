"""fa_prompt_prepare compiles what a call runs, also the general kernel, which short prompts and strides without a tensor map take where the tcgen05 one would do."""
import ctypes as C
import os

import pytest

from flaxattention_b200 import _cabi
from test_serving_host import prompt


@pytest.mark.parametrize("D,dtype", [(64, 0), (128, 1)])
@pytest.mark.parametrize("tokens,keys", [(100, 100), (60000, 60000), (16, 40000), (0, 0)])
def test_the_general_kernel_is_there(tmp_path, D, dtype, tokens, keys):
    L = _cabi.lib()
    L.fa_set_cache_dir(str(tmp_path).encode())
    try:
        def prepare(**kw):
            m = _cabi.Module(None)
            _cabi.check(L.fa_prompt_prepare(m.handle, C.byref(prompt(dtype=dtype, D=D, Dv=D, tokens=tokens, keys=keys, **kw))))
            return set(os.listdir(tmp_path))

        first = prepare()
        assert prepare(flags=16) == first and len(first) > 1  # (FA_FLAG_GENERAL_KERNELS: nothing that was not there)
    finally:
        L.fa_set_cache_dir(os.path.join(os.path.dirname(_cabi.LIB_PATH), "_kernel_cache").encode())
