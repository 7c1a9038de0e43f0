"""Kernels are launched while the one in front of them on the stream is finishing.  Each waits for it before its first access to global memory, whatever its compile-time
parameters are: only that wait makes what earlier kernels wrote visible, also what the kernel in front has itself waited for."""
import os
import re

import pytest

import flaxattention_b200

CSRC = os.path.join(os.path.dirname(os.path.abspath(flaxattention_b200.__file__)), "csrc")


def kernels():
    """(file, text of the body up to its first wait, whether there is one at the body's own level) of every kernel."""
    found = []
    for folder in (CSRC, os.path.join(CSRC, "kernels")):
        for name in sorted(os.listdir(folder)):
            if not name.endswith((".cu", ".cuh")):
                continue
            with open(os.path.join(folder, name)) as f:
                text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
            for m in re.finditer(r"__global__\b[^;{]*\{", text):
                at, depth, start = m.end(), 1, m.end()
                wait = re.compile(r"(if \([^;{}]*\) )?(?:fa_)?grid_wait\(\);|[{}]")
                ok = False
                while depth > 0:
                    w = wait.search(text, at)
                    at = w.end()
                    depth += {"{": 1, "}": -1}.get(w.group(), 0)
                    if "grid_wait" in w.group():
                        ok = depth == 1 and w.group(1) is None
                        break
                head = re.sub(r"\s+", " ", m.group())
                found.append(pytest.param(text[start:w.start()], ok, id=f"{name}-{re.findall(r'(\w+) ?[(]', head)[-1]}-{start}"))
    return found


@pytest.mark.parametrize("before,waits", kernels())
def test_every_kernel_waits_first(before, waits):
    assert waits, "no wait that every launch comes by, or not the first thing"
    # nothing read through the parameters' pointers, and written only where a launch does not fit and ends at once
    before = re.sub(r"if \([^{}]*\{[^{}]*FA_STATUS_BAD_LAUNCH[^{}]*return;\s*\}", "", before)
    assert not re.search(r"\b[pP]\.(p\.)?\w+(\.ptr)?\[|__ldg|atomic|\*\((const )?\w+ ?\*\)", before), before
