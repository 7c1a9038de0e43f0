"""page_step where the new tokens of a batch add up to more than 31 or 32 bits hold: numbers that only the device sees, and that no
batch means, but what they lead to stays within the call's tensors."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def definition(lengths, new, table, free, page, num_tokens, taken):
    """In whole numbers of any size; no more tokens and columns are gone through than there are entries for."""
    table = table.copy()
    positions, slots, requests, starts, out = [], [], [], [], []
    at = 0
    for b, (n, m) in enumerate(zip(lengths.tolist(), new.tolist())):
        n, m = max(n, 0), max(m, 0)
        m = min(m, MOST - n)
        had, need = -(-n // page), -(-(n + m) // page)
        starts.append(min(at, MOST))
        for c in range(had, min(need, table.shape[1])):
            i = taken + c - had
            table[b, c] = max(free[i], -1) if i < len(free) else -1
        taken += need - had
        for pos in range(n, n + min(m, max(num_tokens - at, 0))):
            entry = table[b, pos // page] if pos // page < table.shape[1] else -1
            positions.append(pos)
            requests.append(b)
            slots.append(-1 if entry < 0 else int(entry) * page + pos % page)
        out.append(n + m)
        at += m
    starts.append(min(at, MOST))
    pad = num_tokens - len(positions)
    return [out, positions + [0] * pad, slots + [-1] * pad, requests + [-1] * pad, starts, [min(taken, MOST)]], table


@pytest.mark.parametrize("page", [1, 16, 1 << 20])
@pytest.mark.parametrize("large", [(10, 11), (1022, 1023), (3, 500, 1000), (0, 1024, 2048), (1500, 1501, 1502), (5,)])
@pytest.mark.parametrize("num_tokens", [0, 10, 5000, 200000])
def test_sums_beyond_31_bits(page, large, num_tokens):
    rng = np.random.default_rng(page + len(large) + num_tokens)
    B, width = 2500, 7
    lengths, new = rng.integers(0, 60, B).astype(np.int32), rng.integers(0, 9, B).astype(np.int32)
    new[list(large)] = MOST - rng.integers(0, 3, len(large))
    table, free = rng.integers(0, 1000, (B, width)).astype(np.int32), rng.permutation(1500).astype(np.int32)
    want, want_table = definition(lengths, new, table, free, page, num_tokens, 7)
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    t = dev(table)
    for _ in range(2):
        got = fa.page_step(dev(lengths), dev(new), t, dev(free), page, num_tokens, torch.tensor([7], dtype=torch.int32, device="cuda"))
        for name, x, y in zip(got._fields, got, want):
            assert x.tolist() == y, name
        assert np.array_equal(t.cpu().numpy(), want_table)
