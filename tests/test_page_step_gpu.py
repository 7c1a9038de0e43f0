"""page_step against the same in Python, request by request."""
import numpy as np
import pytest
import torch

import flaxattention_b200 as fa

pytestmark = pytest.mark.gpu


def step(lengths, new, table, free, page, num_tokens, taken):
    """The definition: (results, table) as lists."""
    table = [list(r) for r in table]
    positions, slots, requests, starts, out = [], [], [], [], []
    for b, (n, m) in enumerate(zip(lengths, new)):
        n, m = max(n, 0), max(m, 0)
        starts.append(len(positions))
        for i in range(-(-n // page), -(-(n + m) // page)):
            entry = free[taken] if taken < len(free) else -1
            if i < len(table[b]):
                table[b][i] = max(entry, -1)
            taken += 1
        for pos in range(n, n + m):
            entry = table[b][pos // page] if pos // page < len(table[b]) else -1
            positions.append(pos)
            requests.append(b)
            slots.append(-1 if entry < 0 else entry * page + pos % page)
        out.append(n + m)
    starts.append(len(positions))
    pad = max(num_tokens - len(positions), 0)
    cut = lambda x, fill: x[:num_tokens] + [fill] * pad  # noqa: E731
    return [out, cut(positions, 0), cut(slots, -1), cut(requests, -1), starts, [taken]], table


def run(lengths, new, page, width, free, taken=None, num_tokens=None, stride=0):
    B = len(lengths)
    rng = np.random.default_rng(7)
    table = rng.integers(0, 1000, (B, width))
    num_tokens = sum(max(x, 0) for x in new) if num_tokens is None else num_tokens
    ints = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device="cuda")  # noqa: E731
    big = torch.full((B, width + stride), 77, dtype=torch.int32, device="cuda")
    t = big[:, :width]
    t.copy_(torch.from_numpy(table))
    want, want_table = step(lengths, new, table.tolist(), list(free), page, num_tokens, taken or 0)
    for _ in range(2):  # (again, on what the first call has left: the same)
        got = fa.page_step(ints(lengths), ints(new), t, ints(free), page, num_tokens, None if taken is None else ints([taken]))
        for name, x, y in zip(got._fields, got, want):
            assert x.dtype == (torch.int64 if name == "slots" else torch.int32)
            assert x.tolist() == y, name
        assert t.tolist() == want_table
        assert (big[:, width:] == 77).all()
    torch.cuda.synchronize()
    fa.check_status()


@pytest.mark.parametrize("page", [1, 3, 16, 128])
@pytest.mark.parametrize("B", [1, 2, 31, 257, 1024, 1025, 2500])
def test_requests(page, B):
    rng = np.random.default_rng(B + page)
    lengths, new = rng.integers(0, 100, B), rng.integers(0, 12, B)
    run(lengths.tolist(), new.tolist(), page, 112 // page + 1, rng.permutation(20 * B + 5).tolist(), taken=3, stride=5)
    run(lengths.tolist(), [1] * B, page, 112 // page + 1, rng.permutation(2 * B).tolist())


def test_long_prompts():
    run([0, 5000, 17], [3000, 1, 9000], 16, 700, list(range(2000, 0, -1)))
    run([0], [1], 64, 1, [3])
    run([64], [64], 64, 2, [3])


def test_edges():
    run([0, 0, 5], [0, 0, 0], 4, 3, [1, 2])              # nothing new
    run([-3, 2, 4], [2, -5, 1], 4, 3, [1, 2, 3])         # below 0 counts as 0
    run([3, 4, 0], [6, 4, 9], 4, 8, [9, 8])              # the list is too short
    run([3, 4, 0], [6, 4, 9], 4, 8, [9, -2, 8, 7, 6, 5])  # an entry of it that is no page
    run([3, 4, 0], [6, 4, 9], 4, 8, [])                  # there is none
    run([3, 4, 0], [6, 4, 9], 4, 8, [9, 8, 7], taken=5)  # all taken
    run([3, 4, 0], [6, 4, 9], 4, 2, list(range(20)))     # the table is too narrow
    run([3, 4, 0], [6, 4, 9], 4, 0, list(range(20)))
    run([3, 4], [2, 3], 4, 4, list(range(20)), num_tokens=11)  # padding
    run([3, 4], [2, 9], 4, 4, list(range(20)), num_tokens=4)   # fewer tokens than there are
    run([3] * 1500, [3] * 1500, 1, 7, list(range(5000)), num_tokens=10)
    run([], [], 4, 3, [1], num_tokens=3)
    run([2 ** 31 - 5], [3], 2 ** 30, 2, [1, 2])


def test_refusals():
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = dict(lengths=i(1, 2), new_tokens=i(1, 1), block_table=torch.zeros(2, 3, dtype=torch.int32, device="cuda"), free_pages=i(4), page_size=16, num_tokens=2)
    version = args["block_table"]._version
    fa.page_step(**args)
    assert args["block_table"]._version > version
    for kw, err in ((dict(lengths=i(1)), ValueError), (dict(new_tokens=i(1, 1).long()), ValueError), (dict(block_table=args["block_table"][:1]), ValueError),
                    (dict(block_table=args["block_table"].long()), ValueError), (dict(block_table=args["block_table"][:1].expand(2, 3)), ValueError),
                    (dict(page_size=0), ValueError), (dict(num_tokens=-1), ValueError), (dict(num_tokens=2 ** 31), ValueError), (dict(free_pages=i(1, 2, 3, 4)[::2]), ValueError),
                    (dict(taken=i(1, 2)), ValueError), (dict(lengths=i(1, 2).cpu()), RuntimeError), (dict(page_size=1.5), TypeError), (dict(free_pages=None), TypeError)):
        with pytest.raises(err):
            fa.page_step(**{**args, **kw})
