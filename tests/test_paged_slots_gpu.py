"""GPU: slots of a paged cache where the counts say far more than the call has room for."""
import numpy as np
import pytest
import torch

from blockedattention_b200 import blockPagedSlots
from test_paged_gpu import check_slots, ints

pytestmark = pytest.mark.gpu


def by_pages(lengths, new, table, free, taken, size, tokens):
    """The definition page by page, and token by token only as far as there are slots."""
    table, slots, after = np.array(table, np.int64), [], []
    columns = table.shape[1]
    for r, (old, n) in enumerate(zip(lengths, new)):
        n = min(n, 2 ** 31 - 1 - old)
        for col in range(min(-(-old // size), columns), min(-(-(old + n) // size), columns)):
            table[r, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(old, min(old + n, old + tokens - len(slots))):
            page = table[r, p // size] if p // size < columns else -1
            slots.append(int(page) * size + p % size if page >= 0 else -1)
        after.append(old + n)
    return slots + [-1] * (tokens - len(slots)), after, taken, table


@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("size,columns", [(16, 5), (1, 40), (1 << 30, 2), (1 << 20, 3000)])
@pytest.mark.parametrize("requests,tokens", [(1, 7), (50, 0), (50, 300), (300, 5), (1500, 9000)])
def test_counts_far_beyond_the_slots(cuda_device, requests, tokens, size, columns, advance):
    """Counts of up to 2^31 - 1 tokens a request: every page is entered, and the call ends as soon as one with small counts."""
    rs = np.random.RandomState(requests + size % 1000)
    lengths = rs.randint(0, 60, requests)
    new = np.where(rs.rand(requests) < 0.3, rs.randint(0, 9, requests), 2 ** 31 - 1 - rs.randint(0, 99, requests))
    new[0] = 2 ** 31 - 1
    table = np.full((requests, columns), -9)
    free = rs.permutation(requests * columns // 2 + 4)
    want = by_pages(lengths.tolist(), new.tolist(), table, free, 2, size, tokens)
    args = [ints(lengths), ints(new), ints(table), ints(free), ints([2])]
    slots, after, used = blockPagedSlots(*args, size, tokens, advance=advance)
    assert slots.tolist() == want[0] and after.tolist() == want[1] and used.tolist() == [want[2]]
    assert np.array_equal(args[2].cpu().numpy(), want[3])


@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 700, 9000, 30000, 61000])
def test_some_slots_missing(cuda_device, tokens, advance):
    rs = np.random.RandomState(tokens)
    check_slots(rs.randint(0, 40, 2000), rs.randint(0, 60, 2000), 7, 16, tokens=tokens, advance=advance)
    check_slots(rs.randint(0, 40, 30), rs.randint(0, 4000, 30), 150, 32, tokens=tokens, spare=-900, advance=advance)
