"""append into a cache with block scales: what it reports of rows that do not stand together, and values that are not finite in
blocks that several waves share."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, StepPlan, append, read

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF = torch.bfloat16


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# 8 K/V heads: a block of threads looks at 1, 2, 4, 8 and 16 rows
@pytest.mark.parametrize("N", [40, 600, 1100, 2100, 4200])
@pytest.mark.parametrize("piece", [1, 2, 8, 15])
def test_a_parted_block_is_reported(N, piece):
    """A block of slots whose rows 1 to 15 others part, wherever in the call it stands; and none where nothing parts it."""
    heads, page = 8, 16
    n_pages = N // 16 + 4
    cache = KVCache(n_pages, page, heads, 64, 64, dtype=E4M3, block_scales=True)
    rows = torch.ones(N, heads, 64, dtype=BF, device="cuda")
    slots = np.arange(N) + 32                              # pages 0 and 1 are for the block in two pieces and what parts it
    parted = list(range(piece - 1, -1, -1)) + [15]         # the last slot of page 0 behind the others
    at = i32(np.arange(N))

    def status(order):
        plan = StepPlan(slots=i32(order), positions=at, status=word())
        append(cache, plan, rows, rows)
        return plan.status.item()
    for gap in (0, 1, 9, 14, 15):
        for first in (0, 5, N - piece - gap - 1):
            order = slots.copy()
            order[first:first + piece + gap + 1] = parted[:piece] + list(range(16, 16 + gap)) + parted[piece:]
            # the filler's own blocks, where the pieces stand amid one
            inside = first % 16 != 0 and first + piece + gap + 1 < N
            if inside:
                order[:first] = -1
                order[first + piece + gap + 1:first + 64] = -1
            assert (status(order) != 0) == (gap > 0), (first, gap)
    assert (read(cache, i32(np.arange(16, 31)))[0] == 1.0).all()
