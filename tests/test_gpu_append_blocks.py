"""append into a cache with block scales: what it reports of rows that do not stand together, and what drafts leave behind that are
dropped."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, PageTable, StepPlan, append, read

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


def test_a_dropped_step_leaves_its_scale(rng):
    """Drafts of a step that is not committed: the lengths stay, the scale that the drafts raised too, with the older rows rounded to
    it; a cache with a scale for each head holds what it held."""
    old, new = (torch.from_numpy(rng.standard_normal((n, 1, 64)).astype(np.float32)).to(BF).cuda() for n in (5, 2))

    def after(cache):
        pt = PageTable(1, 1, 1, 16)
        append(cache, pt.step(i32([5]), 5), old, old)
        before = cache.k.view(torch.uint8).clone()
        plan = pt.step(i32([7]), 2, commit=False)
        append(cache, plan, new * 1024, new * 1024)
        plan.check()
        assert pt.lens.item() == 5
        return before[0, 0, :5].cpu().view(E4M3), cache.k[0, 0, :5].cpu(), pt
    cache = KVCache(1, 16, 1, 64, 64, dtype=E4M3, k_scale=1.0, v_scale=1.0)
    before, now, _ = after(cache)
    assert torch.equal(before.view(torch.uint8), now.view(torch.uint8))
    cache = KVCache(1, 16, 1, 64, 64, dtype=E4M3, block_scales=True)
    first = KVCache(1, 16, 1, 64, 64, dtype=E4M3, block_scales=True)
    append(first, StepPlan(slots=i32(np.arange(5)), positions=i32(np.arange(5))), old, old)
    before, now, pt = after(cache)
    grown = cache.k_scale.item() - first.k_scale.item()
    assert grown > 5 and torch.equal((before.float() * 2.0 ** -grown).to(E4M3).view(torch.uint8), now.view(torch.uint8))
    # later tokens of the block have that scale too; a request that begins again has its own
    top = cache.k_scale.item()
    append(cache, pt.step(i32([6]), 1), old[:1], old[:1])
    assert cache.k_scale.item() == top
    pt.step(i32([0]), 0)
    append(cache, pt.step(i32([5]), 5), old, old)
    assert torch.equal(cache.k_scale, first.k_scale) and torch.equal(cache.k[0, 0, :5].view(torch.uint8), first.k[0, 0, :5].view(torch.uint8))
