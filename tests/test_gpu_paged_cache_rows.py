"""GPU: PagedCache with a slot map of more than 4096 rows (its page_map in two launches), eager and captured, and what a step
allocates."""

import random

import pytest
import torch

import test_gpu_paged_cache as S
from kvskip_amd.paged import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("pages", [40, 6])
def test_serving_many_rows(gpu, monkeypatch, fmt, captured, pages):
    monkeypatch.setattr(S, "ROWS", 4200)
    S.test_serving(gpu, fmt, captured, pages)


@pytest.mark.parametrize("rows,most", [(64, 0), (4096, 0), (4097, 1)])
def test_step_allocates(gpu, rows, most):
    """A step allocates nothing up to 4096 rows, and page_map's workspace above."""
    c = PagedCache(1, 16, 1, 64, 4, 256, rows, "int8")
    new, drop = torch.ones(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.bool, device="cuda")
    count = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]
    before = count()
    c.step(new, drop)
    assert count() - before == most


def test_a_step_over_many_pages(gpu):
    """256 requests whose prompts fill 8192 rows, one after another, then all of them end: every page comes back."""
    rng = random.Random(3)
    c = PagedCache(1, 400, 1, 64, 256, 128, 8192, "e4m3")
    left = [rng.randrange(1, 33) for _ in range(256)]
    new = torch.tensor(left, dtype=torch.int32, device="cuda")
    c.step(new)
    assert c.lens.tolist() == left and int(c.short) == 0
    held = [-(-n // 64) for n in left]
    assert c.held.tolist() == held and int(c.free_count) == 400 - sum(held)
    slots = c.slot_map.tolist()
    assert sorted(s for s in slots if s >= 0) == sorted(c.block_table[b, 0].item() * 64 + i for b in range(256) for i in range(left[b]))
    c.step(torch.zeros_like(new), torch.ones(256, dtype=torch.bool, device="cuda"))
    assert not c.lens.any() and not c.held.any() and int(c.free_count) == 400
    assert sorted(c.free_pages.tolist()) == list(range(400)) and (c.slot_map == -1).all()
