"""GPU: plans over fewer rows than a step brings: the rows that are there keep their positions and their results."""

import pytest
import torch

from attend_side import Step, check
from kvskip_amd.paged import PagedCache

pytestmark = pytest.mark.gpu


def first_rows(s, rows):
    """The step without the rows from `rows` on."""
    s.rows, s.q = rows, s.q[:rows]
    return s


@pytest.mark.parametrize("rows", [1, 5, 63, 64, 100, 129, 191])
@pytest.mark.parametrize("shared", [False, True])
def test_rows_that_are_left_out(gpu, rows, shared):
    kw = dict(shared=[100], of=[0, -1, 0, 0]) if shared else {}
    s = Step([(70, 64), (150, 1), (200, 64), (90, 63)], 8, 2, 128, "e4m3", 31, prefix=[0, 60, 30, 0], **kw)
    pos, ref = s.positions(), [x[:rows] for x in s.exact(window=90)]
    first_rows(s, rows)
    p = s.plan(window=90)
    assert p.positions.tolist() == pos[:rows]
    check(s.call(p), ref, 128, rows)


def test_rows_before_the_first(gpu):
    """starts below 0: the rows from 0 on are the request's later ones."""
    s = Step([(150, 80), (30, 30)], 8, 2, 64, "int8", 32)
    pos, ref = s.positions(), [x[50:] for x in s.exact()]
    s.starts, s.rows, s.q = [x - 50 for x in s.starts], s.rows - 50, s.q[50:]
    p = s.plan()
    assert p.positions.tolist() == pos[50:]
    check(s.call(p), ref, 64)


def test_ends_of_any_size(gpu):
    """More rows than any request can have: they lie before its first token and see what a prefix shows them."""
    for end in (2 ** 28 - 1, 2 ** 28, 2 ** 31 - 1):
        s = Step([(90, 20)], 8, 2, 128, "e4m3", 33, prefix=[40])
        s.starts = [0, end]
        for window in (0, 50, 2 ** 31 - 1):
            r = s.call(s.plan(window=window))
            check(r, s.exact(window=window), 128, (end, window))
        assert s.plan().positions.tolist() == s.positions()
        s.prefix = None
        r = s.call(s.plan())
        assert not r["out"].any() and bool((r["lse"] == -torch.inf).all())


def test_a_cache_asked_for_fewer_rows(gpu):
    c = PagedCache(1, 8, 2, 64, 3, 200, 128, "e4m3")
    c.step(torch.tensor([40, 30, 20], dtype=torch.int32, device="cuda"))
    full, some = c.plan(90, 8), c.plan(55, 8)
    assert some.positions.tolist() == full.positions.tolist()[:55] == [*range(40), *range(15)]
