"""GPU: the records that kvskip_attend_plan writes, one by one, against the model whose bounds the CPU tests hold."""

import random

import pytest
import torch

import attend_model as M
from kvskip_amd import kvskip as K
from test_attend_plan import cases

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def compare(c):
    m = M.Plan(**c)
    P, B = len(c.get("shared", ())), len(c["lens"])
    table = torch.zeros(B, c["T"] // 64, dtype=torch.int32, device="cuda")
    kw = dict(shared_table=torch.zeros(P, c["shared_T"] // 64, dtype=torch.int32, device="cuda"), shared_lens=i32(c["shared"]),
              shared_of=i32(c["of"])) if P else {}
    p = K.attend_plan(i32(c["starts"]), i32(c["lens"]), c["rows"], table, c["Hq"], c["Hkv"], max_rows=c.get("max_rows", 0),
                      window=c.get("window", 0), prefix_lens=i32(c["prefix"]) if "prefix" in c else None, **kw)
    work = p.work.cpu()
    units, n, first, last = M.records(work)
    assert p.positions.tolist() == m.positions
    assert (first, last) == (m.first, m.last) or m.first == m.last == first == last
    assert sorted(units) == sorted(m.units)
    per = [u.n for u in units]
    assert all(a >= b - max(per) // 31 - 1 for a, b in zip(per, per[1:]))        # longest first, by classes of a 31st of the longest
    at = M.at_joins(c["rows"], B, c["Hq"], c["Hkv"], P, c.get("max_rows", 0))
    assert M.joins(work, at, n) == m.joins
    return m


def test_records(gpu):
    """Random steps, and those of the CPU test whose tables are of moderate size."""
    rng, seen = random.Random(9), 0
    for c in cases():
        if c["T"] % 64 or c.get("shared_T", 0) % 64 or c["T"] // 64 * len(c["lens"]) > 1 << 20 or c["rows"] > 40000 or c["Hq"] > 128:
            continue
        if rng.random() < 0.5:
            compare(c)
            seen += 1
    assert seen > 100


def test_the_most_requests_and_prefixes(gpu):
    rng, B = random.Random(10), 2048
    new = [rng.choice([1, 1, 1, 0, 20]) for _ in range(B)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    m = compare(dict(starts=starts, lens=[rng.randint(0, 640) for _ in range(B)], rows=starts[-1], Hq=16, Hkv=8, T=640,
                     shared=[rng.randint(0, 192) for _ in range(64)], shared_T=192, of=[b % 65 for b in range(B)], max_rows=1))
    assert m.queued and len(m.joins) > 256
