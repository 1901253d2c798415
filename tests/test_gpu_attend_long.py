"""GPU: attention over a step's rows whose units are long: many pages a wavefront in small tiles and many turns in large ones, plans
with more tiles than a round of workgroups, the most units of a tile, joins in more than one round.

A plan shortens units until every CU has some, so a unit is long where the tiles alone fill the card: a few requests are repeated to as
many tiles as that takes, and the repeated ones must have the first ones' bits."""

import pytest
import torch

import attend_model as M
from attend_side import Step, check

pytestmark = pytest.mark.gpu

KINDS = [("e4m3", 128), ("int8", 128), ("e4m3", 64), ("int8", 64)]
MODS = [(0.0, False), (30.0, True)]


def crowd(step, times):
    """The step's requests `times` over, over the same pages."""
    n = step.rows
    step.base_rows, step.base_starts, step.base_lens, step.base_table, step.base_q = n, step.starts, step.lens, step.table, step.q
    step.starts = step.starts + [x + n * i for i in range(1, times) for x in step.starts[1:]]
    step.lens, step.rows = step.lens * times, n * times
    step.table, step.q = step.table.repeat(times, 1), step.q.repeat(times, 1, 1)
    return step


def exact_of_one(s, **kw):
    saved = s.starts, s.lens, s.rows, s.table, s.q
    s.starts, s.lens, s.rows, s.table, s.q = s.base_starts, s.base_lens, s.base_rows, s.base_table, s.base_q
    ref = s.exact(**kw)
    s.starts, s.lens, s.rows, s.table, s.q = saved
    return ref


def units_of(plan):
    return M.records(plan.work.cpu())[0]


def run(s, what, softcap=0.0, slopes=None, window=0, max_rows=0, least=None, large=None):
    plan = s.plan(window=window, max_rows=max_rows)
    units = units_of(plan)
    if least is not None:
        assert max(u.n for u in units if large is None or u.kind & 1 == large) > least, what
    r = s.call(plan, softcap, slopes)
    n = s.base_rows
    first = {k: v[:n] for k, v in r.items()}
    check(first, exact_of_one(s, window=window, softcap=softcap, slopes=slopes), s.D, what, softcap=softcap)
    bits = lambda t: t.view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)
    for i in range(n, s.rows, n):
        assert all(torch.equal(bits(r[k][i:i + n].contiguous()), bits(first[k].contiguous())) for k in r), (what, i)
    return units


@pytest.mark.parametrize("cap,biased", MODS)
@pytest.mark.parametrize("fmt,D", KINDS)
def test_small_tiles_of_many_pages(gpu, fmt, D, cap, biased):
    """More than 256 pages a unit: a wavefront's list is gathered again (more than 64 pages each)."""
    s = Step([(64 * 301, 1), (64 * 299 - 17, 1), (64 * 270 + 3, 1)], 16, 8, D, fmt, 51, signed=biased)
    slopes = torch.linspace(0.0005, 0.004, 16) if biased else None
    run(crowd(s, 21), (fmt, D), cap, slopes, max_rows=1, least=256, large=0)


@pytest.mark.parametrize("cap,biased", MODS)
@pytest.mark.parametrize("fmt,D", KINDS)
def test_large_tiles_of_many_pages(gpu, fmt, D, cap, biased):
    """More than 120 pages a unit: the page list of a large tile is gathered three times."""
    s = Step([(64 * 131, 64), (64 * 130 - 17, 60), (64 * 127 + 3, 64)], 16, 8, D, fmt, 52, signed=biased)
    slopes = torch.linspace(0.001, 0.01, 16) if biased else None
    run(crowd(s, 21), (fmt, D), cap, slopes, least=120, large=1)


def several(fmt, D, seed, **kw):
    """Ten pages a wavefront of small tiles, forty a large one."""
    s = Step([(64 * 41, 1), (64 * 40 - 30, 1), (64 * 40, 50)], 16, 8, D, fmt, seed, **kw)
    return s


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("fmt,D", KINDS)
def test_scores_that_rise_inside_a_unit(gpu, fmt, D, signed, rising):
    """References that every page passes, and ones that none does after the first."""
    s = several(fmt, D, 53, signed=signed)
    for b in range(3):
        for i in range(s.table.shape[1]):
            p = s.table[b, i]
            if p >= 0:
                x = 2.0 ** ((i if rising else 40 - i) / 6 - 9)
                s.ks[p] = s.ks[p].sign() * x
                s.vs[p] = s.vs[p].sign() * 2.0 ** -12 / x
    run(crowd(s, 21), (fmt, D), least=30)


@pytest.mark.parametrize("cap,biased", MODS)
@pytest.mark.parametrize("fmt,D", KINDS)
def test_scales_far_apart_inside_a_unit(gpu, fmt, D, cap, biased):
    """V's scales up to 2^60 apart from page to page, some of them 0, some scores far away: what is heavy changes from page to page."""
    s = several(fmt, D, 54, signed=True)
    g = torch.Generator().manual_seed(55)
    s.vs = s.vs.sign() * torch.exp2(torch.randint(-40, 21, s.vs.shape, generator=g).float())
    s.vs[torch.rand(s.vs.shape, generator=g) < 0.1] = 0.0
    s.ks *= torch.exp2(torch.randint(-3, 3, s.ks.shape, generator=g).float())
    s.ks[torch.rand(s.ks.shape, generator=g) < 0.1] = 0.0
    run(crowd(s, 21), (fmt, D), cap, torch.linspace(0.001, 0.01, 16) if biased else None, least=30)


def test_large_scores_inside_a_unit(gpu):
    """Scores around 2^11: references past 2^10, which the short form of the weights does not serve."""
    for fmt, D in KINDS:
        s = several(fmt, D, 56)
        s.scale *= 2.0 ** 9
        ref = exact_of_one(crowd(s, 21))
        assert ref[1].abs().max() > 2.0 ** 10
        plan = s.plan()
        assert max(u.n for u in units_of(plan)) > 30
        r = s.call(plan)
        assert r["out"].isfinite().all()
        ds = (D + 8) * 2.0 ** -23 * ref[3] + 2.0 ** -20 * ref[1].abs()
        assert ((r["lse"][:s.base_rows].double().cpu() - ref[1]).abs() <= ds).all(), (fmt, D)


def test_windows_and_prefixes_inside_a_unit(gpu):
    for fmt, D in KINDS:
        s = several(fmt, D, 57, prefix=[700, 0, 1000] * 21)
        run(crowd(s, 21), (fmt, D), window=1500, least=20)


def test_what_no_row_sees_inside_a_unit(gpu):
    """NaN codes and scales before a row's window, behind a row and past the end, in tiles of many pages; missing pages between."""
    for D in (64, 128):
        s = several("e4m3", D, 58)
        s.k, s.v = s.k.view(torch.uint8), s.v.view(torch.uint8)
        for b, t, d in ((0, 64 * 18 + 3, 5), (0, 64 * 30 + 63, 40), (1, 64 * 17 + 9, 63), (2, 64 * 40 - 20, 11), (2, 64 * 39, 12),
                        (2, 64 * 20 + 1, 13), (2, 64 * 20 + 49, 14)):
            s.v[s.table[b, t // 64], :, t % 64, d] = 0x7f if d % 2 else 0xff
        s.k[s.table[1, 39], 3, 20] = 0x7f                     # seen: a row of NaN
        s.v[s.table[1, 39], :, 35:] = 0x7f                    # past the end
        s.k, s.v = s.k.view(torch.float8_e4m3fn), s.v.view(torch.float8_e4m3fn)
        for b, i in ((0, 20), (0, 21), (0, 22), (0, 23), (1, 25), (2, 30), (2, 33)):
            p = int(s.table[b, i])
            s.table[b, i] = -1 if i % 2 else s.k.shape[0]
            s.ks[p], s.vs[p] = torch.nan, torch.inf           # (no table names it any more)
        s = crowd(s, 21)
        units = run(s, D, window=64 * 22 + 11)
        assert max(u.n for u in units) > 20
        ref = exact_of_one(s, window=64 * 22 + 11)[0]
        assert ref[0].isnan().any() and not ref[0].isnan().all() and ref[2:].isnan().any() and not ref[2:].isnan().all()


@pytest.mark.parametrize("fmt,Hq,D", [("e4m3", 16, 128), ("int8", 8, 64)])
def test_more_tiles_than_a_round(gpu, fmt, Hq, D):
    """Queued units: prompts and single tokens, more tiles than workgroups at once."""
    s = Step([(300, 300), (1, 1), (64 * 20, 40), (64 * 9 + 1, 1), (65, 2)], Hq, 8, D, fmt, 59)
    s = crowd(s, 30)
    plan = s.plan()
    assert sum(u.i0 == 0 for u in units_of(plan)) > 64
    run(s, (fmt, D))
    run(s, (fmt, D), window=100)


@pytest.mark.parametrize("D", [64, 128])
def test_the_most_units_of_a_tile(gpu, D):
    """One request of 1025 pages and one KV head: 128 units, joined by 128 partial results a row."""
    s = Step([(64 * 64, 1)], 4, 1, D, "e4m3", 60)
    s.lens, s.table = [64 * 1024 + 9], s.table[:, torch.randint(0, 64, (1025,), generator=torch.Generator().manual_seed(61))].contiguous()
    plan = s.plan()
    assert len(units_of(plan)) == 128
    check(s.call(plan), s.exact(), D)


def test_joins_in_more_than_one_round(gpu):
    """More runs of rows than the join has workgroups: its shared memory is used again."""
    s = Step([(60 + b, 40) for b in range(16)], 16, 8, 64, "int8", 62, shared=[200], of=[0] * 64)
    s = crowd(s, 4)
    plan = s.plan()
    assert M.records(plan.work.cpu())[1] * 8 > 2 * 2048
    run(s, "joins")
