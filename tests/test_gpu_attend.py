"""GPU: attention of a step's rows over 8-bit pages (kvskip.attend_plan, kvskip.attend) against the 64-bit oracle: lengths from
none on, every head layout, prompts and single tokens together, masks that leave rows nothing, shared prefixes, values that
no row may see."""

import pytest
import torch

from attend_side import Step, check
from kvskip_amd import kvskip as K

pytestmark = pytest.mark.gpu

HEADS = [(4, 4, 64), (8, 2, 64), (8, 2, 128), (14, 2, 128), (8, 1, 128), (16, 1, 64), (24, 1, 128), (3, 1, 64)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_single_tokens(gpu, fmt, Hq, Hkv, D):
    lens = [1, 64, 65, 0, 127, 500, 2, 1300, 63]
    s = Step([(n, 1) for n in lens], Hq, Hkv, D, fmt, 1 + Hq)
    for most in (1, 0):                                 # the tiles for single tokens, and those beside large ones
        p = s.plan(max_rows=most)
        assert p.positions.tolist() == s.positions()
        check(s.call(p), s.exact(), D, (fmt, Hq, most))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_prompts_chunks_and_tokens(gpu, fmt, Hq, Hkv, D):
    reqs = [(70, 70), (1, 1), (300, 1), (0, 0), (200, 129), (513, 37), (64, 64), (5, 0), (130, 2)]
    s = Step(reqs, Hq, Hkv, D, fmt, 2 + Hq, pad=3, lead=2, signed=True)
    p = s.plan()
    assert p.positions.tolist() == s.positions()
    r = s.call(p)
    check(r, s.exact(), D, (fmt, Hq))
    assert not r["out"][:2].any() and not r["out"][-3:].any() and bool((r["lse"][-3:] == -torch.inf).all())


@pytest.mark.parametrize("max_rows", [0, 1, 4])
def test_more_rows_than_said(gpu, max_rows):
    s = Step([(700, 150), (33, 1), (90, 8)], 8, 2, 128, "e4m3", 3)
    check(s.call(s.plan(max_rows=max_rows)), s.exact(), 128, max_rows)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 2 ** 31 - 1])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(gpu, window, D):
    s = Step([(900, 1), (400, 300), (64, 64), (1, 1), (65, 2)], 8, 2, D, "e4m3", 4)
    check(s.call(s.plan(window=window)), s.exact(window=window), D, window)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("fmt,D", [("e4m3", 128), ("int8", 64)])
def test_prefixes(gpu, window, fmt, D):
    reqs, prefix = [(300, 300), (300, 300), (130, 1), (500, 200), (64, 64), (90, 90)], [0, 170, 64, 500, 9999, -5]
    s = Step(reqs, 8, 2, D, fmt, 5, prefix=prefix)
    check(s.call(s.plan(window=window)), s.exact(window=window), D, (window, fmt))


def test_rows_that_see_nothing(gpu):
    """More rows than tokens: those at negative positions see nothing, but for what a prefix shows them; a request without tokens."""
    reqs, prefix = [(3, 10), (0, 4), (2, 100), (40, 60)], [0, 0, 0, 25]
    for pre in (None, prefix):
        s = Step(reqs, 8, 2, 128, "e4m3", 6, prefix=pre)
        r = s.call(s.plan())
        check(r, s.exact(), 128, pre)
        assert not r["out"][:7].any() and bool((r["lse"][10:14] == -torch.inf).all())


@pytest.mark.parametrize("cap", [0.5, 20.0, 1e5])
@pytest.mark.parametrize("fmt,Hq,Hkv,D", [("e4m3", 8, 2, 128), ("int8", 14, 2, 128), ("e4m3", 8, 2, 64)])
def test_caps(gpu, cap, fmt, Hq, Hkv, D):
    s = Step([(200, 1), (300, 300), (65, 3)], Hq, Hkv, D, fmt, 7, signed=True)
    check(s.call(s.plan(), softcap=cap), s.exact(softcap=cap), D, (cap, fmt), softcap=cap)
    s = Step([(200, 1), (64, 1)], Hq, Hkv, D, fmt, 7)
    check(s.call(s.plan(max_rows=1), softcap=cap), s.exact(softcap=cap), D, (cap, fmt), softcap=cap)


@pytest.mark.parametrize("cap,window", [(0.0, 0), (30.0, 0), (0.0, 100)])
def test_bias(gpu, cap, window):
    g = torch.Generator().manual_seed(8)
    for Hq, Hkv, D in ((8, 2, 128), (14, 2, 64)):
        slopes = torch.randn(Hq, generator=g) * 0.2          # of either sign
        s = Step([(700, 1), (200, 150), (1, 1), (90, 60)], Hq, Hkv, D, "int8", 9, prefix=[0, 190, 1, 80])
        for most in (0, 1):
            check(s.call(s.plan(window=window, max_rows=most), softcap=cap, slopes=slopes), s.exact(window, cap, slopes), D,
                  (cap, window, most), softcap=cap)


@pytest.mark.parametrize("fmt,Hq,Hkv,D", [("e4m3", 8, 2, 128), ("int8", 14, 2, 128), ("e4m3", 4, 4, 64)])
@pytest.mark.parametrize("window", [0, 150])
def test_shared_prefixes(gpu, fmt, Hq, Hkv, D, window):
    reqs = [(100, 1), (65, 1), (1, 1), (300, 1), (0, 0), (64, 1), (20, 20), (200, 90), (5, 1), (30, 1)]
    of = [0, 1, 0, -1, 0, 0, 2, 0, 7, 3]                      # 7: no such prefix; 3: an empty one
    s = Step(reqs, Hq, Hkv, D, fmt, 10, shared=[130, 64, 500, 0], of=of, pad=1)
    p = s.plan(window=window)
    assert p.positions.tolist() == s.positions()
    check(s.call(p), s.exact(window=window), D, (fmt, window))


@pytest.mark.parametrize("n", [1, 3, 8, 9, 40, 150])
def test_a_batch_behind_one_prefix(gpu, n):
    """Single tokens in small and large tiles over the prefix."""
    s = Step([(1 + 13 * b % 90, 1) for b in range(n)], 8, 2, 128, "e4m3", 11, shared=[777], of=[0] * n,
             prefix=[50 * (b % 2) for b in range(n)])
    for window in (0, 60):
        check(s.call(s.plan(max_rows=1, window=window)), s.exact(window=window), 128, (n, window))


def test_shared_with_caps_and_bias(gpu):
    slopes = torch.linspace(0.01, 0.4, 14)
    s = Step([(90, 1), (10, 10), (1, 1), (200, 1)], 14, 2, 128, "int8", 12, shared=[300, 90], of=[0, 0, 1, 0])
    check(s.call(s.plan(), softcap=15.0, slopes=slopes), s.exact(softcap=15.0, slopes=slopes), 128, softcap=15.0)


@pytest.mark.parametrize("D", [64, 128])
def test_long_lists_in_stages(gpu, D):
    """Units of more than 64 steps a wavefront (the page list's gathers) and of more than 64 pages in large tiles."""
    s = Step([(64 * 330 + 5, 1), (64 * 150, 130)], 2, 1, D, "e4m3", 13)
    check(s.call(s.plan()), s.exact(), D)
    s = Step([(64 * 70 + 5, 70)] * 24, 16, 8, 64, "int8", 14)   # 192 tiles a head: uncut
    check(s.call(s.plan()), s.exact(), 64)


def test_what_no_row_sees(gpu):
    """NaN and infinities in keys after a row, before its window, past the sequence's end and on pages that no table names
    do not reach it; those that it sees do."""
    for D, Hq in ((128, 8), (64, 8)):
        for reqs, window, most in (([(130, 130), (100, 40), (70, 1)], 0, 0), ([(130, 130), (200, 3), (150, 1)], 50, 0),
                                   ([(150, 1), (90, 1), (64, 1)], 50, 1)):
            s = Step(reqs, Hq, 2, D, "e4m3", 15)
            kb, vb = s.k.view(torch.uint8), s.v.view(torch.uint8)
            for b, t, d in ((0, 100, 3), (0, 127, 50), (1, 37, 0), (1, 88, 63), (2, 20, 33), (2, 63, 10)):
                if t < reqs[b][0]:
                    vb[s.table[b, t // 64], :, t % 64, d] = 0x7f if d % 2 else 0xff
            for b, t in ((0, 120), (1, 5)):
                kb[s.table[b, t // 64], 1, t % 64, 2] = 0x7f
            for b, (n, _) in enumerate(reqs):               # rows past the end, and free pages
                if n % 64:
                    vb[s.table[b, n // 64], :, n % 64:] = 0x7f
                    kb[s.table[b, n // 64], :, n % 64:] = 0xff
            free = sorted(set(range(s.k.shape[0])) - set(s.table.flatten().tolist()))
            vb[free], kb[free] = 0x7f, 0x7f
            s.ks[free], s.vs[free] = torch.nan, torch.inf
            ref = s.exact(window=window)
            assert ref[0].isnan().any() and not ref[0].isnan().all()
            check(s.call(s.plan(window=window, max_rows=most)), ref, D, (D, window, most))


def test_scales_that_are_not_numbers(gpu):
    """A page's NaN scale reaches the rows that see one of its keys and no others."""
    s = Step([(200, 200), (130, 1)], 8, 2, 128, "int8", 16)
    s.vs[s.table[0, 2], 0] = torch.nan
    s.ks[s.table[0, 1], 1] = torch.nan
    r = s.call(s.plan())
    out = r["out"].isnan().all(-1)
    assert not out[:128, :4].any() and bool(out[128:200, :4].all())
    assert not out[:64, 4:].any() and bool(out[64:200, 4:].all()) and not out[200].any()


def test_queries_that_are_not_numbers(gpu):
    s = Step([(90, 20), (70, 1)], 8, 2, 128, "e4m3", 17)
    s.q[3, 5, 7] = torch.nan
    s.q[9, 0, 0] = torch.inf
    r = s.call(s.plan())
    bad = r["out"].isnan().all(-1).cpu()
    want = torch.zeros_like(bad)
    want[3, 5] = want[9, 0] = True
    assert torch.equal(bad, want) and torch.equal(r["out"].isnan().any(-1).cpu(), want)


def test_pages_outside_the_pool(gpu):
    """Their keys are not there: the rest is attended, and a row that has no other gets zeros."""
    s = Step([(200, 1), (130, 100), (64, 1)], 8, 2, 128, "e4m3", 18)
    s.table[0, 1], s.table[1, 0], s.table[2, 0] = -1, s.k.shape[0], 2 ** 31 - 1
    r = s.call(s.plan())
    check(r, s.exact(), 128)
    assert not r["out"][-1].any() and bool((r["lse"][-1] == -torch.inf).all())


def test_starts_that_do_not_rise(gpu):
    s = Step([(100, 4), (90, 3), (80, 2)], 8, 2, 128, "e4m3", 19, pad=2)
    for starts in ([0, 4, 3, 9], [5, 4, 7, 9]):
        s.starts = starts
        p = s.plan()
        r = s.call(p)
        assert not r["out"].any() and bool((r["lse"] == -torch.inf).all()) and p.positions.tolist() == [-1] * s.rows
    s.starts = [-3, 4, 7, 40]                                 # clamped to the rows
    check(s.call(s.plan()), s.exact(), 128)


@pytest.mark.parametrize("big", [2.0 ** 60, 2.0 ** -60])
def test_large_and_small_scores(gpu, big):
    """Scores far from 0 take no weight from the largest, and queries of any magnitude are exact."""
    s = Step([(200, 130), (300, 1)], 8, 2, 128, "int8", 20)
    s.q, s.scale = (s.q.float() * big).to(torch.bfloat16), s.scale / big
    check(s.call(s.plan()), s.exact(), 128, big)
    s.scale *= 2.0 ** 20                                      # scores near 2^20: a handful of keys weigh anything
    r = s.call(s.plan())
    assert r["out"].isfinite().all()
    ref = s.exact()
    assert ((r["lse"].double().cpu() - ref[1]).abs() <= (128 + 8) * 2.0 ** -23 * ref[3] + 2.0 ** -20 * ref[1].abs()).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 2, 64)])
def test_scales_of_any_size(gpu, Hq, Hkv, D):
    """V's scales 2^60 apart: a row whose weight lies on small values is as exact as another."""
    s = Step([(64 * 3, 150), (64 * 3, 1)], Hq, Hkv, D, "int8", 21)
    for b in range(2):
        s.vs[s.table[b, 0]], s.vs[s.table[b, 1]], s.vs[s.table[b, 2]] = 2.0 ** -40, 2.0 ** 20, 2.0 ** -40
        s.ks[s.table[b, 1]] = 0.0                            # scores 0
        s.k[s.table[b, 1]] = 0
    s.q *= 16
    check(s.call(s.plan()), s.exact(), D)


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("fmt,D", [("int8", 128), ("e4m3", 64)])
def test_scores_that_rise(gpu, fmt, D, rising, signed):
    """Scores that grow, or fall, by half a power of two a page, V's scales the other way: references that every page
    passes, and ones that no later page does."""
    s = Step([(64 * 14 + 9, 260), (64 * 14, 1)], 8, 2, D, fmt, 23, signed=signed)
    for b in range(2):
        for i in range(14):
            x = 2.0 ** ((i if rising else 13 - i) / 2 - 9)
            s.ks[s.table[b, i]] = s.ks[s.table[b, i]].sign() * x
            s.vs[s.table[b, i]] = s.vs[s.table[b, i]].sign() * 2.0 ** -12 / x
    check(s.call(s.plan()), s.exact(), D)


def test_strides(gpu):
    """q as a slice of a fused projection, pools and scales as views, tables of more columns than needed."""
    s = Step([(90, 60), (130, 1)], 8, 2, 128, "e4m3", 22, width=9)
    P = s.k.shape[0]
    qkv = torch.zeros(s.rows, 8 + 4, 128, dtype=torch.bfloat16, device="cuda")
    qkv[:, 1:9] = s.q.cuda()
    pool = torch.zeros(P, 2, 2, 64, 144, dtype=torch.uint8, device="cuda")
    pool[:, 0, :, :, :128], pool[:, 1, :, :, 16:] = s.k.view(torch.uint8).cuda(), s.v.view(torch.uint8).cuda()
    sc = torch.stack([s.ks, s.vs], -1).cuda()
    table = torch.full((2, 14), -1, dtype=torch.int32, device="cuda")
    table[:, 3:12] = s.table.cuda()
    plan = K.attend_plan(s.i32(s.starts), s.i32(s.lens), s.rows, table[:, 3:12], 8, 2)
    pool = pool.view(torch.float8_e4m3fn)
    r = K.attend(qkv[:, 1:9], pool[:, 0, :, :, :128], pool[:, 1, :, :, 16:], s.scale, plan, sc[..., 0], sc[..., 1])
    check(r, s.exact(), 128)


def test_results_do_not_depend_on_the_run(gpu):
    """The same bits from every plan of the same step, whatever order its units came in."""
    s = Step([(500, 1), (300, 200), (64, 64), (900, 1)], 8, 2, 128, "e4m3", 23, shared=[200], of=[0, 0, -1, 0])
    first = s.call(s.plan())
    for _ in range(5):
        r = s.call(s.plan())
        assert torch.equal(r["out"], first["out"]) and torch.equal(r["lse"], first["lse"])


def test_no_rows(gpu):
    s = Step([(50, 1)], 8, 2, 128, "e4m3", 24)
    plan = K.attend_plan(s.i32([0, 0]), s.i32([50]), 0, s.table.cuda(), 8, 2)
    r = K.attend(s.q[:0].cuda(), s.k.cuda(), s.v.cuda(), s.scale, plan, s.ks.cuda(), s.vs.cuda())
    assert r["out"].shape == (0, 8, 128) and r["lse"].shape == (0, 8) and plan.positions.shape == (0,)


def test_captured(gpu):
    """Plan and attention of two layers in a graph, replayed with other lengths, tables and queries between eager calls."""
    a = Step([(300, 1), (200, 90), (64, 64)], 8, 2, 128, "e4m3", 25)
    b = Step([(190, 64), (20, 1), (310, 90)], 8, 2, 128, "e4m3", 26)
    cu = lambda *t: [x.cuda() for x in t]
    starts, lens, table = a.i32(a.starts), a.i32(a.lens), torch.zeros(3, 5, dtype=torch.int32, device="cuda")
    q, k, v, ks, vs = cu(a.q, a.k, a.v, a.ks, a.vs)
    table[:, :a.table.shape[1]] = a.table.cuda()
    run = lambda: [K.attend(x, k, v, a.scale, p, ks, vs, softcap=c)["out"]
                   for p in [K.attend_plan(starts, lens, a.rows, table, 8, 2)] for x, c in ((q, 0.0), (-q, 30.0))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run()
    for s in (a, b, a, b):
        n = min(s.rows, a.rows)
        starts.copy_(s.i32(s.starts).clamp(max=a.rows)), lens.copy_(s.i32(s.lens))
        for page in range(s.table.shape[1]):
            table[:, page] = s.table[:, page].cuda().clamp(max=a.k.shape[0] - 1)
        q[:n].copy_(s.q[:n])
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = run()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_on_another_stream_and_two_at_once(gpu):
    s = Step([(500, 1), (300, 200)], 8, 2, 128, "e4m3", 27)
    args = [x.cuda() for x in (s.q, s.k, s.v, s.ks, s.vs)]
    plan = s.plan()
    ref = K.attend(args[0], args[1], args[2], s.scale, plan, args[3], args[4])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        with torch.cuda.stream(st):
            got.append([K.attend(args[0], args[1], args[2], s.scale, plan, args[3], args[4]) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(r["out"], ref["out"]) for rs in got for r in rs)
