"""GPU: a step whose new rows pass the slot map's end (page_map with lens_out, PagedCache.step): requests whose rows do not
all fit are not served, keep what they had, and are counted."""

import random

import pytest
import torch

from kvskip_amd import ext as E
from kvskip_amd.paged import PagedCache
from oracle import pages as OPG
from test_gpu_pages import I32, _dev, _state

pytestmark = pytest.mark.gpu


def _compare(lens, new, held, table, free, count, rows, form):
    """form: "in place" (lens_out is seq_lens, held and free_count updated), "apart" (buffers of their own), "lens" (lens_out
    alone a buffer of its own)."""
    want = OPG.page_map(lens, new, held, table, free, count, rows, whole=True)
    B = len(lens)
    ln, bt, fr, cn, hd = _dev(lens), _dev(table), _dev(free), _dev([count]), _dev(held)
    slots = torch.full((rows,), -5, **I32)
    kw = dict(lens_out=ln if form == "in place" else torch.full((B,), -99, **I32))
    if form == "apart":
        kw.update(held_out=torch.empty(B, **I32), free_count_out=torch.empty(1, **I32))
    _, starts, short = E.page_map(ln, _dev(new), hd, bt, fr, cn, slots, **kw)
    got = (slots.tolist(), starts.tolist(), int(short), bt.tolist(), fr.tolist(), kw.get("held_out", hd).tolist(),
           int(kw.get("free_count_out", cn)), kw["lens_out"].tolist())
    for name, a, b in zip(("slots", "starts", "short", "table", "free", "held", "count", "lens"), got, want):
        assert a == b, (form, name)
    return want


@pytest.mark.parametrize("B,width,rows", [(1, 3, 100), (7, 30, 300), (65, 20, 700), (65, 20, 4097), (300, 12, 5000),
                                          (2048, 3, 4096), (2048, 3, 9000)])
@pytest.mark.parametrize("tight", [False, True])
def test_page_map(gpu, B, width, rows, tight):
    rng = random.Random(B * 17 + rows + tight)
    pages = B * width * (1 if tight else 2) + 3
    held, table, free, count = _state(rng, B, width, pages, width)
    if tight:
        count = count // 3
        free[count:] = [-1] * (len(free) - count)
    lens, new = [], []
    for h in held:
        n = 0 if rng.random() < 0.2 else rng.randrange(1, 64 * width + 1)
        lens.append(n)
        new.append(min(n, rng.choice([0, 1, 2, 65, 200, 3 * rows // B])))
    shorts = [_compare(lens, new, held, table, free, count, rows, form)[2] for form in ("in place", "apart", "lens")]
    assert shorts[0] > 0 or sum(new) <= rows


def test_odd_values(gpu):
    """Sums that passed 31 bits, lengths below zero and past the row, requests that give pages and bring too many rows, no
    rows at all."""
    held, table = [2, 1, 0, 3, 0], [[5, 1, -1, -1], [0, -1, -1, -1], [-1] * 4, [2, 3, 6, -1], [-1] * 4]
    free, count = [7, 4, 9, 8, -1, -1, -1, -1, -1, -1], 4
    wrap = 2 ** 31 - 1 + 100 - 2 ** 32              # 100 tokens and 2^31 - 1 more
    for lens, new in [([-5, 300, 64, 129, 0], [-3, 9, 900, -2, 4]), ([128, 64, 257, 10 ** 9, 1], [0, 1, 257, 10 ** 9, 1]),
                      ([5, 64, 64, 20, 5], [5, 0, 64, 20, 5]), ([100, wrap, 64, 20, 5], [0, 2 ** 31 - 1, 0, 20, 0]),
                      ([wrap, 64, 0, 129, 70], [2 ** 31 - 1, 0, 0, 1, 0])]:
        for rows in (0, 1, 5, 70, 5000):
            for form in ("in place", "apart", "lens"):
                _compare(lens, new, held, table, free, count, rows, form)
                _compare(lens, new, held, table, free, 0, rows, form)


def test_lens_out_refused(gpu):
    i = torch.zeros(2, **I32)
    for bad in (torch.zeros(3, **I32), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="lens_out"):
            E.page_map(i, i, i, torch.zeros(2, 1, **I32), i, i[:1], i, lens_out=bad)


@pytest.mark.parametrize("captured", [False, True])
def test_cache_step(gpu, captured):
    """A request whose prompt passes the map's end is left as it was: nobody attends bytes that no row was written to."""
    HKV, HQ, D, ROWS = 2, 4, 64, 100
    c = PagedCache(1, 12, HKV, D, 4, 320, ROWS, "int8")
    for p in (*c.pools[0], ):
        p.fill_(127)                                    # what a page's last user left
    for s in c.scales[0]:
        s.fill_(1e30)
    new_d, k_d = torch.zeros(4, **I32), torch.zeros(ROWS, HKV, D, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(4, HQ, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()

    def step():
        c.step(new_d)
        c.write(0, k_d, k_d)
        return c.decode(0, q, 0.125)

    run = step
    if captured:
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = step()

        def run():
            torch.cuda.synchronize()
            g.replay()
            return r

    lens = [0] * 4
    last = None
    for t, new in enumerate([(30, 40, 20, 10), (1, 0, 101, 0), (1, 99, 1, 0), (0, 2 ** 31 - 1, 0, 1), (50, 0, 50, 0),
                             (1, 1, 1, 1)]):
        k = torch.randn(ROWS, HKV, D, generator=torch.Generator().manual_seed(t)).to(torch.bfloat16)
        new_d.copy_(torch.tensor(new, dtype=torch.int32)), k_d.copy_(k)
        r_now = run()
        torch.cuda.synchronize()
        at, short = 0, 0
        for b, a in enumerate(new):
            at += a
            if a > 0 and at > ROWS:
                short += 1
            else:
                lens[b] += a
        assert c.lens.tolist() == lens and int(c.short) == short == (0, 1, 1, 2, 0, 0)[t], t
        out = r_now["out"].float().cpu()
        assert torch.isfinite(out).all() and out.abs().max() < 10, t
        if last is not None:      # requests that got nothing answer as before: another cut of the batch adds in another order,
            for b in range(4):    # so two bf16 roundings (2^-8 of the value each) and fp32 sums of values below 10 (2^-16 each)
                if lens[b] == last[0][b]:
                    assert ((out[b] - last[1][b]).abs() <= 2.0 ** -7 * last[1][b].abs() + 20 * 2.0 ** -16).all(), (t, b)
        last = list(lens), out
        held = c.held.tolist()
        assert all(-(-n // 64) == h for n, h in zip(lens, held)) and int(c.free_count) == 12 - sum(held)
