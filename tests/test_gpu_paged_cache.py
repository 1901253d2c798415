"""GPU: a serving loop on paged.PagedCache (page_map, cache_write and decode together, as they are used): requests come in
with prompts, decode and end, over two layers, eagerly and with the step captured in a graph. Each step's attention is
checked against the oracle on the values that the oracle's own pages hold, written beside it; and those against the keys
and values that went in."""

import random

import pytest
import torch

from cache8_side import check_out
from kvskip_amd.paged import PagedCache
from oracle import attention as O
from oracle import pages as OPG

pytestmark = pytest.mark.gpu

LAYERS, HKV, HQ, D, B, TOKENS, ROWS = 2, 2, 6, 64, 5, 640, 512


class Beside:
    """The oracle's cache: pages by lists, codes and scales by the oracle's writer, and the rows as they went in."""

    def __init__(self, fmt, pages):
        self.fmt = fmt
        self.lens, self.held = [0] * B, [0] * B
        self.table, self.free, self.count = [[-1] * (TOKENS // 64) for _ in range(B)], list(range(pages)), pages
        self.pools = [[torch.zeros(pages, HKV, 64, D, dtype=torch.uint8) for _ in "kv"] for _ in range(LAYERS)]
        self.scales = [[torch.zeros(pages, HKV) for _ in "kv"] for _ in range(LAYERS)]
        self.rows = [[[[], []] for _ in range(B)] for _ in range(LAYERS)]

    def step(self, new, drop):
        for b in range(B):
            if drop[b]:
                self.lens[b] = 0
                for l in range(LAYERS):
                    self.rows[l][b] = [[], []]
        self.lens = [n + a for n, a in zip(self.lens, new)]
        self.slots, self.starts, short, self.table, self.free, self.held, self.count = OPG.page_map(
            self.lens, new, self.held, self.table, self.free, self.count, ROWS)
        self.lens = [n - (a if n > 64 * h else 0) for n, h, a in zip(self.lens, self.held, new)]
        return short

    def write(self, l, k, v):
        for i, x in enumerate((k, v)):
            OPG.cache_write(x, self.slots, self.pools[l][i], self.scales[l][i], self.fmt)
            for b in range(B):
                for r in range(self.starts[b], min(self.starts[b + 1], ROWS)):
                    if self.slots[r] >= 0:
                        self.rows[l][b][i].append(x[r].double())

    def values(self, l, b):
        """k, v [1, Hkv, len, D] of request b in 64 bits and v's scale of each token."""
        pages = self.table[b][:-(-self.lens[b] // 64)]
        out = []
        for i in range(2):
            sc = self.scales[l][i][pages].double()                      # [pages, Hkv]
            x = OPG.decode_values(self.pools[l][i][pages], self.fmt) * sc[..., None, None]
            sc = sc.T.repeat_interleave(64, 1)[:, :self.lens[b]]
            x = x.transpose(0, 1).reshape(HKV, -1, D)[:, :self.lens[b]]
            # e4m3: half a step, 2^-4 of the value, or below its smallest normal code 2^-10 of the scale, again for each
            # move to a larger scale; int8: half of the scale, and half of each scale it had before, so less than one
            went = torch.stack(self.rows[l][b][i], 1)
            tol = sc[..., None] if self.fmt == "int8" else went.abs() * 2.0 ** -4 + sc[..., None] * 2.0 ** -9
            assert ((x - went).abs() <= tol).all()
            out.append(x[None])
        return *out, sc[None]


def _script(rng, steps):
    """new tokens and drops of each step."""
    lens = [0] * B
    for t in range(steps):
        new, drop = [], []
        for b in range(B):
            d = lens[b] > 0 and (rng.random() < 0.1 or lens[b] > TOKENS - 70)
            if d:
                lens[b] = 0
            a = (rng.choice([0, 5, 64, 100]) if rng.random() < 0.6 else 0) if lens[b] == 0 else 1
            lens[b] += a
            new.append(a), drop.append(d)
        yield new, drop


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("pages", [40, 6])
def test_serving(gpu, fmt, captured, pages):
    rng = random.Random(7)
    g = torch.Generator().manual_seed(3)
    cache, beside = PagedCache(LAYERS, pages, HKV, D, B, TOKENS, ROWS, fmt), Beside(fmt, pages)
    dev = "cuda"
    new_d, drop_d = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.bool, device=dev)
    k_d, v_d = (torch.zeros(LAYERS, ROWS, HKV, D, dtype=torch.bfloat16, device=dev) for _ in "kv")
    q_d = torch.zeros(B, HQ, D, dtype=torch.bfloat16, device=dev)

    def step():
        cache.step(new_d, drop_d)
        outs = []
        for l in range(LAYERS):
            cache.write(l, k_d[l], v_d[l])
            outs.append(cache.decode(l, q_d, D ** -0.5))
        return outs

    shorts = 0
    if captured:
        step()                                          # nothing new: no page, no row
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
    for t, (new, drop) in enumerate(_script(rng, 40)):
        k, v = (torch.randn(LAYERS, ROWS, HKV, D, generator=g).mul(2.0 ** (t % 5)).to(torch.bfloat16) for _ in "kv")
        q = torch.randn(B, HQ, D, generator=g).to(torch.bfloat16)
        new_d.copy_(torch.tensor(new, dtype=torch.int32)), drop_d.copy_(torch.tensor(drop))
        k_d.copy_(k), v_d.copy_(v), q_d.copy_(q)
        if captured:
            torch.cuda.synchronize()
            graph.replay()
        else:
            outs = step()
        torch.cuda.synchronize()
        short = beside.step(new, drop)
        shorts += short
        assert cache.lens.tolist() == beside.lens and cache.slot_map.tolist() == beside.slots and int(cache.short) == short
        for l in range(LAYERS):
            beside.write(l, k[l], v[l])
            for i in range(2):
                assert torch.equal(cache.pools[l][i].cpu().view(torch.uint8), beside.pools[l][i])
                assert torch.equal(cache.scales[l][i].cpu(), beside.scales[l][i])
            for b in range(B):
                if beside.lens[b] == 0:
                    assert not outs[l]["out"][b].any() and torch.isinf(outs[l]["lse"][b]).all()
                    continue
                kk, vv, vs = beside.values(l, b)
                r = {x: outs[l][x][b:b + 1].cpu() for x in ("out", "lse")}
                check_out(r, O.decode(q[b:b + 1], kk, vv, D ** -0.5), q[b:b + 1], kk, vv, D ** -0.5, what=(t, l, b),
                          v_scale=vs)
    assert (shorts > 0) == (pages == 6)


def test_take_off(gpu):
    """A negative count takes tokens off the end, and their pages back; the next ones go in their place."""
    c = PagedCache(1, 4, 1, 64, 2, 192, 160, "int8")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for new, lens, held in (((130, 5), [130, 5], [3, 1]), ((-70, 1), [60, 6], [1, 1]), ((-100, 0), [0, 6], [0, 1]),
                            ((64, -6), [64, 0], [1, 0])):
        c.step(i32(*new))
        assert c.lens.tolist() == lens and c.held.tolist() == held and int(c.free_count) == 4 - sum(held)
