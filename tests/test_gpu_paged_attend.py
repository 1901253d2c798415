"""GPU: a serving loop on paged.PagedCache whose steps bring prompts, chunks of prompts and single tokens together, behind shared
prefixes or none: page_map, the plan, norms and rotations at the plan's positions, rows into pages and their attention, as they
are used, over two layers, eagerly and captured in a graph. Each step's rotated rows and attention are checked against the
oracle over what the pages hold; what they hold against the rows that went in, at their positions."""

import random

import pytest
import torch

from attend_side import check
from kvskip_amd import ext
from kvskip_amd.paged import PagedCache
from oracle import attend as OA

pytestmark = pytest.mark.gpu

LAYERS, HKV, HQ, D, B, TOKENS, ROWS = 2, 2, 8, 64, 6, 640, 400
FREQ = (10000.0 ** (-2 * torch.arange(D // 2, dtype=torch.float64) / D)).float()


class Loop:
    def __init__(self, fmt, pages, shared=(200, 65), seed=1):
        self.c = PagedCache(LAYERS, pages, HKV, D, B, TOKENS, ROWS, fmt, shared=shared)
        self.g = torch.Generator().manual_seed(seed)
        self.w = [(1 + 0.2 * torch.randn(D, generator=self.g)).to(torch.bfloat16) for _ in "qk"]
        self.wd = [x.cuda() for x in self.w]
        self.freq = FREQ.cuda()
        self.qkv = torch.zeros(LAYERS, ROWS, HQ + 2 * HKV, D, dtype=torch.bfloat16, device="cuda")

    def fill(self):
        x = torch.randn(*self.qkv.shape, generator=self.g).to(torch.bfloat16)
        self.qkv.copy_(x)
        return x

    def layer(self, l, plan, rows, write, **kw):
        """One layer's way from the projection's output to the heads' output."""
        q, k, v = self.qkv[l, :rows].split([HQ, HKV, HKV], 1)
        q, k = ext.norm_rope(q, k, plan.positions, self.freq, *self.wd)
        write(l, k, v)
        return q, k, self.c.attend(l, q, D ** -0.5, plan, **kw)

    def check(self, got, x, l, plan, starts, lens, table, window=0, shared=True, **kw):
        c = self.c
        q, k, r = got
        rows = q.shape[0]
        pos = plan.positions.cpu()
        sh = shared and dict(shared_table=c.shared_table.cpu(), shared_lens=c.shared_lens.tolist(), shared_of=c.shared_of.tolist()) or {}
        assert pos.tolist() == OA.positions(starts, lens, rows, sh.get("shared_lens"), sh.get("shared_of"))
        for y, z, w in ((q, x[l, :rows, :HQ], self.w[0]), (k, x[l, :rows, HQ:HQ + HKV], self.w[1])):
            want = OA.norm_rope(z, pos, FREQ, w)
            n = torch.sqrt((z.double() ** 2).mean(-1, keepdim=True) + 1e-6)
            top = (z.double() / n * w.double()).abs().amax(-1, keepdim=True)
            assert ((y.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * top).all()
        kp, vp = (p.cpu() for p in c.pools[l])
        ks, vs = (s.cpu() for s in c.scales[l])
        check(r, OA.attend(q.cpu(), kp, vp, ks, vs, D ** -0.5, starts, lens, table, window=window, **kw, **sh), D, (l, rows))
        return kp, ks, k.cpu()


def test_prefixes_prompts_and_steps(gpu):
    for fmt, captured in (("e4m3", False), ("int8", True)):
        s, rng = Loop(fmt, 50), random.Random(5)
        c = s.c
        # the prefixes, each as a prompt of its own
        for i, n in enumerate((200, 37)):
            x = s.fill()
            plan = c.plan_prefix(i, n, HQ)
            for l in range(LAYERS):
                got = s.layer(l, plan, n, lambda l, k, v: c.write_prefix(l, i, k, v))
                kp, ks, k = s.check(got, x, l, plan, [0, n], [n], c.shared_table[i:i + 1].cpu(), shared=False)
                held = torch.cat([kp[p].float() * ks[p][:, None, None] for p in c.shared_table[i].tolist() if p >= 0], 1)[:, :n]
                step = ks[c.shared_table[i, 0]].max() if fmt == "int8" else 0.0
                assert ((held.transpose(0, 1) - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 0.02 + step).all()
        assert c.shared_lens.tolist() == [200, 37]
        c.shared_of.copy_(torch.tensor([0, 1, -1, 0, 0, 1], dtype=torch.int32))
        new_d = torch.zeros(B, dtype=torch.int32, device="cuda")
        drop_d = torch.zeros(B, dtype=torch.bool, device="cuda")

        def run():
            c.step(new_d, drop_d)
            plan = c.plan(ROWS, HQ)
            near = c.plan(ROWS, HQ, window=50)
            return plan, near, [s.layer(l, plan if l == 0 else near, ROWS, c.write) for l in range(LAYERS)]

        if captured:
            run()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                plan, near, got = run()
        lens = [0] * B
        for t in range(12):
            new, drop = [], []
            for b in range(B):
                d = lens[b] > 0 and rng.random() < 0.12
                a = rng.choice([0, 1, 64, 90, 130]) if lens[b] == 0 or d else rng.choice([1, 1, 1, 30])
                lens[b] = a if d else lens[b] + a
                new.append(a), drop.append(d)
            while sum(new) > ROWS - 3:
                b = max(range(B), key=lambda b: new[b])
                lens[b], new[b] = lens[b] - new[b] // 2, new[b] - new[b] // 2
            x = s.fill()
            new_d.copy_(torch.tensor(new, dtype=torch.int32)), drop_d.copy_(torch.tensor(drop))
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                plan, near, got = run()
            torch.cuda.synchronize()
            assert c.lens.tolist() == lens and int(c.short) == 0
            starts, table = c.starts.tolist(), c.block_table.cpu()
            for l in range(LAYERS):
                p = plan if l == 0 else near
                kp, ks, k = s.check(got[l], x, l, p, starts, lens, table, window=p.window)
                for b in range(B):                     # the last new row of each request, where its page should have it
                    if new[b]:
                        at, row = lens[b] - 1, starts[b + 1] - 1
                        page = table[b, at // 64]
                        held = kp[page, :, at % 64].float() * ks[page][:, None]
                        assert ((held - k[row].float()).abs() <= 2.0 ** -4 * k[row].float().abs() + 2 * ks[page][:, None]).all()


def test_short_of_pages(gpu):
    """A request without pages keeps the tokens it had; the others' rows are as in a step without it."""
    s = Loop("e4m3", 5, shared=())
    c = s.c
    x = s.fill()
    c.step(torch.tensor([100, 300, 64, 0, 0, 0], dtype=torch.int32, device="cuda"))
    plan = c.plan(ROWS, HQ)
    assert int(c.short) == 2 and c.lens.tolist() == [100, 0, 0, 0, 0, 0]
    q, k, r = s.layer(0, plan, ROWS, c.write)
    kp, vp, ks, vs = (t.cpu() for t in (*c.pools[0], *c.scales[0]))
    ref = OA.attend(q.cpu()[:100], kp, vp, ks, vs, D ** -0.5, [0, 100], [100], c.block_table.cpu()[:1])
    check({y: r[y][:100] for y in r}, ref, D)
    assert bool(r["out"].isfinite().all())
