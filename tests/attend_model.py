"""What kvskip_attend_plan writes, in Python (csrc/attend.hpp has the records, csrc/attend_plan.hip the rules): for the test of its bounds on the CPU,
and of the kernel's records against it on the GPU."""

from collections import namedtuple

FEW, MANY, PAGE, SLOTS, LEAST, LEAST_QUEUED, MOST_UNITS, JOIN_ROWS = 16, 128, 64, 512, 4, 16, 128, 8
MOST_END = 1 << 28

Unit = namedtuple("Unit", "kind row0 v0 nv p0 pre table len base a1 b0 i0 n part")
Join = namedtuple("Join", "row0 v0 n part ns step more more_ns more_step")
Request = namedtuple("Request", "first n pos0 len base pre group")


def clamp(x, lo, hi):
    return min(max(x, lo), hi)


def span(lo, hi, base, n, pre, window):
    end = min(n, max(hi - base + 1, 0))
    since = max(lo - window + 1 - base, 0) if window else 0
    a1 = (min(max(pre - base, 0), n) + PAGE - 1) // PAGE
    b0 = max(since // PAGE, a1)
    return a1, b0, a1 + max((end + PAGE - 1) // PAGE - b0, 0)


class Plan:
    """starts [B + 1], lens [B]; shared: the prefixes' lengths, of: which one each request is behind."""

    def __init__(self, starts, lens, rows, Hq, Hkv, T, shared=(), of=None, shared_T=0, prefix=None, max_rows=0, window=0):
        B, G = len(lens), Hq // Hkv
        window = min(window, 1 << 30)
        most = max_rows if 0 < max_rows < rows else rows
        many = MANY if most * G > FEW or (shared and rows * G > FEW) else 0
        height = lambda virt: FEW if many == 0 or virt <= FEW else many
        rises = all(a <= b for a, b in zip(starts, starts[1:]))
        reqs = []
        for b in range(B if rises else 0):
            first, end = clamp(starts[b], 0, rows), min(starts[b + 1], MOST_END)
            n = min(max(end, first), rows) - first
            g = of[b] if shared and 0 <= of[b] < len(shared) else -1
            base = clamp(shared[g], 0, shared_T) if g >= 0 else 0
            m = clamp(lens[b], 0, T)
            reqs.append(Request(first, n, base + m - (end - first), m, base, clamp(prefix[b], 0, base + m) if prefix else 0,
                                g if base else -1))
        self.first = reqs[0].first if reqs else 0
        self.last = clamp(starts[-1], self.first, rows) if reqs else 0
        self.positions = [-1] * rows
        for r in reqs:
            for i in range(r.n):
                self.positions[r.first + i] = r.pos0 + i
        # tiles: (request or ~prefix, v0, virtual rows of its owner, pages)
        tiles = []
        for b, r in enumerate(reqs):
            virt = r.n * G
            for v0 in range(0, virt, height(virt)):
                v1 = min(v0 + height(virt), virt) - 1
                tiles.append((b, v0, virt, span(r.pos0 + v0 // G, r.pos0 + v1 // G, r.base, r.len, r.pre, window)))
        own, place, groups, row0 = len(tiles), {}, [], 0
        self.rows = []
        for g in range(len(shared)):
            mine = [b for b, r in enumerate(reqs) if r.group == g and r.n > 0]
            count = 0
            for b in mine:
                place[b] = count
                count += reqs[b].n
                self.rows += [(reqs[b].first + i, reqs[b].pos0 + i, reqs[b].pre) for i in range(reqs[b].n)]
            virt, tile0 = count * G, len(tiles)
            if mine:
                s = span(min(reqs[b].pos0 for b in mine), 2 ** 31 - 2, 0, reqs[mine[0]].base, max(reqs[b].pre for b in mine), window)
                tiles += [(~g, v0, virt, s) for v0 in range(0, virt, height(virt))]
            groups.append((row0, virt, tile0))
            row0 += count
        # the pages of a unit
        pages = sum(t[3][2] for t in tiles)
        room = max(SLOTS // Hkv, 1)
        self.queued = True
        if len(tiles) <= room:
            c0 = max(LEAST, (pages + room - 1) // room)
            for i in range(16):
                c = c0 + (c0 * i + 15) // 16
                if sum((t[3][2] + c - 1) // c for t in tiles) <= room:
                    self.queued = False
                    break
        if self.queued:
            c = max(LEAST_QUEUED, (pages * Hkv + 2 * SLOTS - 1) // (2 * SLOTS))
        self.chunk = c
        self.n_tiles, self.units, self.joins, self.parts, first_part = len(tiles), [], [], 0, []
        for who, v0, virt, (a1, b0, n) in tiles:
            nv, ns = min(height(virt), virt - v0), clamp((n + c - 1) // c, 1, MOST_UNITS)
            group = reqs[who].group if who >= 0 else ~who
            part = -1
            if group >= 0 or ns > 1:
                part, self.parts = self.parts, self.parts + nv * ns
            first_part.append((part, nv, ns))
            big = 1 if many and height(virt) == many else 0
            for i in range(ns):
                i0 = n * i // ns
                at = part + i * nv if part >= 0 else -1
                if who >= 0:
                    r = reqs[who]
                    self.units.append(Unit(big, r.first, v0, nv, r.pos0, r.pre, who, r.len, r.base, a1, b0, i0, n * (i + 1) // ns - i0, at))
                else:
                    self.units.append(Unit(2 | big, groups[~who][0], v0, nv, 0, 0, ~who, clamp(shared[~who], 0, shared_T), 0, a1, b0,
                                           i0, n * (i + 1) // ns - i0, at))
        for (who, v0, virt, _), (part, nv, ns) in zip(tiles[:own], first_part):
            r, i = reqs[who], 0
            while part >= 0 and i < nv:
                n = min(nv - i, JOIN_ROWS)
                more = (0, 0, 0)
                if r.group >= 0:
                    _, gv, tile0 = groups[r.group]
                    v, h = place[who] * G + v0 + i, height(gv)
                    n = min(n, h - v % h)
                    p, w, k = first_part[tile0 + v // h]
                    more = (p + v % h, k, w)
                self.joins.append(Join(r.first, v0 + i, n, part + i, ns, nv, *more))
                i += n


def records(work):
    """(units, joins' count, first and last row) of a plan's workspace on the host; joins() reads the joins, which begin at `at`."""
    w = work.tolist()
    units = [Unit(*w[16 + 16 * i:16 + 16 * i + 14]) for i in range(w[0])]
    return units, w[1], w[2], w[3]


def joins(work, at, n):
    w = work.tolist()
    return [Join(*w[at + 12 * i:at + 12 * i + 9]) for i in range(n)]


def at_joins(rows, B, Hq, Hkv, shared, max_rows):
    """Where a plan's joins begin in its workspace."""
    virt, most = rows * (Hq // Hkv), max_rows if 0 < max_rows < rows else rows
    h = MANY if most * (Hq // Hkv) > FEW or (shared and virt > FEW) else FEW
    tiles = virt // h + B + (virt // h + shared if shared else 0)
    return 16 + 16 * (tiles + 2 * SLOTS // Hkv + 1)
