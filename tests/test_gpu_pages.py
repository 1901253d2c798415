"""GPU: a serving step's block tables and slot map (kvskip_page_map) and its rows into pages (kvskip_cache_write) against
the oracle, value for value: both are exact (whole numbers; codes that are roundings of exact quotients)."""

import random

import pytest
import torch

from kvskip_amd import ext as E
from oracle import pages as OPG

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def _dev(x):
    return torch.tensor(x, **I32)


def _state(rng, B, width, pages, most):
    """held pages of each request (at most `most`), table and free stack, as lists."""
    order = list(range(pages))
    rng.shuffle(order)
    held = [min(rng.randrange(most + 1), width) for _ in range(B)]
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-9] * (width - h))
        at += h
    return held, table, order[at:] + [-1] * at, pages - at


def _compare(lens, new, held, table, free, count, rows, in_place, stride=0):
    B, width = len(lens), len(table[0])
    want = OPG.page_map(lens, new, held, table, free, count, rows)
    buf = torch.full((B, width + stride), -77, **I32)
    bt = buf[:, :width]
    bt.copy_(_dev(table))
    fr, cn, hd = _dev(free), _dev([count]), _dev(held)
    slots = torch.full((rows,), -5, **I32)
    kw = {} if in_place else dict(held_out=torch.empty(B, **I32), free_count_out=torch.empty(1, **I32))
    s, starts, short = E.page_map(_dev(lens), _dev(new), hd, bt, fr, cn, slots, **kw)
    got = (slots.tolist(), starts.tolist(), int(short), bt.tolist(), fr.tolist(), kw.get("held_out", hd).tolist(),
           int(kw.get("free_count_out", cn)))
    for name, a, b in zip(("slots", "starts", "short", "table", "free", "held", "count"), got, want):
        assert a == b, name
    if stride:
        assert (buf[:, width:] == -77).all()
    if not in_place:
        assert hd.tolist() == held and int(cn) == count
    return got


@pytest.mark.parametrize("B,width,rows", [(1, 1, 1), (1, 40, 64), (7, 30, 300), (64, 20, 4096), (65, 20, 4097),
                                          (300, 12, 5000), (1025, 5, 2000), (2048, 3, 4096), (2048, 3, 9000)])
@pytest.mark.parametrize("tight", [False, True])
def test_page_map(gpu, B, width, rows, tight):
    rng = random.Random(B * 31 + rows + tight)
    pages = B * width * (1 if tight else 2) + 3
    held, table, free, count = _state(rng, B, width, pages, width)
    if tight:
        count = count // 3
        free[count:] = [-1] * (len(free) - count)
    lens, new = [], []
    for h in held:
        role = rng.random()
        n = 0 if role < 0.2 else rng.randrange(1, 64 * width + 1)
        lens.append(n)
        new.append(min(n, rng.choice([0, 1, 1, 2, 65, 200])))
    for in_place in (False, True):
        _compare(lens, new, held, table, free, count, rows, in_place, stride=3 * in_place)


def test_page_map_odd_values(gpu):
    """Lengths below zero and past the row, more new tokens than tokens, no rows, no free page."""
    held, table = [2, 1, 0, 3, 0], [[5, 1, -1, -1], [0, -1, -1, -1], [-1] * 4, [2, 3, 6, -1], [-1] * 4]
    free, count = [7, 4, 9, 8, -1, -1, -1, -1, -1, -1], 4
    for lens, new in [([-5, 300, 64, 129, 0], [3, 9, 900, -2, 4]), ([128, 64, 257, 10 ** 9, 1], [0, 1, 257, 10 ** 9, 1]),
                      ([0, 0, 0, 0, 0], [0] * 5), ([2 ** 31 - 1] * 5, [2 ** 31 - 1] * 5)]:
        for rows in (0, 1, 70, 5000):
            _compare(lens, new, held, table, free, count, rows, True)
            _compare(lens, new, held, table, free, 0, rows, False)


def test_page_map_bad_state(gpu):
    """Counts and page ids that no step leaves: nothing is read or written outside the tensors, slots stay in the pool."""
    pages, width = 6, 4
    for count in (-3, 100):
        bt = torch.full((2, width), 2 ** 30, **I32)
        fr, hd, cn = torch.full((pages,), 77, **I32), _dev([9, -4]), _dev([count])
        slots = torch.empty(256, **I32)
        E.page_map(_dev([130, 70]), _dev([130, 70]), hd, bt, fr, cn, slots)
        assert (slots == -1).all() and 0 <= int(cn) <= pages


def test_serving_steps(gpu):
    """Sixty steps in place: requests come, decode and end; no page is lost or held twice."""
    rng = random.Random(4)
    B, width, pages = 12, 9, 60
    bt, fr, cn, hd = torch.full((B, width), -1, **I32), _dev(list(range(pages))), _dev([pages]), torch.zeros(B, **I32)
    slots = torch.empty(512, **I32)
    lens = [0] * B
    state = ([0] * B, [[-1] * width for _ in range(B)], list(range(pages)), pages)
    for step in range(60):
        new, after = [], []
        for n in lens:
            if n == 0:
                a = rng.randrange(1, 200) if rng.random() < 0.4 else 0
            elif rng.random() < 0.08 or n >= 64 * width - 3:
                a = -n
            else:
                a = rng.choice([1, 1, 1, -min(n - 1, 2)])     # a step back: rejected drafts
            after.append(n + a)
            new.append(max(a, 0))
        _, starts, short = E.page_map(_dev(after), _dev(new), hd, bt, fr, cn, slots)
        held, table, free, count = state
        want = OPG.page_map(after, new, held, table, free, count, 512)
        assert slots.tolist() == want[0] and starts.tolist() == want[1] and int(short) == want[2]
        state = (want[5], want[3], want[4], want[6])
        assert hd.tolist() == state[0] and int(cn) == state[3] and bt.tolist() == state[1] and fr.tolist() == state[2]
        live = [bt[b, j].item() for b in range(B) for j in range(state[0][b])] + fr[:state[3]].tolist()
        assert sorted(live) == list(range(pages))
        # a request that was not served keeps its length (its pages do not cover more)
        lens = [n if -(-n // 64) <= state[0][b] else lens[b] for b, n in enumerate(after)]


# ---------------------------------------------------------------- cache_write

def _pool(P, Hkv, D, fmt, seed, filled=True):
    g = torch.Generator().manual_seed(seed)
    if not filled:
        return torch.full((P, Hkv, 64, D), 0x15, dtype=torch.uint8), torch.zeros(P, Hkv)
    x = torch.randn(P, Hkv, 64, D, generator=g, dtype=torch.float64)
    s = torch.tensor([[OPG.pow2_scale(float(x[p, h].abs().max()), fmt) for h in range(Hkv)] for p in range(P)])
    return OPG.encode(x / s.double()[..., None, None], fmt), s


def _typed(codes, fmt):
    return codes.cuda().view({"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[fmt])


def _canon(codes, fmt):
    """e4m3 NaN codes of either sign as one."""
    c = codes.cpu().view(torch.uint8).clone()
    if fmt == "e4m3":
        c[(c & 127) == 127] = 127
    return c


def _write(fmt, k, v, slots, kp, ks, vp, vs):
    dk, dv, dks, dvs = _typed(kp, fmt), _typed(vp, fmt), ks.cuda(), vs.cuda()
    E.cache_write(k.cuda() if not k.is_cuda else k, v.cuda() if not v.is_cuda else v, _dev(slots), dk, dv, dks, dvs)
    for x, codes, sc, d, ds in ((k, kp, ks, dk, dks), (v, vp, vs, dv, dvs)):
        codes, sc = codes.clone(), sc.clone()
        OPG.cache_write(x.cpu(), slots, codes, sc, fmt)
        assert torch.equal(ds.cpu(), sc), "scales"
        assert torch.equal(_canon(d, fmt), _canon(codes, fmt)), "codes"
    return dk, dv, dks, dvs


def _rows(N, Hkv, D, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(N, Hkv, D, generator=g) * gain).to(torch.bfloat16)


def _slots_of(pages, start, n):
    return [pages[p // 64] * 64 + p % 64 for p in range(start, start + n)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (3, 128), (8, 64)])
@pytest.mark.parametrize("start,n", [(0, 1), (0, 64), (0, 65), (63, 1), (63, 2), (10, 190), (64, 64), (1, 300), (5, 0)])
def test_write_rows(gpu, fmt, Hkv, D, start, n):
    kp, ks = _pool(8, Hkv, D, fmt, 1)
    vp, vs = _pool(8, Hkv, D, fmt, 2)
    pages = [5, 0, 7, 2, 3, 6]
    _write(fmt, _rows(n, Hkv, D, 3), _rows(n, Hkv, D, 4, 9.0), _slots_of(pages, start, n), kp, ks, vp, vs)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("N", [40, 3000])
def test_write_many_requests(gpu, fmt, N):
    """Decode steps and prompts of many requests in one map, rows without a slot between them."""
    rng = random.Random(N)
    P, Hkv, D = N + 40, 2, 64
    kp, ks = _pool(P, Hkv, D, fmt, 1)
    vp, vs = _pool(P, Hkv, D, fmt, 2)
    order = list(range(P))
    rng.shuffle(order)
    slots = []
    while len(slots) < N:
        pages = [order.pop() for _ in range(rng.choice([1, 1, 1, 3]))]
        r = rng.randrange(64)
        n = 1 if len(pages) == 1 else 64 * len(pages) - r
        slots += _slots_of(pages, r, n) + [rng.choice([-1, 64 * P, -2 ** 31, 2 ** 31 - 1])] * rng.choice([0, 0, 2])
    N = len(slots)
    _write(fmt, _rows(N, Hkv, D, 5, 3.0), _rows(N, Hkv, D, 6, 0.01), slots, kp, ks, vp, vs)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_growth(gpu, fmt):
    """A page filled row by row, each row larger than those before now and then: codes move to the larger scale."""
    D, Hkv = 64, 2
    kp, ks = _pool(2, Hkv, D, fmt, 0, filled=False)
    vp, vs = kp.clone(), ks.clone()
    dk, dv, dks, dvs = _typed(kp, fmt), _typed(vp, fmt), ks.cuda(), vs.cuda()
    rng = random.Random(1)
    for r in range(70):
        k, v = _rows(1, Hkv, D, r, 2.0 ** rng.uniform(-3, 0.1 * r)), _rows(1, Hkv, D, 1000 + r, 2.0 ** rng.uniform(-3, 1))
        slot = [64 + r if r < 64 else r - 64]
        E.cache_write(k.cuda(), v.cuda(), _dev(slot), dk, dv, dks, dvs)
        OPG.cache_write(k, slot, kp, ks, fmt)
        OPG.cache_write(v, slot, vp, vs, fmt)
        assert torch.equal(dks.cpu(), ks) and torch.equal(dvs.cpu(), vs), r
        assert torch.equal(_canon(dk, fmt), kp) and torch.equal(_canon(dv, fmt), vp), r


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_odd_values(gpu, fmt):
    """Zeros, infinities, NaN, the largest and the smallest magnitudes, borders of the scale's steps; scales that are not
    positive and finite."""
    D, Hkv = 64, 1
    inf, big = float("inf"), float(torch.finfo(torch.bfloat16).max)
    rows = [torch.zeros(D), torch.full((D,), inf), torch.full((D,), float("nan")), torch.full((D,), big),
            torch.full((D,), 1e-40), torch.full((D,), -448.0), torch.full((D,), 450.0), torch.full((D,), 127.0),
            torch.full((D,), 127.5), torch.full((D,), 2.0 ** -126), torch.linspace(-448, 448, D), torch.linspace(-1, 1, D)]
    rows[11][7] = -inf
    rows[10][3] = float("nan")
    for i, x in enumerate(rows):
        k = x.to(torch.bfloat16).view(1, 1, D)
        for was in (0.0, -1.0, float("nan"), inf, 0.5, 2.0 ** -126):
            for slot in (0, 9):
                kp, _ = _pool(1, Hkv, D, fmt, i)
                _write(fmt, k, -k, [slot], kp, torch.full((1, 1), was), kp.clone(), torch.full((1, 1), 1.0))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_repeated_slots(gpu, fmt):
    """A slot twice in a run: the last row is kept; more than 64 rows of one page: later ones come later."""
    D, Hkv = 128, 2
    rng = random.Random(2)
    for slots in ([70, 70, 71, 70], [64 + rng.randrange(64) for _ in range(64)], [64 + rng.randrange(64) for _ in range(200)]):
        kp, ks = _pool(3, Hkv, D, fmt, 1)
        vp, vs = _pool(3, Hkv, D, fmt, 2)
        n = len(slots)
        _write(fmt, _rows(n, Hkv, D, 3, 2.0), _rows(n, Hkv, D, 4, 0.5), slots, kp, ks, vp, vs)


@pytest.mark.parametrize("D", [64, 128])
def test_write_strides(gpu, D):
    """Slices of a fused projection's rows, and pools and scales that are slices of larger ones."""
    P, Hkv, N = 6, 4, 130
    qkv = _rows(N, 16 + 2 * Hkv, D, 1).cuda()
    k, v = qkv[:, 16:16 + Hkv], qkv[:, 16 + Hkv:]
    big = torch.full((P, 2, Hkv + 1, 70, D), 0x11, dtype=torch.uint8, device="cuda")
    pools = big.view(torch.float8_e4m3fn)[:, :, :Hkv, 3:67]
    sc = torch.zeros(2, Hkv, P, device="cuda").permute(2, 0, 1)
    slots = _slots_of([4, 1, 3], 30, N)
    E.cache_write(k, v, _dev(slots), pools[:, 0], pools[:, 1], sc[:, 0], sc[:, 1])
    for i, x in enumerate((k, v)):
        codes, s = torch.full((P, Hkv, 64, D), 0x11, dtype=torch.uint8), torch.zeros(P, Hkv)
        OPG.cache_write(x.cpu(), slots, codes, s, "e4m3")
        assert torch.equal(sc[:, i].cpu(), s)
        assert torch.equal(big[:, i, :Hkv, 3:67].cpu(), codes)
    assert (big[:, :, Hkv:] == 0x11).all() and (big[:, :, :, :3] == 0x11).all() and (big[:, :, :, 67:] == 0x11).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [1, 77, 5000])
def test_write_bf16(gpu, D, N):
    P, Hkv = (N + 63) // 64 + 3, 3
    k, v = _rows(N, Hkv, D, 1).cuda(), _rows(N, Hkv, D, 2).cuda()
    kp, vp = (torch.full((P, Hkv, 64, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    order = list(range(P))
    random.Random(N).shuffle(order)
    slots = _slots_of(order, 17, N)
    want_k, want_v = kp.clone(), vp.clone()
    s = torch.tensor(slots, device="cuda")
    want_k[s // 64, :, s % 64], want_v[s // 64, :, s % 64] = k, v
    E.cache_write(k, v, _dev(slots), kp, vp)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_write_pool_past_32_bits(gpu):
    """A page past 2^32 bytes of a pool."""
    P, Hkv, D = 70000, 8, 128
    pool = torch.empty(P, Hkv, 64, D, dtype=torch.int8, device="cuda")
    sc = torch.zeros(P, Hkv, device="cuda")
    k = _rows(3, Hkv, D, 1)
    slots = [(P - 1) * 64 + r for r in (0, 1, 2)]
    E.cache_write(k.cuda(), k.cuda(), _dev(slots), pool, torch.empty_like(pool), sc, sc.clone())
    codes, s = torch.zeros(1, Hkv, 64, D, dtype=torch.uint8), torch.zeros(1, Hkv)
    OPG.cache_write(k, [0, 1, 2], codes, s, "int8")
    assert torch.equal(sc[-1].cpu(), s[0])
    assert torch.equal(pool[-1, :, :3].cpu().view(torch.uint8), codes[0, :, :3])


def test_streams_and_graphs(gpu):
    """A step's map and writes captured and replayed in place, against eager steps."""
    B, width, pages, Hkv, D = 4, 8, 20, 2, 64

    def fresh():
        return dict(bt=torch.full((B, width), -1, **I32), fr=_dev(list(range(pages))), cn=_dev([pages]),
                    hd=torch.zeros(B, **I32), slots=torch.full((128,), -1, **I32), lens=torch.zeros(B, **I32),
                    new=torch.zeros(B, **I32), k=torch.zeros(128, Hkv, D, dtype=torch.bfloat16, device="cuda"),
                    kp=torch.zeros(pages, Hkv, 64, D, dtype=torch.int8, device="cuda"),
                    vp=torch.zeros(pages, Hkv, 64, D, dtype=torch.int8, device="cuda"),
                    ks=torch.zeros(pages, Hkv, device="cuda"), vs=torch.zeros(pages, Hkv, device="cuda"))

    def step(s):
        s["lens"] += s["new"]
        E.page_map(s["lens"], s["new"], s["hd"], s["bt"], s["fr"], s["cn"], s["slots"])
        E.cache_write(s["k"], s["k"], s["slots"], s["kp"], s["vp"], s["ks"], s["vs"])

    a, b = fresh(), fresh()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(b)                                        # nothing new: no row has a slot
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(b)
    for i in range(6):
        new = _dev([[30, 1, 0, 64], [1, 1, 1, 1], [1, 60, 1, 1]][min(i, 2)])
        rows = _rows(128, Hkv, D, i, 1.0 + i).cuda()
        for s in (a, b):
            s["new"].copy_(new)
            s["k"].copy_(rows)
        step(a)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x in a:
            assert torch.equal(a[x], b[x]), (i, x)
