"""CPU: every record of a plan (tests/attend_model.py, which the GPU tests hold against the kernel's) lies inside the workspace and
the partial results that attend_sizes counts (tests/attend_sizes_check.hip), for random steps and those that push each bound."""

import ctypes
import os
import random
import subprocess

import pytest

from attend_model import Plan, at_joins
from kvskip_amd import _native
from kvskip_amd._native import AttendPlanArgs

HIPCC = "/opt/rocm/bin/hipcc"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def sizes(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc absent")
    exe = tmp_path_factory.mktemp("sizes") / "attend_sizes_check"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{ROOT}/include", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", os.path.join(ROOT, "tests", "attend_sizes_check.hip"), "-o", str(exe)], check=True,
                   capture_output=True)

    def of(cases):
        text = "".join("%d %d %d %d %d %d %d %d\n" % (c["rows"], len(c["lens"]), c["Hq"], c["Hkv"], c["T"], len(c.get("shared", ())),
                                                      c.get("shared_T", 0), c.get("max_rows", 0)) for c in cases)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout
        names = "tiles joins units parts at_units at_joins at_tiles at_rows total".split()
        return [dict(zip(names, map(int, line.split()))) for line in out.splitlines()]
    return of


def step(rng, B, news, T, Hq, Hkv, P=0, shared_T=0, **kw):
    """A step of B requests: rows drawn by news(), lengths up to T."""
    new = [news() for _ in range(B)]
    lens = [rng.choice([0, 1, 63, 64, 65, T, rng.randint(0, T), max(0, n - rng.randint(0, 3))]) for n in new]
    starts = [rng.choice([0, 0, 0, 3, -5])]
    for n in new:
        starts.append(starts[-1] + n)
    c = dict(starts=starts, lens=lens, rows=max(1, starts[-1] + rng.choice([0, 0, 7, -9])), Hq=Hq, Hkv=Hkv, T=T, **kw)
    if P:
        c.update(shared=[rng.choice([0, 1, 64, 65, shared_T, rng.randint(0, shared_T)]) for _ in range(P)], shared_T=shared_T,
                 of=[rng.randint(-1, P) for _ in range(B)])
    if rng.random() < 0.4:
        c["prefix"] = [rng.choice([0, 0, 70, T, 10 ** 6, -1]) for _ in range(B)]
    return c


def cases():
    rng = random.Random(6)
    heads = [(1, 1), (8, 8), (32, 8), (14, 2), (17, 1), (128, 1), (64, 64), (1024, 512), (600, 600), (9, 3)]
    for i in range(400):
        Hq, Hkv = rng.choice(heads)
        few = 16 // min(16, Hq // Hkv)
        news = rng.choice([lambda: 1, lambda: rng.randint(0, 3), lambda: rng.choice([1, 1, 1, rng.randint(1, 400)]), lambda: few + 1,
                           lambda: 128 // (Hq // Hkv) + 1, lambda: rng.randint(0, 900)])
        P = rng.choice([0, 0, 1, 2, 5, 64])
        yield step(rng, rng.choice([1, 2, 7, 64, 65, 150]), news, rng.choice([64, 64 * 5, 64 * 17, 64 * 500, 1 << 17, 1 << 27]), Hq, Hkv,
                   P, rng.choice([64, 640, 1 << 16]) * bool(P), max_rows=rng.choice([0, 0, 1, 2, 300]),
                   window=rng.choice([0, 0, 1, 64, 200, 5000, 2 ** 31 - 1]))
    # every tile one page over a chunk, in one round and queued; the most units of a tile; the most requests and prefixes
    for Hkv in (1, 2, 8, 64):
        for B in (1, 3, 512 // Hkv, 512 // Hkv + 1, 700):
            for per in (4, 5, 16, 17, 33, 600, 4097):
                yield dict(starts=list(range(B + 1)), lens=[64 * per] * B, rows=B, Hq=2 * Hkv, Hkv=Hkv, T=64 * per, max_rows=1)
                yield dict(starts=list(range(0, 9 * B + 1, 9)), lens=[64 * per - 63] * B, rows=9 * B, Hq=2 * Hkv, Hkv=Hkv, T=64 * per)
    B = 2048
    yield dict(starts=list(range(B + 1)), lens=[rng.randint(0, 5000) for _ in range(B)], rows=B, Hq=8, Hkv=8, T=5056, max_rows=1)
    yield dict(starts=list(range(0, 33 * B + 1, 33)), lens=[rng.randint(0, 5000) for _ in range(B)], rows=33 * B, Hq=8, Hkv=2, T=5056,
               shared=[100 + i for i in range(64)], shared_T=192, of=[b % 64 for b in range(B)])
    yield dict(starts=[0, 1 << 17], lens=[1 << 17], rows=1 << 17, Hq=8, Hkv=1, T=1 << 17)


def test_records_lie_inside_what_is_counted(sizes):
    every = [c for c in cases() if c["rows"] * c["Hq"] <= 1 << 26]     # (more is refused)
    lib, pushed = _native.lib(), dict(queued=0, most=0, split=0)
    for c, z in zip(every, sizes(every)):
        m = Plan(**c)
        what = {k: v for k, v in c.items() if not isinstance(v, list) or len(v) < 8}
        assert m.n_tiles <= z["tiles"] and len(m.units) <= z["units"] and len(m.joins) <= z["joins"] and m.parts <= z["parts"], what
        assert z["at_units"] == 16 and z["at_joins"] >= 16 + 16 * z["units"] and z["at_tiles"] >= z["at_joins"] + 12 * z["joins"], what
        assert z["at_rows"] >= z["at_tiles"] + 8 * z["tiles"] and z["total"] >= z["at_rows"] + 4 * len(m.rows), what
        assert max(z["total"], z["parts"]) < 2 ** 31 and all(z["at_" + x] % 4 == 0 for x in ("units", "joins", "tiles", "rows")), what
        assert z["at_joins"] == at_joins(c["rows"], len(c["lens"]), c["Hq"], c["Hkv"], len(c.get("shared", ())), c.get("max_rows", 0))
        p = AttendPlanArgs()
        p.B, p.rows, p.Hq, p.Hkv, p.T = len(c["lens"]), c["rows"], c["Hq"], c["Hkv"], c["T"]
        p.shared, p.shared_T, p.max_rows = len(c.get("shared", ())), c.get("shared_T", 0), c.get("max_rows", 0)
        assert lib.kvskip_attend_work_ints(ctypes.byref(p)) == z["total"], what
        assert lib.kvskip_attend_part_rows(ctypes.byref(p)) == z["parts"], what
        for u in m.units:
            assert u.part < 0 or u.part + u.nv <= m.parts
        # what is joined is written: each joined row's partial rows are those of its units, and no unit's rows are read twice
        read = [0] * m.parts
        for j in m.joins:
            assert 1 <= j.n <= 8 and j.ns + j.more_ns <= 256
            for s in range(j.ns):
                for i in range(j.n):
                    read[j.part + s * j.step + i] += 1
            for s in range(j.more_ns):
                for i in range(j.n):
                    read[j.more + s * j.more_step + i] += 1
        assert all(x == 1 for x in read), what
        pushed["queued"] += m.queued and len(m.units) > m.n_tiles
        pushed["most"] += max((j.ns for j in m.joins), default=0) == 128
        pushed["split"] += any(j.n < 8 and j.more_ns for j in m.joins)
    assert all(n >= 10 for n in pushed.values()), pushed


def test_sizes_refused():
    lib = _native.lib()
    for kw in (dict(Hq=7, Hkv=2), dict(B=0), dict(rows=0), dict(T=0), dict(B=2049), dict(shared=65, shared_T=64)):
        p = AttendPlanArgs()
        p.B, p.rows, p.Hq, p.Hkv, p.T = 3, 100, 32, 8, 4096
        for x, y in kw.items():
            setattr(p, x, y)
        assert lib.kvskip_attend_work_ints(ctypes.byref(p)) == -1 and lib.kvskip_attend_part_rows(ctypes.byref(p)) == -1
