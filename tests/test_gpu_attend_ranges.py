"""GPU: attention over a step's rows at the ends of what its scales can be."""

import pytest
import torch

from attend_side import Step, check

pytestmark = pytest.mark.gpu


def check_any_size(r, ref, D, what):
    """attend_side.check, for results of any size. Its bound has half a step of a bf16 as 2^-8 of the value, which holds from 2^-126 on:
    below, bf16's step is 2^-133 whatever the value, so a result rounded right is off by up to 2^-134."""
    out, lse, mass, reach, grain = ref
    ds = (D + 8) * 2.0 ** -23 * reach
    got = r["out"].double().cpu()
    tol = (2 * ds[..., None] + 2.0 ** -11 + 2.0 ** -16) * mass + 2.0 ** -32 * grain + 2.0 ** -8 * out.abs() + 2.0 ** -134
    bad = ~((got - out).abs() <= tol)
    assert not bad.any(), (what, bad.sum().item(), bad.nonzero()[:4].tolist())
    check(dict(out=ref[0], lse=r["lse"]), ref, D, what)          # (places and lse)


@pytest.mark.parametrize("fmt,Hq,Hkv,D", [("int8", 8, 2, 128), ("e4m3", 8, 2, 64)])
@pytest.mark.parametrize("exps", [(-126, -126), (-121, -101), (-130, -126), (-126, 20), (100, 118)])
def test_value_scales_of_any_size(gpu, exps, fmt, Hq, Hkv, D):
    """V's scales from the smallest that rows are written with (and below, where fp32 holds fewer bits) to the largest: as exact
    as others."""
    for most, reqs in ((0, [(64 * 9, 150), (64 * 3 + 5, 1)]), (1, [(64 * 9, 1), (64 * 30 + 5, 1)])):
        s = Step(reqs, Hq, Hkv, D, fmt, 41)
        g = torch.Generator().manual_seed(42)
        e = torch.randint(exps[0], exps[1] + 1, s.vs.shape, generator=g)
        s.vs = torch.ldexp(torch.ones(s.vs.shape, dtype=torch.float64), e).float()
        s.q *= 4                                              # weights far apart
        ref = s.exact()
        assert (s.vs > 0).all() and ref[0].isfinite().all() and (ref[2] > 0).any()
        check_any_size(s.call(s.plan(max_rows=most)), ref, D, (exps, most))


@pytest.mark.parametrize("Hq,Hkv,D,most", [(8, 2, 128, 0), (8, 2, 64, 0), (8, 2, 128, 1)])
@pytest.mark.parametrize("slopes", [False, True])
def test_caps_of_any_size(gpu, Hq, Hkv, D, most, slopes):
    """A cap far above every score changes none of them: 2^-60 of a score or less; one far below makes all of them equal."""
    s = Step([(200, 1), (300, 300 if most == 0 else 1)], Hq, Hkv, D, "e4m3", 43)
    s.k[:, :, 3] = 0.0                                        # scores of exactly 0 too
    s.k[:, :, 9] = 0.0
    sl = torch.linspace(0.01, 0.1, Hq) if slopes else None
    plan = s.plan(max_rows=most)
    for cap in (1e30, 1e37, 3.4e38):
        check(s.call(plan, cap, sl), s.exact(0, 0.0, sl), D, cap)
    for cap in (1e-50, 1e-45, 1e-38, 1e-37, 1e-30, 1e-15):
        ref = s.exact(0, cap, sl)
        check(s.call(plan, cap, sl), ref, D, cap, softcap=cap)
        assert slopes or (ref[1].exp() - ref[1].exp().round()).abs().max() < 1e-9       # (as many keys as are seen)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
def test_every_code_is_exact(gpu, fmt, D):
    """One key with scores 0 and a scale that is a power of two, whole or odd: the result is the value itself, which bf16 holds."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 127) != 127] if fmt == "e4m3" else codes
    n = codes.numel()
    for rows, most in ((1, 1), (64, 0)):
        for e in (-2, -1, 0, 5, -101):
            s = Step([(64, rows)], 4, 1, D, fmt, 45)
            s.lens, s.starts, s.rows = [1] * n, list(range(n + 1)), n
            if rows > 1:                                          # (large tiles: each request brings rows that see nothing, and one)
                s.starts, s.rows = list(range(0, 33 * n + 1, 33)), 33 * n
            s.q = torch.randn(s.rows, 4, D, generator=torch.Generator().manual_seed(46)).to(torch.bfloat16)
            s.k = torch.zeros(n, 1, 64, D, dtype=torch.uint8).view(s.k.dtype)
            s.v = codes.view(n, 1, 1, 1).expand(n, 1, 64, D).contiguous().view(s.v.dtype)
            s.ks, s.vs = torch.ones(n, 1), torch.full((n, 1), 2.0 ** e)
            s.table = torch.arange(n, dtype=torch.int32).view(n, 1)
            out = s.call(s.plan(max_rows=most))["out"].double().cpu().view(n, -1, 4, D)
            want = s.v[:, 0, 0].double()[:, None] * 2.0 ** e
            assert torch.equal(out[:, -1], want.expand(n, 4, D)) and not out[:, :-1].any(), (fmt, D, rows, e)
