"""GPU: weights of attention over a step's rows hold more than one fp16 part: sums of values that cancel."""

import pytest
import torch

from attend_side import Step
from test_gpu_attend_long import crowd, exact_of_one, units_of

pytestmark = pytest.mark.gpu


def cancelling(reqs, Hq, Hkv, D, fmt, seed):
    """Values of alternating sign under scores near 0, whose own bounds are small."""
    s = Step(reqs, Hq, Hkv, D, fmt, seed)
    s.q = (s.q.float() * 2.0 ** -6).to(torch.bfloat16)
    s.ks.fill_(2.0 ** (-7 if fmt == "e4m3" else -5.6))
    s.vs.copy_(torch.exp2(torch.rand(s.vs.shape, generator=torch.Generator().manual_seed(seed)) - 4))
    v = torch.zeros(s.v.shape)
    v[:, :, 0::2], v[:, :, 1::2] = 120.0, -120.0
    s.v = v.to(s.v.dtype)
    return s


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (14, 2, 64), (32, 1, 128)])
@pytest.mark.parametrize("kind", ["tokens", "prompts"])
def test_sums_that_cancel(gpu, kind, Hq, Hkv, D, fmt):
    """|out - ref| <= (2 ds + 2^-18) sum p |v| + 2^-32 max(p |vs|) sum |code| + 2^-8 |ref|, with ds the score's bound of
    attend_side.check: a weight in two fp16 parts is off by 2^-23, v_exp_f32, factors and joins by 2^-19 beside it. One fp16
    part is off by up to 2^-12 of each, which the opposite values do not take off again: with 2 to 64 keys of about equal
    weight, far over the bound in some of the thousands of results."""
    reqs = [(n, 1) for n in range(2, 66, 2)] if kind == "tokens" else [(64, 64), (130, 130), (40, 40)]
    s = cancelling(reqs, Hq, Hkv, D, fmt, 40 + Hq)
    plan = s.plan(max_rows=1 if kind == "tokens" else 0)
    for cap, slopes in ((0.0, None), (50.0, torch.full((Hq,), 2.0 ** -12))):
        out, lse, mass, reach, grain = s.exact(0, cap, slopes)
        r = s.call(plan, cap, slopes)
        ds = (D + 8) * 2.0 ** -23 * reach + (2.0 ** -22 * cap + 2.0 ** -20 * reach) * bool(cap)
        if cap:                       # below an eighth of the cap in every row: off by 2^-20 of a score, not of the cap
            assert reach.max() < cap / 8
            ds = (D + 8) * 2.0 ** -23 * reach + 2.0 ** -20 * reach
        assert (2 * ds).max() < 2.0 ** -12, "the scores' bound would cover what is tested"
        tol = (2 * ds[..., None] + 2.0 ** -18) * mass + 2.0 ** -32 * grain + 2.0 ** -8 * out.abs()
        bad = (r["out"].double().cpu() - out).abs() > tol
        assert not bad.any(), (cap, bad.sum().item(), ((r["out"].double().cpu() - out).abs() / mass.clamp(min=1e-30)).max().item())


@pytest.mark.parametrize("fmt,D", [("int8", 128), ("e4m3", 64)])
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("drop", [16, 24, 26, 28])
def test_beside_a_heavy_key_of_value_zero(gpu, drop, new, fmt, D):
    """Every key but the first has about 2^-drop of the first's weight, whose value is 0: the others' sum keeps its bits.
    A weight is off by half of fp16's finest step, 2^-25, where 2^10 stands for the heaviest p |vs| of a wavefront's keys: by 2^-35 of
    that at most, and evenly spread below it, so by 2^-35 / sqrt(3) in the root of the mean square; the sum by as much times the root of the sum
    of the codes' squares, errors of different keys being independent (a factor of 2 for what of that is not so). Beside it: half a
    bf16 step, 2^-8 / sqrt(3) of the result in the norm, the scores' errors (the first key's is one product, exact, and three
    factors: 2^-22 of it; the others' (D + 8) 2^-23 of their magnitudes), and 2^-18 for weights, exponentials and joins."""
    s = Step([(64 * 40, new)], 16, 8, D, fmt, 71)
    g = torch.Generator().manual_seed(72)
    s.q = (torch.randn(s.q.shape, generator=g) * 0.5).to(torch.bfloat16)
    s.q[..., 0] = 8.0
    k, v, p = s.k.float(), s.v.float(), s.table[0, 0]
    k[..., 0], k[p], v[p, :, 0] = 0.0, 0.0, 0.0
    k[p, :, 0, 0] = 96.0
    s.k, s.v = k.to(s.k.dtype), v.to(s.v.dtype)
    s.vs.fill_(2.0 ** -6)
    s.ks.fill_(2.0 ** -7)
    top = drop * 0.6931471805599453
    s.ks[p] = top / (s.scale * 8.0 * 96.0)
    s = crowd(s, 63)
    plan = s.plan(max_rows=new)
    assert all(u.n == 40 and u.kind == int(new > 1) for u in units_of(plan))
    out, lse, mass, reach, grain = exact_of_one(s)
    assert ((lse - top).abs() < 1.0).all()
    n, G = s.base_rows, 2
    got = s.call(plan)["out"][:n].double().cpu()
    others = s.scale * (s.base_q[..., 1:].double().abs().amax() * k[..., 1:].abs().sum(-1).amax().double() * 2.0 ** -7).item()
    ds = 2.0 ** -22 * top + (D + 8) * 2.0 ** -23 * others
    heavy = torch.exp(top - lse) * 2.0 ** -6                                  # p |vs| of the first key
    codes = v[s.base_table[0].long()].double().pow(2).sum(2).sum(0).sqrt()    # [Hkv, D]: root of the codes' squares
    finest = heavy[..., None] * codes.repeat_interleave(G, 0)[None]
    err = (got - out).norm().item()
    tol = (2 * 2.0 ** -35 / 3 ** 0.5 * finest.norm() + 2.0 ** -8 / 3 ** 0.5 * out.norm() + (2 * ds + 2.0 ** -18) * mass.norm()).item()
    assert err <= tol, (err / out.norm().item(), tol / out.norm().item())
