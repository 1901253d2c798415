"""GPU: weights of attention over a step's rows hold more than one fp16 part: sums of values that cancel."""

import pytest
import torch

from attend_side import Step

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
