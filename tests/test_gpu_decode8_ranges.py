"""GPU: decode attention over a cache held in 8 bits at the ends of what V's scales can be (kvskip_decode8)."""

import pytest
import torch

from kvskip_amd import kvskip as K
from oracle import attend as OA

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,Hq,D,S", [("int8", 4, 128, 2), ("int8", 4, 64, 3), ("e4m3", 4, 128, 3), ("e4m3", 32, 64, 2), ("int8", 24, 128, 2)])
@pytest.mark.parametrize("exps", [(-8, -4), (-126, -126), (-121, -101), (-130, -126), (-126, 20), (100, 118)])
def test_value_scales_of_any_size(gpu, exps, fmt, Hq, D, S):
    """From the smallest that rows are written with (and below, where fp32 holds fewer bits) to the largest. Bound of out_f32 (as
    tests/attend_side.py derives it for the same arithmetic): scores off by (D + 8) 2^-23 of their magnitudes, twice; weights
    in two parts, exponentials, factors and sums by 2^-16 of the sum of magnitudes; 2^-32 max(p |vs|) for each |code|; and fp32's
    least step, 2^-149, twice a partial result that is below 2^-126."""
    g = torch.Generator().manual_seed(44)
    B, Hkv, nb = 2, 2, 31
    T, P = nb * 64 - 17, 2 * nb
    if fmt == "int8":
        k, v = ((torch.randn(P, Hkv, 64, D, generator=g) * 40).round().clamp(-127, 127).to(torch.int8) for _ in "kv")
    else:
        k, v = ((torch.randn(P, Hkv, 64, D, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in "kv")
    ks = torch.exp2(torch.rand(P, Hkv, generator=g) * 4 - 8)
    vs = torch.ldexp(torch.ones(P, Hkv, dtype=torch.float64), torch.randint(exps[0], exps[1] + 1, (P, Hkv), generator=g)).float()
    table = torch.randperm(P, generator=g).to(torch.int32).view(B, nb)
    q = (torch.randn(B, Hq, D, generator=g) * 4).to(torch.bfloat16)          # weights far apart
    lens = [T, T - 700]
    r = K.decode(q.cuda(), k.cuda(), v.cuda(), D ** -0.5, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 block_table=table.cuda(), T=T, k_scale=ks.cuda(), v_scale=vs.cuda(), out_f32=True, num_splits=S)
    out, lse, mass, reach, grain = OA.attend(q, k, v, ks, vs, D ** -0.5, [0, 1, 2], lens, table)
    ds = (D + 8) * 2.0 ** -23 * reach
    got = r["out_f32"].double().cpu()
    tol = (2 * ds[..., None] + 2.0 ** -16) * mass + 2.0 ** -32 * grain + (2 * 4 * S + 1) * 2.0 ** -149
    bad = ~((got - out).abs() <= tol)
    assert not bad.any(), (bad.sum().item(), ((got - out).abs() / mass.clamp(min=1e-300)).max().item())
    assert ((r["lse"].double().cpu() - lse).abs() <= ds + 2.0 ** -20 * (1 + lse.abs())).all()
