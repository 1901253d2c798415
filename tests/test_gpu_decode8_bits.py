"""GPU: what out_f32 and lse of decode attention over a cache held in 8 bits hold (kvskip_decode8), beyond a bf16 output.

Bounds. q is held in fp16 (e4m3) or in steps of 2^-29 of its head's largest element (int8): off by 2^-30 of it. A score is a
sum of D products, each off by 2^-23 of the largest at worst, times two fp32 factors: ds = (D + 8) 2^-23 A + 2^-30 A', with A
the largest scale sum |q_d k_d| and A' that of the head's largest |q| in every place. A weight is off by its score's error,
twice (its own and the normaliser's), by 2^-22 for its two fp16 parts and by 2^-20 for v_exp_f32 and the block's factors;
sums over tokens are fp32 sums, 2^-17 of the sum of magnitudes for up to 128 terms in a row. So
|out_f32 - ref| <= (2 ds + 2^-22 + 2^-16) sum p |v|."""

import math

import pytest
import torch

from cache8_side import cache, typed
from kvskip_amd import kvskip as K
from oracle import attention as O
from oracle import pages as OPG

pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "int8"]


def _ds(q, k, scale):
    D = q.shape[-1]
    A = O.scores(q.double().abs(), k.abs(), abs(scale)).amax(-1)
    top = q.double().abs().amax(-1, keepdim=True).expand(*q.shape)
    return (D + 8) * 2.0 ** -23 * A + 2.0 ** -30 * O.scores(top, k.abs(), abs(scale)).amax(-1)


def _check(r, q, k, v, scale):
    out, lse = O.decode(q.double(), k, v, scale)
    ds = _ds(q, k, scale)
    tol = (2 * ds[..., None] + 2.0 ** -22 + 2.0 ** -16) * O.decode(q.double(), k, v.abs(), scale)[0]
    err = (r["out_f32"].cpu().double() - out).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    err = (r["lse"].cpu().double() - lse).abs()
    assert (err <= ds + 2.0 ** -18 * (1 + lse.abs())).all(), err.max().item()


def _case(B, Hq, Hkv, D, T, fmt, seed):
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    return (q, *cache((B, Hkv), T, D, fmt, seed + 1), *cache((B, Hkv), T, D, fmt, seed + 2))


def _decode(q, kc, ks, vc, vs, fmt, scale, **kw):
    return K.decode(q.cuda(), typed(kc, fmt), typed(vc, fmt), scale, k_scale=ks.cuda(), v_scale=vs.cuda(), out_f32=True, **kw)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (4, 1, 64), (7, 1, 128), (8, 1, 64), (16, 1, 128), (9, 1, 64)])
@pytest.mark.parametrize("T,S,stats", [(1, 1, False), (200, 1, True), (1537, 3, False), (1537, 1, True)])
def test_weights(gpu, fmt, Hq, Hkv, D, T, S, stats):
    q, kc, ks, k, vc, vs, v = _case(2, Hq, Hkv, D, T, fmt, T + Hq)
    _check(_decode(q, kc, ks, vc, vs, fmt, D ** -0.5, num_splits=S, stats=stats), q, k, v, D ** -0.5)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq", [2, 8, 16])
def test_one_token(gpu, fmt, Hq):
    """Each finite code alone, under a scale of 24 bits: out is their product, of a weight of 22 bits and one fp32 sum."""
    codes = torch.arange(256, dtype=torch.uint8)
    if fmt == "e4m3":
        codes = codes[(codes & 127) != 127]
    n = codes.numel()
    vc = codes.view(n, 1, 1, 1).expand(n, 1, 1, 64).contiguous()
    for vs in (0.3, 1 / 3, 7e-20, 2.0 ** -110 * 1.7):
        s = torch.full((n, 1, 1), vs)
        q = torch.randn(n, Hq, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        r = _decode(q, torch.zeros_like(vc), torch.ones(n, 1, 1), vc, s, fmt, 1.0)
        want = OPG.decode_values(codes, fmt) * float(s[0])
        got = r["out_f32"].double().cpu()
        assert ((got - want[:, None, None]).abs() <= 2.0 ** -21 * want.abs()[:, None, None]).all(), vs


@pytest.mark.parametrize("Hq", [4, 8, 16])
def test_small_elements_of_a_query(gpu, Hq):
    """One element 2^16 times the others, where K holds zeros: the others make the scores."""
    q, kc, ks, k, vc, vs, v = _case(1, Hq, 1, 64, 130, "int8", 5)
    q[..., 7] = 2.0 ** 17
    kc[..., 7], k[..., 7] = 0, 0
    _check(_decode(q, kc, ks, vc, vs, "int8", 0.125), q, k, v, 0.125)
