"""Inputs and bounds of the tests of caches held in 8 bits."""

import math

import torch

from oracle import pages as OPG

DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def cache(lead, T, D, fmt, seed, spread=2.0):
    """Codes uint8 [*lead, T, D], scales fp32 [*lead, nb] and values float64, on the CPU: each block's magnitude its own
    (a factor of 2^-spread .. 2^spread), scales not powers of two."""
    g = torch.Generator().manual_seed(seed)
    nb = math.ceil(T / 64)
    x = torch.randn(*lead, nb * 64, D, generator=g, dtype=torch.float64).view(*lead, nb, 64, D)
    x = x * torch.exp2((torch.rand(*lead, nb, 1, 1, generator=g, dtype=torch.float64) * 2 - 1) * spread)
    sc = (x.abs().amax((-1, -2)) / OPG.QMAX[fmt]).float()
    codes = OPG.encode(x / sc.double()[..., None, None], fmt)
    val = OPG.decode_values(codes, fmt) * sc.double()[..., None, None]
    return (codes.view(*lead, nb * 64, D)[..., :T, :].contiguous(), sc, val.view(*lead, nb * 64, D)[..., :T, :].contiguous())


def typed(codes, fmt, device="cuda"):
    return codes.to(device).view(DTYPE[fmt])


def check_out(r, ref, q, k, v, scale, keep=None, what="", v_scale=None):
    """r: K.decode's dict (on the CPU), ref: (out, lse) in 64 bits of q, k, v (values, [B, Hkv, T, D]).
    Bounds. q is held in steps of at most 2^-21 of its head's largest element where it is not exact: off by 2^-22 of it.
    A score is then a sum of D products, each cut at 2^-23 of the largest at worst in the matrix unit, times two fp32
    factors: |ds| <= (D + 8) 2^-23 A + 2^-22 A' with A the largest scale sum |q_d k_d| and A' that of the head's largest
    |q| in every place. A weight is off by its score's error, twice (its own and the normaliser's), by 2^-11 where it is
    rounded to fp16 (with its block's scale), and by 2^-20 for v_exp_f32 and the block's factors; the sums over tokens are
    fp32 sums: 2^-17 of the sum of magnitudes for up to 128 terms in a row. So |out - ref| <= (2 ds + 2^-11 + 2^-16)
    sum p |v|, plus half a bf16 step 2^-8 |ref|.
    With v_scale ([B, Hkv, T], each token's, powers of two) also the spacing of fp16 below 2^-14, which no relative error
    covers where the heaviest tokens hold exact zeros: a weight p vs times 2^7 / 2^r is off by 2^-25 there, and the
    reference r is log2 of the largest p vs of the wavefront or at most 2^7 below it, so by 2^-32 max(p vs) of a weight, for
    each |code| = |v| / vs of the sum."""
    out, lse = ref
    B, Hq, D = q.shape
    G = Hq // k.shape[1]
    from oracle import attention as O

    A = (O.scores(q.double().abs(), k.abs(), abs(scale))).amax(-1)                     # [B, Hq]
    top = q.double().abs().amax(-1, keepdim=True).expand(B, Hq, D)
    ds = (D + 8) * 2.0 ** -23 * A + 2.0 ** -22 * O.scores(top, k.abs(), abs(scale)).amax(-1)
    absv = O.decode(q.double(), k, v.abs(), scale, keep=keep)[0]
    tol = (2 * ds[..., None] + 2.0 ** -11 + 2.0 ** -16) * absv
    if v_scale is not None:
        vs = v_scale.double().repeat_interleave(G, 1)
        top = (torch.softmax(O.scores(q.double(), k, scale), -1) * vs).amax(-1, keepdim=True)
        tol = tol + 2.0 ** -32 * top * (v.abs().repeat_interleave(G, 1) / vs[..., None]).sum(2)
    got = r["out"].double()
    bad = (got - out).abs() > tol + 2.0 ** -8 * out.abs()
    assert not bad.any(), (what, "out", (got - out).abs().max().item())
    if "out_f32" in r:
        bad = (r["out_f32"].double() - out).abs() > tol
        assert not bad.any(), (what, "out_f32", ((r["out_f32"].double() - out).abs() / absv.clamp(min=1e-300)).max().item())
    none = torch.isinf(lse)
    assert torch.equal(none, torch.isinf(r["lse"])), (what, "empty rows")
    err = torch.where(none, torch.zeros_like(lse), (r["lse"].double() - lse.nan_to_num(neginf=0.0)).abs())
    assert (err <= ds + 2.0 ** -18 * (1 + lse.nan_to_num(neginf=0.0).abs())).all(), (what, "lse", err.max().item())
    return ds


def check_stats(r, q, k, scale, ds, keep=None, what=""):
    from oracle import attention as O

    M, S = O.block_stats(q, k, scale, keep=keep)
    m, s = r["blk_max"].double(), r["blk_sum"].double()
    none = torch.isinf(M)
    assert torch.equal(none, torch.isinf(m)) and not s[none].any(), (what, "unread blocks")
    z = torch.zeros_like(M)
    em = torch.where(none, z, (m - M.nan_to_num(neginf=0.0)).abs())
    assert (em <= ds[..., None] + 2.0 ** -21 * M.nan_to_num(neginf=0.0).abs()).all(), (what, "blk_max", em.max().item())
    assert ((s - S).abs() <= (2 * ds[..., None] + 2.0 ** -18) * S).all(), (what, "blk_sum", (s - S).abs().max().item())
