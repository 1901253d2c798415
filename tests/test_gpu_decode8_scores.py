"""GPU: decode attention over a cache held in 8 bits with scores from 2^4 to 2^120 (kvskip_decode8). Each head's largest score
is at least an eighth above its next, so its token has the whole weight: out_f32 is that token's value, of a weight of 22
bits and one sum, 2^-21 of itself; lse is the score, a whole number times factors of fp32 (the scale's and the block's, the
products, ln 2): 2^-21 of itself."""

import pytest
import torch

from cache8_side import typed
from kvskip_amd import kvskip as K
from oracle import pages as OPG

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,D,T,S", [(4, 64, 1000, 1), (4, 128, 1000, 3), (8, 128, 700, 1), (16, 64, 1000, 2), (16, 128, 64, 1)])
def test_large_scores(gpu, fmt, Hq, D, T, S):
    g = torch.Generator().manual_seed(Hq + D)
    nb = -(-T // 64)
    top, rest = (0x7e, 0x70) if fmt == "e4m3" else (127, 100)     # 448 and up to 256; 127 and up to 100
    for e in (6, 16, 20, 24, 28, 32, 40, 60, 100):
        kc = torch.zeros(1, 1, T, D, dtype=torch.uint8)
        kc[0, 0, :, 5] = torch.randint(0, rest + 1, (T,), generator=g).to(torch.uint8)
        plus, minus = torch.randperm(T, generator=g)[:2].tolist()
        kc[0, 0, plus, 5], kc[0, 0, minus, 5] = top, 0x80 | top if fmt == "e4m3" else 256 - top
        vc = torch.randint(0, 256, (1, 1, T, D), generator=g).to(torch.uint8)
        if fmt == "e4m3":
            vc[(vc & 127) == 127] = 3
        ks = 0.5 * (1 + 0.05 * torch.rand(1, 1, nb, generator=g))
        vs = torch.exp2(80 * torch.rand(1, 1, nb, generator=g) - 40)
        q = torch.zeros(1, Hq, D)
        q[0, :, 5] = 2.0 ** e * (1 + torch.rand(Hq, generator=g))
        q[0, 1::2] *= -1
        q = q.to(torch.bfloat16)
        r = K.decode(q.cuda(), typed(kc, fmt), typed(vc, fmt), 0.1, k_scale=ks.cuda(), v_scale=vs.cuda(), out_f32=True,
                     num_splits=S)
        val = OPG.decode_values(vc, fmt)[0, 0]
        for h in range(Hq):
            t = (plus, minus)[h % 2]
            want = val[t] * float(vs[0, 0, t // 64])
            got = r["out_f32"][0, h].cpu().double()
            assert ((got - want).abs() <= 2.0 ** -21 * want.abs()).all(), (e, h, "out")
            lse = abs(float(q[0, h, 5])) * 0.1 * (448 if fmt == "e4m3" else 127) * float(ks[0, 0, t // 64])
            assert abs(float(r["lse"][0, h]) - lse) <= 2.0 ** -21 * lse, (e, h, "lse")
