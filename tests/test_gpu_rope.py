"""GPU: norms of queries and keys and their rotation (ext.norm_rope) against the 64-bit oracle."""

import pytest
import torch

from kvskip_amd import ext
from oracle import attend as OA

pytestmark = pytest.mark.gpu


def make(N, Hq, Hkv, D, rot, axes, seed, norm=True, far=131072, wide=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(N, h, D, generator=g).mul(3).to(torch.bfloat16) for h in (Hq, Hkv))
    pos = torch.randint(-2, far, (axes, N), generator=g, dtype=torch.int32)
    freq = (10000.0 ** (-2 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1))).float()
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wide) if norm else None for _ in "qk"]
    return q, k, pos, freq, w


def close(got, want, x, weight, mscale, eps):
    """Bounds: y is x times fp32 factors (the sum of squares is off by 2^-20 of itself for up to 256 terms, rsqrt by 2^-22), the
    angle exact to 2^-38 of a turn and its sine and cosine to 2^-21, two products and a sum: 2^-19 of |a| + |b|, each at
    most the head's largest |y|; and half a bf16 step, 2^-8 of the value."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -18 * max(1.0, abs(mscale)) * y.abs().amax(-1, keepdim=True)
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), (got.double().cpu() - want).abs().max().item()


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("N,Hq,Hkv,D,rot,axes", [(1, 32, 8, 128, 128, 1), (7, 4, 4, 64, 64, 1), (33, 28, 4, 128, 64, 3),
                                                 (5, 3, 1, 80, 24, 2), (19, 6, 2, 96, 96, 4), (4, 2, 1, 256, 256, 1),
                                                 (9, 5, 1, 8, 8, 1), (2049, 8, 2, 64, 32, 2), (300, 1, 1, 136, 8, 1)])
def test_against_the_formula(gpu, N, Hq, Hkv, D, rot, axes, norm, pairs):
    q, k, pos, freq, w = make(N, Hq, Hkv, D, rot, axes, N + D, norm)
    half = rot // 2
    sections = [half // axes] * (axes - 1) + [half - half // axes * (axes - 1)]
    for mscale in (1.0, 1.3):
        got = ext.norm_rope(q.cuda(), k.cuda(), (pos if axes > 1 else pos[0]).cuda(), freq.cuda(),
                            *(None if x is None else x.cuda() for x in w), eps=1e-5, sections=sections if axes > 1 else None,
                            pairs=pairs, mscale=mscale)
        for o, x, ww in zip(got, (q, k), w):
            assert o.is_contiguous() and o.shape == x.shape
            close(o, OA.norm_rope(x, pos, freq, ww, 1e-5, sections, pairs, mscale), x, ww, mscale, 1e-5)


def test_empty_sections_and_uneven_ones(gpu):
    q, k, pos, freq, w = make(40, 4, 2, 128, 128, 4, 3)
    for sections in ([0, 24, 0, 40], [64, 0, 0, 0], [1, 2, 3, 58]):
        got = ext.norm_rope(q.cuda(), k.cuda(), pos.cuda(), freq.cuda(), w[0].cuda(), w[1].cuda(), sections=sections)
        close(got[0], OA.norm_rope(q, pos, freq, w[0], 1e-6, sections), q, w[0], 1.0, 1e-6)
        close(got[1], OA.norm_rope(k, pos, freq, w[1], 1e-6, sections), k, w[1], 1.0, 1e-6)


def test_one_weight_no_k_no_positions(gpu):
    q, k, pos, freq, w = make(11, 4, 2, 64, 64, 1, 4, wide=torch.float32)
    got = ext.norm_rope(q.cuda(), k.cuda(), pos[0].cuda(), freq.cuda(), q_weight=w[0].cuda())
    close(got[0], OA.norm_rope(q, pos, freq, w[0]), q, w[0], 1.0, 1e-6)
    close(got[1], OA.norm_rope(k, pos, freq), k, None, 1.0, 1e-6)
    got = ext.norm_rope(q.cuda(), None, pos[0].cuda(), freq.cuda(), q_weight=w[0].cuda())
    assert got[1] is None
    close(got[0], OA.norm_rope(q, pos, freq, w[0]), q, w[0], 1.0, 1e-6)
    got = ext.norm_rope(q.cuda(), k.cuda(), None, None, w[0].cuda(), w[1].cuda())
    close(got[1], OA.norm_rope(k, None, None, w[1]), k, w[1], 1.0, 1e-6)
    got = ext.norm_rope(q.cuda(), k.cuda(), None, None)
    assert torch.equal(got[0].cpu(), q) and torch.equal(got[1].cpu(), k)


@pytest.mark.parametrize("N", [3, 2500])
def test_slices_in_place(gpu, N):
    """q and k as slices of a fused projection, turned in place: the bits of a call with outputs of its own, v as it was."""
    q, k, pos, freq, w = make(N, 8, 2, 128, 64, 1, 5)
    qkv = torch.cat([q, k, k], 1).cuda()
    args = pos[0].cuda(), freq.cuda(), w[0].cuda(), w[1].cuda()
    want = ext.norm_rope(q.cuda(), k.cuda(), *args)
    a, b = qkv[:, :8], qkv[:, 8:10]
    got = ext.norm_rope(a, b, *args, q_out=a, k_out=b)
    assert got[0].data_ptr() == qkv.data_ptr()
    assert torch.equal(qkv[:, :8], want[0]) and torch.equal(qkv[:, 8:10], want[1]) and torch.equal(qkv[:, 10:], k.cuda())


def test_far_positions(gpu):
    """Angles of the farthest positions an int32 holds."""
    q, k, pos, freq, _ = make(64, 2, 1, 64, 64, 1, 6, norm=False)
    pos[0] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 123456789] * 16)
    got = ext.norm_rope(q.cuda(), k.cuda(), pos[0].cuda(), freq.cuda())
    close(got[0], OA.norm_rope(q, pos, freq), q, None, 1.0, 0.0)


def test_norms_of_zeros_and_large_heads(gpu):
    q, k, pos, freq, w = make(4, 2, 1, 64, 64, 1, 7)
    q[0] = 0
    q[1] *= 2.0 ** 40
    got = ext.norm_rope(q.cuda(), k.cuda(), pos[0].cuda(), freq.cuda(), w[0].cuda(), w[1].cuda())
    close(got[0], OA.norm_rope(q, pos, freq, w[0]), q, w[0], 1.0, 1e-6)
    assert not got[0][0].any()


def test_captured(gpu):
    q, k, pos, freq, w = (x if isinstance(x, list) else x.cuda() for x in make(50, 8, 2, 128, 128, 3, 8))
    w = [x.cuda() for x in w]
    run = lambda: ext.norm_rope(q, k, pos, freq, *w, sections=[16, 24, 24])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run()
    for i in range(3):
        q.mul_(-1), pos.add_(7)
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(x, y) for x, y in zip(got, run()))


def test_outputs_that_overlap(gpu):
    """Slices of one buffer that share no element are served; an output over the other input, the other output or itself is not."""
    q, k, pos, freq, w = make(5, 4, 2, 64, 64, 1, 9)
    args = pos[0].cuda(), freq.cuda(), w[0].cuda(), w[1].cuda()
    want = ext.norm_rope(q.cuda(), k.cuda(), *args)
    qkv = torch.cat([q, k, k, q], 1).cuda()                    # [5, 12, 64]
    a, b = qkv[:, :4], qkv[:, 4:6]
    ext.norm_rope(a, b, *args, q_out=qkv[:, 8:], k_out=qkv[:, 6:8])
    assert torch.equal(qkv[:, 8:], want[0]) and torch.equal(qkv[:, 6:8], want[1])
    assert torch.equal(qkv[:, :4], q.cuda()) and torch.equal(qkv[:, 4:6], k.cuda())
    both = torch.zeros(4 + 2, 5, 64, dtype=torch.bfloat16, device="cuda")
    ext.norm_rope(a, b, *args, q_out=both[:4].transpose(0, 1), k_out=both[4:].transpose(0, 1))
    assert torch.equal(both[:4].transpose(0, 1), want[0]) and torch.equal(both[4:].transpose(0, 1), want[1])
    kept = qkv.clone()
    for kw in (dict(q_out=qkv[:, 3:7]), dict(q_out=qkv[:, 1:5]), dict(k_out=qkv[:, 3:5]), dict(k_out=qkv[:, 5:7]),
               dict(q_out=qkv[:, 6:10], k_out=qkv[:, 8:10]), dict(q_out=a[:1].expand(5, 4, 64)),
               dict(k_out=both[:1].transpose(0, 1).expand(5, 2, 64))):
        with pytest.raises(RuntimeError, match="norm_rope: an output"):
            ext.norm_rope(a, b, *args, **kw)
    assert torch.equal(qkv, kept)
