"""GPU: rows written to pages whose scale the caller brought, no power of two (kvskip_cache_write): codes are round(x / scale)
and round(code * old / new), ties to even, of the exact quotients."""

import random

import pytest
import torch

from oracle import pages as OPG
from test_gpu_pages import _slots_of, _write

pytestmark = pytest.mark.gpu


def _brought(fmt, n, seed):
    """Scales of 24 bits: amax / qmax of bf16 maxima, small odd whole numbers (quotients that are ties), random ones, and some
    below the smallest normal number."""
    rng = random.Random(seed)
    qmax = OPG.QMAX[fmt]
    s = [rng.randrange(128, 256) * 2.0 ** rng.randrange(-20, 8) / qmax for _ in range(n // 2)]
    s += [float(rng.randrange(3, 100, 2)) for _ in range(n // 4)]
    s += [rng.uniform(1, 2) * 2.0 ** rng.randrange(-70, 30) for _ in range(n - len(s) - 4)]
    s += [3e-39, 2.0 ** -130, 1e-36, 1.5 * 2.0 ** 100]
    return torch.tensor(s, dtype=torch.float32)


def _near_ties(s, fmt, D, seed):
    """bf16 rows [D] for each scale: the bf16 values next to its codes' borders."""
    g = torch.Generator().manual_seed(seed)
    grid = (torch.arange(0, 128) if fmt == "int8" else torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn)).double()
    mid = (grid[1:] + grid[:-1]) / 2
    pick = mid[torch.randint(len(mid), (len(s), D), generator=g)] * s.double()[:, None]
    sign = torch.randint(2, (len(s), D), generator=g) * 2 - 1
    return (pick * sign).float().to(torch.bfloat16)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows", [1, 7])
def test_kept_scales(gpu, fmt, rows):
    """Rows that fit the scale: one page each, from row 9 on."""
    P, D = 400, 128
    ks, vs = _brought(fmt, P, 1), _brought(fmt, P, 2)
    k, v = ([_near_ties(s, fmt, D, 10 * i + r) for r in range(rows)] for i, s in enumerate((ks, vs)))
    k, v = (torch.stack(x, 1).reshape(P * rows, 1, D) for x in (k, v))
    k[::3, 0, 5], k[::3, 0, 6], v[::3, 0, 7] = float("nan"), 0.0, -0.0
    codes = torch.randint(0, 126, (P, 1, 64, D), generator=torch.Generator().manual_seed(3)).to(torch.uint8)
    slots = [s for pg in range(P) for s in _slots_of([pg], 9, rows)]
    _, _, dks, dvs = _write(fmt, k, v, slots, codes, ks.view(P, 1), codes.clone(), vs.view(P, 1))
    assert (dks.cpu().view(-1) == ks).float().mean() > 0.8       # (borders of the largest codes round up past the scale)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows", [1, 7])
def test_grown_scales(gpu, fmt, rows):
    """Rows that do not fit: the codes that are there, every one of them, move to a power of two."""
    P, D = 200, 64
    ks, vs = _brought(fmt, P, 4), _brought(fmt, P, 5)
    grow = torch.tensor([random.Random(i).choice([1.01, 3.0, 40.0]) for i in range(P)])
    k, v = ((s * OPG.QMAX[fmt] * grow)[:, None, None].expand(P, rows, D).reshape(P * rows, 1, D).to(torch.bfloat16)
            for s in (ks, vs))
    codes = torch.arange(256, dtype=torch.uint8).repeat(16).view(1, 1, 64, D).expand(P, 1, 64, D).clone()
    slots = [s for pg in range(P) for s in _slots_of([pg], 20, rows)]
    _, _, dks, _ = _write(fmt, k, v, slots, codes, ks.view(P, 1), codes.clone(), vs.view(P, 1))
    assert (torch.frexp(dks.cpu())[0] == 0.5).float().mean() > 0.9


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_infinities(gpu, fmt):
    """An infinity is the largest code, whatever the scale; under a scale that covers every bf16 value it is kept."""
    ks = torch.tensor([[3.0], [3e38], [2.7e36]])
    k = torch.tensor([[float("inf"), -float("inf"), 5.0, -0.0] * 16] * 3, dtype=torch.bfloat16).view(3, 1, 64)
    codes = torch.full((3, 1, 64, 64), 40, dtype=torch.uint8)
    _, _, dks, _ = _write(fmt, k, -k, [9, 64 + 9, 128 + 9], codes, ks, codes.clone(), ks.clone())
    assert dks[1, 0].item() == ks[1, 0].item()
