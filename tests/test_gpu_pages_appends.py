"""GPU: rows appended to part-filled pages whose scale grows (kvskip_cache_write by whole workgroups), value for value."""

import random

import pytest
import torch

from test_gpu_pages import _pool, _rows, _slots_of, _write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hkv,D", [(2, 64), (2, 128)])
def test_growing_appends(gpu, fmt, Hkv, D):
    """300 requests append 5 to 60 rows to a page that holds 1 to 60, most of them past its page's scale:
    every wavefront of a workgroup moves its share of the older rows to the larger one."""
    rng = random.Random(D)
    P = 300
    kp, ks = _pool(P, Hkv, D, fmt, 1)
    vp, vs = _pool(P, Hkv, D, fmt, 2)
    order = list(range(P))
    rng.shuffle(order)
    slots, gains = [], []
    for pg in order:
        at = rng.randrange(1, 60)
        n = min(64 - at, rng.randrange(5, 61))
        slots += _slots_of([pg], at, n)
        gains += [2.0 ** rng.choice([1, 2, 5, 9])] * n
    N = len(slots)
    gain = torch.tensor(gains).view(N, 1, 1)
    k, v = ((_rows(N, Hkv, D, s).float() * gain).to(torch.bfloat16) for s in (3, 4))
    _, _, dks, dvs = _write(fmt, k, v, slots, kp, ks, vp, vs)
    # (a gain of 2, a quarter of the pages, may stay below the next power of two)
    assert (dks.cpu() > ks).float().mean() > 0.5 and (dvs.cpu() > vs).float().mean() > 0.5
