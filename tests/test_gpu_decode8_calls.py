"""GPU: calls of decode attention over a cache held in 8 bits that its arguments allow: scales of either sign and zero, a split
count of none."""

import pytest
import torch

from test_gpu_decode8_bits import _case, _check, _decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq", [4, 7, 16])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.1])
def test_signs(gpu, fmt, Hq, scale):
    """The softmax scale, a block's K scale and its V scale are negative, or zero."""
    q, kc, ks, k, vc, vs, v = _case(2, Hq, 1, 64, 700, fmt, Hq)
    g = torch.Generator().manual_seed(Hq)
    for s, x in ((ks, k), (vs, v)):
        f = torch.randint(-1, 2, s.shape, generator=g).float()
        s.mul_(f)
        x.mul_(f.double().repeat_interleave(64, -1)[..., :700, None])
    for S in (1, 3):
        _check(_decode(q, kc, ks, vc, vs, fmt, scale, num_splits=S), q, k, v, scale)


def test_no_splits_refused(gpu):
    q, kc, ks, k, vc, vs, v = _case(1, 2, 1, 64, 100, "int8", 1)
    for S in (0, -1):
        with pytest.raises(RuntimeError, match="num_splits in 1..256"):
            _decode(q, kc, ks, vc, vs, "int8", 1.0, num_splits=S)
    assert _decode(q, kc, ks, vc, vs, "int8", 1.0)["num_splits"] == 1
