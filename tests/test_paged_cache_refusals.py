"""PagedCache.step's refusals leave the cache as it was (no GPU: every call ends before a launch)."""

import pytest
import torch

from kvskip_amd.paged import PagedCache


def test_refused_steps_change_nothing():
    c = PagedCache(1, 2, 1, 64, 3, 100, 8, device="cpu")
    c.lens.copy_(torch.tensor([5, 6, 7]))
    ones, off = torch.ones(3, dtype=torch.int32), torch.ones(3, dtype=torch.bool)
    for new, drop in ((torch.ones(6, dtype=torch.int32)[::2], None), (ones, torch.ones(6, dtype=torch.bool)[::2]),
                      (ones.to("meta"), None), (ones, off.to("meta")), (ones, off), (ones, None)):
        with pytest.raises(RuntimeError, match="step: new_lens int32"):
            c.step(new, drop)
        assert c.lens.tolist() == [5, 6, 7]
