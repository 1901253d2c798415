"""PagedCache's refusals (no GPU: every call ends before a launch)."""

import pytest
import torch

from kvskip_amd.paged import PagedCache


def test_construction():
    with pytest.raises(ValueError, match="fmt in"):
        PagedCache(1, 1, 1, 64, 1, 64, 1, "bf16", device="cpu")
    for requests in (0, 257):
        with pytest.raises(ValueError, match="requests in 1..256"):
            PagedCache(1, 1, 1, 64, requests, 64, 1, device="cpu")


def test_step_refuses_and_changes_nothing():
    c = PagedCache(1, 2, 1, 64, 3, 100, 8, device="cpu")
    assert c.T == 128 and c.block_table.shape == (3, 2)
    ones = torch.ones(3, dtype=torch.int32)
    for new, drop in ((ones.long(), None), (ones[:2], None), (ones, torch.ones(3)), (ones, torch.ones(2, dtype=torch.bool))):
        with pytest.raises(RuntimeError, match="step: new_lens int32"):
            c.step(new, drop)
        assert not c.lens.any()
