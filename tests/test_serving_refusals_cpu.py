"""What the serving entry points refuse, or leave as it was, before anything reaches a GPU."""

import pytest
import torch

from tiktok_techjam_2026_track3_b200 import ops


def test_workspaces_that_would_be_used_are_dense_and_on_the_device():
    """The kernels get a workspace's address alone."""
    here, there = torch.device("cpu"), torch.device("cuda", 0)
    own = torch.empty(64, dtype=torch.float32)
    assert ops._workspace(own, 256, here) is own
    assert ops._workspace(own, 0, here) is own
    fresh = ops._workspace(own, 257, here)                    # too small: replaced, as without one
    assert fresh.numel() == 257 and fresh.dtype == torch.uint8
    assert ops._workspace(None, 8, here).numel() == 8
    for bad, need in ((own, 256), (torch.empty(64), 1)):      # a host address
        with pytest.raises(RuntimeError, match="workspace must be a contiguous tensor on cuda:0"):
            ops._workspace(bad, need, there)
    for bad in (own[::2], torch.empty(1).expand(64), torch.empty(8, 8)[:, :4]):
        with pytest.raises(RuntimeError, match="workspace must be a contiguous"):
            ops._workspace(bad, bad.numel() * 4, here)
