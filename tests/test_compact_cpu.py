"""Arguments of the nets in microscaled storage (no GPU)."""
import pytest
import torch

from lich_amd.compact import CompactNet


@pytest.mark.parametrize("shape", [(8,), (1, 8), (4, 1), (8, 4)])
def test_targets_that_would_broadcast_are_refused(shape):
    net = CompactNet((4, 6, 5), 8, weights=[torch.zeros(4, 6), torch.zeros(6, 5)], device="cpu")
    with pytest.raises(ValueError, match="targets"):
        net.step(torch.zeros(5, 8), torch.zeros(shape))
