"""Sizes that the operators' arguments cannot hold are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_loss_refuses_sizes_beyond_int32(cuda_lib):
    """Without the refusal 2^32 + 5 columns would count as 5."""
    from tributary_b200.loss_ops import distill_loss
    target = torch.tensor(1, device="cuda")
    wide = torch.zeros(1, dtype=torch.bfloat16, device="cuda")
    for v in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="up to"):
            distill_loss(wide.expand(v), target)
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="up to"):
        distill_loss(torch.zeros(8, device="cuda"), target, ids.expand(2 ** 31), ids.float().expand(2 ** 31))
