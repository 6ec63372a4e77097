"""What the categorical loss keeps for its backward is set by its inputs alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,v", [(600, 300), (600, 20001), (3, 100003)])
def test_rows_without_a_teacher_keep_the_same_statistics(cuda_lib, rows, v):
    """A row for each of the kernel's forms (a warp, a block, a cluster of
    blocks), after calls whose teachers leave something else behind."""
    from tributary_b200.loss_ops import _distill_loss
    weights = (2.0, 0.7, 1e-2, 0.6)
    z = torch.randn(rows, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(v))
    target = torch.arange(rows, dtype=torch.int32, device="cuda")
    ids = torch.arange(8, dtype=torch.int32, device="cuda").expand(rows, 8).contiguous()
    none = torch.full_like(ids, -1)
    kept = []
    for top in (7.5, 1e4):
        teacher = torch.full((rows, 8), top, device="cuda")
        _distill_loss(z, target, ids, teacher, *weights)
        kept.append(_distill_loss(z, target, none, teacher, *weights)[1][-1])
        _distill_loss(z, target, ids, teacher, *weights)
        kept.append(_distill_loss(z, target, None, None, *weights)[1][-1])
    for stats in kept:
        assert torch.equal(stats, kept[0])
        assert (stats[4 * rows:] == 0).all() and not stats.isnan().any()
