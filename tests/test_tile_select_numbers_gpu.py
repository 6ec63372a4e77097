"""Selection of key tiles where fp32 is not enough: subnormal numbers, means
that fall between two values, scores that differ by what a step of sixteen
products may lose. The choice is the definition's in 64 bits, bit for bit."""
import pytest
import torch

from test_operator_derivatives_gpu import full_plan
from test_tile_select_gpu import TILE, choose, qkv

pytestmark = pytest.mark.gpu


def assert_definition(q, k, keep, group):
    from tributary_b200.attention import select_tiles
    b, _, s, _ = q.shape
    _, plan = full_plan(b, s)
    _, selected = select_tiles(plan, q, k, keep, group)
    mask = torch.ones(b, s, s, dtype=torch.bool, device="cuda")
    want = choose(q, k, mask, keep, group)
    assert torch.equal(selected, want), (keep, group, int((selected != want).sum()))
    return selected


@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("q_scale,k_scale", [(0, -128), (-128, 0), (-60, -70), (0, -131)])
def test_subnormal_numbers_count(cuda_lib, d, q_scale, k_scale):
    """Queries or keys of 2^-126 and less, or whose means are."""
    s, h = 1100, 2
    q, k, _ = qkv(17, 1, h, s, d)
    q, k = (torch.ldexp(x.double(), torch.tensor(e, device="cuda")).bfloat16() for x, e in ((q, q_scale), (k, k_scale)))
    assert q.abs().max() > 0 and k.abs().max() > 0
    for group in (1, 2, 16, 128):
        for keep in (1, 3):
            assert_definition(q, k, keep, group)
