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


@pytest.mark.parametrize("group", [1, 64, 128])
def test_mean_of_a_run_cut_short_is_a_quotient(cuda_lib, group):
    """A last tile of 49 keys whose mean lies 2^-24 below the middle of two bf16
    values: rounded to fp32 it is the middle, and from there the even value
    1.40625. The sum times 1 / 49 is one step of 64 bits less, and would give
    1.3984375, which another tile has."""
    s = 3 * TILE + 49
    rows = [-49 * 2.0 ** -24, 129 / 256] + [186 / 128] * 36 + [185 / 128] * 11
    rows = torch.tensor(rows, dtype=torch.float64, device="cuda")
    assert len(rows) == 49 and torch.equal(rows.bfloat16().double(), rows)
    assert (rows.sum() / torch.full_like(rows[0], 49)).float().bfloat16().item() == 1.40625
    k = torch.zeros(1, 1, s, 32, dtype=torch.bfloat16, device="cuda")
    k[0, 0, TILE:2 * TILE, 0] = 1.3984375
    k[0, 0, 3 * TILE:, 0] = rows.bfloat16()
    q = torch.zeros_like(k)
    q[..., 0] = 1
    selected = assert_definition(q, k, 1, group)
    assert selected[0, 0].tolist() == [True, False, False, True]
    # the same run as queries: its group against two tiles on either side of zero
    k2 = torch.zeros_like(k)
    k2[0, 0, :TILE, 0], k2[0, 0, :TILE, 1] = 1, -1.40234375
    k2[0, 0, TILE:2 * TILE, 0], k2[0, 0, TILE:2 * TILE, 1] = -1, 1.40234375
    q2 = torch.zeros_like(k)
    q2[..., 1] = 1
    q2[0, 0, 3 * TILE:, 0] = rows.bfloat16()
    assert_definition(q2, k2, 1, group)
