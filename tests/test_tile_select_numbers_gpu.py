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


@pytest.mark.parametrize("h", [1, 64, 512])
@pytest.mark.parametrize("below", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("sign", [1, -1])
def test_products_that_fp32_steps_may_lose(cuda_lib, h, below, sign):
    """A tile whose score is 1 and then, in every later step of 16 products,
    16 of them ``below`` bits under the last place of 1 in fp32 (or 15, and one
    that just misses that place); the other tile's score lies a part of their
    sum away from 1, down to one unit. What a step loses decides the order in
    fp32, unless the near scores are compared in 64 bits."""
    d, s = 64, 3 * TILE
    n = h * d
    q = torch.full((n,), 2.0 ** -12, dtype=torch.float64)
    q[0] = 1
    for mixed in (False, True):
        product = torch.full((n,), 2.0 ** -(23 + below) * (1 - 2.0 ** -8), dtype=torch.float64)
        if mixed:
            product[15::16] = 2.0 ** -23 * (1 - 2.0 ** -8)
        product[:16] = 0
        extra = product.sum()
        for part in (0.97, 0.5, 0.1, None):
            first = sign * (product / q)
            first[0] = sign
            second = torch.zeros(n, dtype=torch.float64)
            second[0], second[1] = sign, sign * (2.0 ** -23 if part is None else part * extra) / q[1]
            k = torch.zeros(n, s, dtype=torch.float64)
            k[:, TILE:2 * TILE], k[:, 2 * TILE:] = first[:, None], second[:, None]
            k = k.view(h, d, s).transpose(1, 2)[None].bfloat16().cuda().contiguous()
            wide = q.view(h, 1, d).expand(h, s, d)[None].bfloat16().cuda().contiguous()
            assert_definition(wide, k, 1, 1)


@pytest.mark.parametrize("d,h", [(32, 3), (64, 40)])
def test_near_equal_tiles_of_mixed_exponents_and_signs(cuda_lib, d, h):
    """Keys of 2^-20 to 2^0 with both signs, every tile a copy of one whose
    few smallest components differ by one step."""
    g = torch.Generator(device="cuda").manual_seed(d)
    tiles, s = 9, 9 * TILE

    def mixed(*shape):
        e = torch.randint(-20, 1, shape, device="cuda", generator=g).double()
        return (torch.randn(*shape, device="cuda", generator=g).double() * 2 ** e).bfloat16()

    one = mixed(1, h, 1, 1, d).expand(1, h, tiles, 1, d).clone()
    small = one.abs() < 2.0 ** -12
    step = torch.randint(-1, 2, one.shape, device="cuda", generator=g).double() * 2.0 ** -7
    one = torch.where(small, (one.double() * (1 + step)).bfloat16(), one)
    k = one.expand(1, h, tiles, TILE, d).reshape(1, h, s, d).contiguous()
    q = mixed(1, h, s, d)
    for keep in (1, 4, 7):
        assert_definition(q, k, keep, 1)
        assert_definition(q, k, keep, 32)


@pytest.mark.parametrize("count", [1, 3, 5, 6, 7, 9, 11, 13, 33, 49, 63, 65, 97, 98, 100, 121, 127])
def test_means_of_every_short_run(cuda_lib, count):
    """Small whole numbers, whose sums over ``count`` rows are often a middle
    of two values or near one; sixteen tiles that differ little, the last one
    short, and its queries in groups cut short as well."""
    g = torch.Generator(device="cuda").manual_seed(count)
    s = 15 * TILE + count

    def whole(top):
        return torch.randint(-top, top + 1, (1, 2, s, 32), device="cuda", generator=g).bfloat16()

    q, k = whole(3), whole(9)
    k[:, :, 15 * TILE:] += 3
    for group in (1, 4, 32, 128):
        for keep in (1, 5):
            assert_definition(q, k, keep, group)
    k[0, 0, 15 * TILE] = float("inf")  # a sum that has no remainder
    k[0, 1, TILE] = float("-inf")
    for group in (1, 128):
        assert_definition(q, k, 2, group)


@pytest.mark.parametrize("kind,s,h,d,keeps,sizes", [(3, 900, 2, 64, (3, 1), (1, 128)), (1, 1300, 1, 32, (2, 1), (16, 1)),
                                                    (3, 700, 5, 32, (4, 2), (128, 8))])
def test_selection_from_a_selected_plan(cuda_lib, kind, s, h, d, keeps, sizes):
    """The result is a plan like any other: a second choice, by other queries
    and other groups, among the tiles that the first one left."""
    from test_tile_select_gpu import batch, check_plan, widen
    from tributary_b200.attention import select_tiles
    plan, mask = batch(s, 2, s, kind)
    q, k, _ = qkv(s, 2, h, s, d)
    for keep, size in zip(keeps, sizes):
        plan, selected = select_tiles(plan, q, k, keep, size)
        want = choose(q, k, mask, keep, size)
        assert torch.equal(selected, want)
        mask = mask & widen(want, s, size)
        check_plan(plan, mask)
        q = q.flip(-1).contiguous()
