"""The encoder's own attention over selected tiles (qk_attention with keep),
where tiles are in fact left out: against select_tiles and the selected plan,
against dense attention under the chosen mask, inside a whole training step,
and captured."""
import numpy as np
import pytest
import torch

from encoder_ref import RefOps, dense_attention, dense_masks, make_cells, tiny_config
from rt_cases import TOL_GRAD_ROW, TOL_OUT, max_rel, row_rel
from test_encoder_operators_gpu import PlainOps, device_cells, grads_of
from test_tile_select_gpu import choose, widen

pytestmark = pytest.mark.gpu

KINDS = (0, 1, 2, 3)


def sublayer(kind, s, heads, dh, seed):
    """order, plan, int64 order, dense mask, qkv, tau and an upstream gradient."""
    from tributary_b200.train import build_masks
    cells = make_cells(seed, B=2, S=s)
    t, _, _ = device_cells(cells)
    (order, plan), = build_masks(t, (kind,))
    (wide_order, mask), = dense_masks(cells, (kind,), "cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(2, s, 3 * heads * dh, device="cuda", generator=g).bfloat16()
    tau = (torch.rand(heads, device="cuda", generator=g) + 0.5) * dh ** 0.5
    return order, plan, wide_order, mask, qkv, tau, torch.randn(2, heads, s, dh, device="cuda", generator=g).bfloat16()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,heads,dh,keep,group", [(700, 2, 64, 1, 1), (700, 2, 32, 2, 32), (513, 1, 64, 1, 128),
                                                   (1100, 3, 32, 1, 16)])
def test_sublayer_over_selected_tiles(cuda_lib, kind, s, heads, dh, keep, group):
    from tributary_b200.attention import device_status, select_tiles
    from tributary_b200.tokens import qk_attention, qk_prepare
    order, plan, wide_order, mask, qkv, tau, d_o = sublayer(kind, s, heads, dh, 40 + kind)

    def run(plan, **kw):
        x, t = qkv.clone().requires_grad_(), tau.clone().requires_grad_()
        o = qk_attention(x, order, t, heads, dh, plan, **kw)
        return (o.detach(),) + torch.autograd.grad(o, (x, t), d_o)

    got = run(plan, keep=keep, group=group)
    q, k, _ = qk_prepare(qkv, order, tau, heads, dh)
    chosen_plan, selected = select_tiles(plan, q, k, keep, group)
    apart = run(chosen_plan)
    assert device_status() == 0
    # the same kernels on the same plan: the same bits, but for dq, which is summed by atomic adds
    d = heads * dh
    assert torch.equal(got[0], apart[0]) and torch.equal(got[1][..., d:], apart[1][..., d:])
    for a, b in ((got[1][..., :d], apart[1][..., :d]), (got[2], apart[2])):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max()
    # dense attention in fp32 under the mask that the definition chooses from the same q and k
    want = choose(q, k, mask, keep, group)
    assert torch.equal(selected, want)
    chosen_mask = mask & widen(want, s, group)
    if kind in (1, 3):
        assert chosen_mask.sum() < mask.sum()  # something is left out
    x, t = qkv.float().requires_grad_(), tau.clone().requires_grad_()
    rq, rk, rv = RefOps.qk_prepare(x, wide_order, t, heads, dh)
    o = dense_attention(rq, rk, rv, chosen_mask, dh ** -0.5)
    dx, dt = torch.autograd.grad(o, (x, t), d_o.float())
    assert max_rel(got[0].float().cpu().numpy(), o.detach().cpu().numpy()) < TOL_OUT
    g, ref = got[1].float().cpu().numpy(), dx.cpu().numpy()
    shape = g.shape[:2] + (3 * heads, dh)
    assert max_rel(g, ref) < TOL_OUT and row_rel(g.reshape(shape), ref.reshape(shape)) < TOL_GRAD_ROW
    # d tau of a head is the sum over its rows of <dq, q / |q|>, dq = scale sum_j P_j (dP_j - delta) k_j with |k| = 1 and
    # |dP|, |delta| <= |d_o| max |v|: terms that cancel, entirely where a row sees one key. Each rounding to bf16 is off by
    # 2^-8: of dS and P at most 2 |d_o| max |v| each, of o in delta one; of q and k it moves a score by 2 2^-8 tau scale
    # and P by that share, again of at most 2 |d_o| max |v|
    v_top = rv.norm(dim=-1).max()
    size = d_o.float().norm(dim=-1).sum(dim=(0, 2)) * v_top * dh ** -0.5
    assert ((got[2] - dt).abs() <= 2e-2 * dt.abs() + 2.0 ** -8 * (5 + 4 * tau * dh ** -0.5) * size).all()


@pytest.mark.parametrize("group", [1, 64])
def test_training_step_where_tiles_are_left_out(cuda_lib, monkeypatch, group):
    """Every option of the encoder, four tiles a sample of which two stay. The
    plain model attends under the choices of the kernels' run, each of which is
    the definition's for the q and k it was made from. Outputs within 3e-2 of
    their largest magnitude, gradients within 8e-2 of the parameter's largest
    (bf16 projections on both sides)."""
    from tributary_b200 import attention
    from tributary_b200.encoder import RTEncoder
    from tributary_b200.train import build_masks
    cells = make_cells(51, B=2, S=500, teacher_entries=5)
    t, col, cat = device_cells(cells)
    dense = dense_masks(cells, KINDS, "cuda")
    torch.manual_seed(2)
    cfg = tiny_config(kinds=KINDS, post_norm=True, select_keep=1, select_group=group, distill_weight=0.5,
                      distill_temperature=2.0)
    model = RTEncoder(cfg).cuda()
    choices, own = [], attention.select_tiles

    def select(plan, q, k, keep, size):
        got = own(plan, q, k, keep, size)
        choices.append((q, k, got[1]))
        return got

    monkeypatch.setattr(attention, "select_tiles", select)
    got = grads_of(model, t, build_masks(t, KINDS), col, cat)
    assert len(choices) == len(KINDS) and attention.device_status() == 0
    left_out = 0
    for (q, k, selected), (_, mask) in zip(choices, dense):
        assert torch.equal(selected, choose(q, k, mask, 1, group))
        left_out += int((mask & ~widen(selected, 500, group)).sum())
    assert left_out > 0

    class ChosenOps(PlainOps):
        left = [c[2] for c in choices]

        @classmethod
        def qk_attention(cls, qkv, order, tau, heads, head_dim, mask, scale, keep=None, group=128):
            return PlainOps.qk_attention(qkv, order, tau, heads, head_dim,
                                         mask & widen(cls.left.pop(0), mask.shape[1], group), scale)

    plain = RTEncoder(cfg, ChosenOps()).cuda()
    plain.load_state_dict(model.state_dict())
    want = grads_of(plain, t, dense, col, cat)
    for k in want[0]:
        top = want[0][k].float().abs().max().item()
        assert (got[0][k].float() - want[0][k].float()).abs().max().item() <= 3e-2 * top, k
    assert abs(got[1] - want[1]).item() <= 2e-2 * abs(want[1]).item()
    assert set(got[2]) == set(want[2])
    for n, w in want[2].items():
        gap = (got[2][n] - w).abs().max().item()
        assert got[2][n].isfinite().all() and gap <= 8e-2 * w.abs().max().item(), (n, gap, w.abs().max().item())


def test_captured_step_against_eager_ones(cuda_lib):
    """One graph of the whole step with every option: replayed losses are those
    of the weights before each replay, also on values copied into the batch's
    tensors, and the updates those of eager steps (dq's atomic adds make no two
    runs alike: 3e-2, as for the plain step)."""
    from tributary_b200.attention import device_status
    from tributary_b200.encoder import RTEncoder
    from tributary_b200.train import TrainStep, build_masks
    cfg = tiny_config(d_model=128, n_heads=2, d_ff=256, n_layers=2, kinds=KINDS, post_norm=True, select_keep=1,
                      select_group=16, distill_weight=0.5, distill_temperature=2.0)
    t, col, cat = device_cells(make_cells(61, B=2, S=512, teacher_entries=4))

    def fresh():
        torch.manual_seed(5)
        model = RTEncoder(cfg).cuda()
        return model, TrainStep(model, muon_lr=0.01, adamw_lr=1e-3, capturable=True)

    def loss_of(model):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            return float(model.loss(model(t, build_masks(t, KINDS), col, cat), t, cat))

    m1, s1 = fresh()
    eager = [float(s1(t, build_masks(t, KINDS), col, cat)) for _ in range(5)]
    m2, s2 = fresh()
    s2.capture(t, col, cat, KINDS, warmup=3)
    replayed = []
    for _ in range(2):
        before = loss_of(m2)
        replayed.append(float(s2.replay()))
        assert abs(replayed[-1] - before) <= 1e-5 * abs(before)  # the forward adds in a fixed order
    np.testing.assert_allclose(replayed, eager[3:], rtol=3e-2)
    with torch.no_grad():
        num = sum(float((p - q).float().norm() ** 2) for p, q in zip(m1.parameters(), m2.parameters()))
        den = sum(float(q.float().norm() ** 2) for q in m1.parameters())
    assert (num / den) ** 0.5 < 3e-2
    # each change of the batch's tensors reaches the replay
    for change in (lambda: t["teacher_logits"].mul_(-2.0),
                   lambda: t["teacher_ids"].copy_(torch.where(t["teacher_ids"] >= 0, 15 - t["teacher_ids"], -1)),
                   lambda: t["numeric_values"].mul_(3.0).add_(1.0)):
        kept = loss_of(m2)
        change()
        before = loss_of(m2)
        assert before != kept
        got = float(s2.replay())
        assert abs(got - before) <= 1e-5 * abs(before)
    assert device_status() == 0
