"""What autograd may ask of the fused operators beyond a first backward pass:
refused, not left out."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def full_plan(b, s):
    from tributary_b200.attention import build_tile_plan
    order = torch.arange(s, device="cuda", dtype=torch.int32).to(torch.int16).expand(b, s).contiguous()
    zero = torch.zeros(b, s, dtype=torch.int32, device="cuda")
    return order, build_tile_plan(order, zero, zero, zero, torch.zeros(b, 1, 1, dtype=torch.uint8, device="cuda"),
                                  "full")


def calls():
    """(operator, its differentiable inputs) of each."""
    from tributary_b200.attention import selected_attention
    from tributary_b200.layer_ops import residual_norm
    from tributary_b200.loss_ops import distill_loss
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    _, plan = full_plan(1, 300)
    ids = torch.arange(5, device="cuda").expand(6, 5)
    target = torch.arange(6, device="cuda")
    return {
        "norm": (lambda x, out, gamma, gate, post: residual_norm(x, out, gamma, 1e-6, 0.5, gate, post),
                 [normal(6, 64), normal(6, 64).bfloat16(), normal(64), normal(6, 64).bfloat16(), normal(64)]),
        "loss": (lambda z, teacher: distill_loss(z, target, ids, teacher), [normal(6, 40), normal(6, 5)]),
        "attention": (lambda q, k, v: selected_attention(q, k, v, plan, 1, 16),
                      [normal(1, 2, 300, 32).bfloat16() for _ in range(3)]),
    }


@pytest.mark.parametrize("name", ["norm", "loss", "attention"])
def test_forward_mode_is_refused(cuda_lib, name):
    call, args = calls()[name]
    call(*args)
    for i in range(len(args)):
        for recorded in (False, True):  # another input may have a backward pass
            with forward_ad.dual_level():
                given = [a.clone() for a in args]
                if recorded:
                    given[0].requires_grad_()
                given[i] = forward_ad.make_dual(given[i], torch.ones_like(given[i]))
                with pytest.raises(NotImplementedError):
                    call(*given)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    call(*given)
    call(*args)


@pytest.mark.parametrize("s", [1, 300])
def test_selected_attention_is_differentiable_once(cuda_lib, s):
    from tributary_b200.attention import selected_attention
    from tributary_b200.tokens import qk_attention
    order, plan = full_plan(1, s)
    q, k, v = (torch.randn(1, 2, s, 32, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    for call in (lambda: selected_attention(q, k, v, plan, 1, 16).float().sum(),
                 lambda: selected_attention(q, k, v, plan, 1, 16).float().square().sum()):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(call(), (q, k, v), create_graph=True)
        assert all(g.isfinite().all() for g in torch.autograd.grad(call(), (q, k, v)))
    qkv, tau = torch.randn(1, s, 3 * 64, device="cuda").bfloat16().requires_grad_(), torch.ones(2, device="cuda")
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(qk_attention(qkv, order, tau, 2, 32, plan, keep=1, group=16).float().sum(), qkv,
                            create_graph=True)


def test_attention_gradients_have_no_derivative(cuda_lib):
    """Under a plan as it is: the gradients themselves with create_graph, an
    error instead of a second derivative without the attention's part."""
    from tributary_b200.attention import rt_attention
    _, plan = full_plan(1, 200)
    q, k, v = (torch.randn(1, 2, 200, 32, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    want = torch.autograd.grad(rt_attention(q, k, v, plan).float().sum(), (q, k, v))
    got = torch.autograd.grad(rt_attention(q, k, v, plan).float().sum(), (q, k, v), create_graph=True)
    assert torch.equal(got[2], want[2])
    for a, b in zip(got[:2], want[:2]):  # dq is summed by atomic adds
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * b.float().abs().max()
    for leaf in (q, k, v):
        for g in got:
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(g.float().square().sum(), leaf, retain_graph=True)
