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


def test_encoder_backward_with_create_graph(cuda_lib):
    """The gradients that it has without, and an error instead of second
    derivatives that leave the kernels' parts out."""
    from encoder_ref import make_cells, tiny_config, to_torch
    from tributary_b200.encoder import RTEncoder
    from tributary_b200.train import build_masks
    t, col, cat = to_torch(make_cells(7, B=2, S=128), "cuda")
    torch.manual_seed(1)
    model = RTEncoder(tiny_config(n_layers=2, post_norm=True)).cuda()
    params = [p for n, p in model.named_parameters()]

    def loss():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return model.loss(model(t, build_masks(t, (0, 1, 2, 3)), col, cat), t, cat)

    want = torch.autograd.grad(loss(), params, allow_unused=True)
    again = torch.autograd.grad(loss(), params, allow_unused=True)
    got = torch.autograd.grad(loss(), params, allow_unused=True, create_graph=True)
    for a, b, c in zip(got, want, again):
        assert (a is None) == (b is None)
        if a is not None:  # the atomic adds of dq make no two runs alike
            assert (a - b).abs().max() <= 8 * (c - b).abs().max() + 2.0 ** -8 * b.abs().max()
    norm = sum(g.float().square().sum() for g in got if g is not None)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(norm, params, allow_unused=True)


def test_residual_norm_with_create_graph(cuda_lib):
    from tributary_b200.layer_ops import residual_norm
    x, out, gate = (torch.randn(5, 64, device="cuda") for _ in range(3))
    leaves = [x, out.bfloat16(), torch.randn(64, device="cuda"), gate.bfloat16(), torch.randn(64, device="cuda")]
    for leaf in leaves:
        leaf.requires_grad_()
    x, out, gamma, gate, post = leaves

    def total(**kw):
        y, n = residual_norm(x, out, gamma, 1e-6, 0.5, gate, post, **kw)
        return y.square().sum() + n.float().sum()

    want = torch.autograd.grad(total(), leaves)
    got = torch.autograd.grad(total(create_graph=True), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for g in got:
        for leaf in leaves:
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(g.float().sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="create_graph is not supported"):
        torch.autograd.grad(total(), leaves, create_graph=True)
