"""The encoder on ops whose residual update takes the norm that follows it,
against the same encoder on ops with the two apart: the same arithmetic here,
so the same bits, however the encoder is called."""
import pytest
import torch

from encoder_ref import RefOps, dense_masks, make_cells, tiny_config, to_torch


class FusedOps(RefOps):
    @classmethod
    def residual_norm(cls, x, out, gamma, eps, scale, gate=None, post_gamma=None):
        if post_gamma is not None:
            out = cls.rms_norm(out.float(), post_gamma, eps)
        y = cls.residual_add(x, out, scale) if gate is None else cls.gate_residual(x, out, gate, scale)
        return y, cls.rms_norm(y, gamma, eps)


def models(**kw):
    from tributary_b200.encoder import RTEncoder
    torch.manual_seed(0)
    cfg = tiny_config(n_layers=2, **kw)
    fused, apart = RTEncoder(cfg, FusedOps()), RTEncoder(cfg, RefOps())
    with torch.no_grad():
        for p in fused.parameters():
            p.add_(0.1 * torch.randn_like(p))  # no two norms alike
    apart.load_state_dict(fused.state_dict())
    return fused, apart


def batch():
    cells = make_cells(3, B=1, S=64)
    return (cells,) + to_torch(cells, "cpu")


def assert_same(a, b):
    assert a.keys() == b.keys()
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("post_norm", [False, True])
@pytest.mark.parametrize("kinds,given", [((0, 3, 0), 3), ((0, 3, 0), 2), ((0, 3, 0), 1), ((0, 3, 0), 0), ((0, 3), 3),
                                         ((), 0)])
def test_fewer_and_more_masks_than_sublayers(kinds, given, post_norm):
    """Sublayers without a mask are left out, masks without a sublayer too."""
    cells, t, col, cat = batch()
    masks = dense_masks(cells, (0, 3, 0), "cpu")[:given]
    fused, apart = models(kinds=kinds, post_norm=post_norm)
    assert_same(fused(t, masks, col, cat), apart(t, masks, col, cat))


def seen_by(model, names, register):
    """What hooks on the modules ``names`` get, in order, as (name, tensors)."""
    log = []
    named = dict(model.named_modules())
    for name in names:
        def keep(module, *given, name=name):
            tensors = []
            for g in given:
                for v in g if isinstance(g, tuple) else (g,):
                    if torch.is_tensor(v):
                        tensors.append(v.detach().clone())
            log.append((name, len(given), tensors))
        getattr(named[name], register)(keep)
    return log


HOOKED = ["layers.0.attn.0.norm", "layers.0.attn.1.norm", "layers.0.ffn_norm", "layers.1.attn.0.norm", "final_norm",
          "layers.0.attn.0", "layers.0.attn.1", "layers.1.attn.0", "layers.0.ffn", "layers.0", "layers.1",
          "layers.0.attn.1.post_norm", "layers.1.ffn.post_norm"]


@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook",
                                      "register_full_backward_hook"])
@pytest.mark.parametrize("name", HOOKED + ["all"])
def test_hooks_see_what_they_see_apart(name, register):
    cells, t, col, cat = batch()
    masks = dense_masks(cells, (0, 3), "cpu")
    got = []
    for model in models(kinds=(0, 3), post_norm=True):
        log = seen_by(model, HOOKED if name == "all" else [name], register)
        out = model(t, masks, col, cat)
        model.loss(out, t, cat).backward()
        got.append((log, out, {n: p.grad for n, p in model.named_parameters() if p.grad is not None}))
    (log, out, grads), (want_log, want_out, want_grads) = got
    assert [e[:2] for e in log] == [e[:2] for e in want_log] and len(log) >= (len(HOOKED) if name == "all" else 1)
    for (_, _, a), (_, _, b) in zip(log, want_log):
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))
    assert_same(out, want_out)
    assert_same(grads, want_grads)


def test_hooks_on_every_module():
    cells, t, col, cat = batch()
    masks = dense_masks(cells, (0, 3), "cpu")
    logs = []
    for model in models(kinds=(0, 3)):
        logs.append([])
        at = {m: n for n, m in model.named_modules()}
        handle = torch.nn.modules.module.register_module_forward_hook(
            lambda m, args, out: logs[-1].append((at[m], out.detach().clone())) if torch.is_tensor(out) else None)
        try:
            model(t, masks, col, cat)
        finally:
            handle.remove()
    assert [n for n, _ in logs[0]] == [n for n, _ in logs[1]]
    assert all(torch.equal(a, b) for (_, a), (_, b) in zip(*logs))


class DoubledNorm(torch.nn.Module):
    """Stands where an RMSNorm stood, with a forward of its own."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, ops):
        return 2 * self.inner(x, ops)


class PlainFFN(torch.nn.Module):
    def __init__(self, d, output_scale):
        super().__init__()
        self.lin, self.output_scale = torch.nn.Linear(d, d), output_scale

    def forward(self, x, ops):
        return self.lin(x)


class Wrapped(torch.nn.Module):
    """A layer or sublayer called through another module."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, *args):
        return 0.5 * self.inner(x, *args)


def replace_norm(model):
    for layer in model.layers:
        layer.attn[1].norm = DoubledNorm(layer.attn[1].norm)
    model.layers[1].ffn_norm = DoubledNorm(model.layers[1].ffn_norm)


def replace_final_norm(model):
    model.final_norm = DoubledNorm(model.final_norm)


def patch_forward(model):
    norm = model.layers[1].attn[0].norm
    inner = norm.forward
    norm.forward = lambda x, ops: 3 * inner(x, ops)


def replace_ffn(model):
    torch.manual_seed(5)
    for layer in model.layers:
        layer.ffn = PlainFFN(model.cfg.d_model, 0.25)


def wrap_sublayer(model):
    model.layers[0].attn[1] = Wrapped(model.layers[0].attn[1])
    model.layers[1].attn[0] = Wrapped(model.layers[1].attn[0])


def wrap_layer(model):
    model.layers[1] = Wrapped(model.layers[1])


@pytest.mark.parametrize("change", [replace_norm, replace_final_norm, patch_forward, replace_ffn, wrap_sublayer,
                                    wrap_layer])
def test_replaced_modules_run(change):
    cells, t, col, cat = batch()
    masks = dense_masks(cells, (0, 3), "cpu")
    fused, apart = models(kinds=(0, 3))
    before = fused(t, masks, col, cat)
    for model in (fused, apart):
        change(model)
    got = fused(t, masks, col, cat)
    assert_same(got, apart(t, masks, col, cat))
    assert not torch.equal(got["num"], before["num"])


def test_ops_that_replace_the_kernels_parts():
    """Ops derived from the library's with a norm, a residual or all of their
    parts replaced: the replacements run."""
    from tributary_b200.encoder import KernelOps, RTEncoder

    class Derived(KernelOps):
        qk_attention = classmethod(lambda cls, qkv, order, tau, heads, head_dim, mask, scale: RefOps.attention(
            *RefOps.qk_prepare(qkv, order, tau, heads, head_dim), mask, scale))
        heads_unpermute, rms_norm, swiglu, gate_residual, residual_add = (
            staticmethod(getattr(RefOps, n))
            for n in ("heads_unpermute", "rms_norm", "swiglu", "gate_residual", "residual_add"))

    cells, t, col, cat = batch()
    masks = dense_masks(cells, (0, 3), "cpu")
    _, apart = models(kinds=(0, 3))
    own = RTEncoder(apart.cfg, Derived())
    own.load_state_dict(apart.state_dict())
    assert_same(own(t, masks, col, cat), apart(t, masks, col, cat))


@pytest.mark.parametrize("name", ["rms_norm", "gate_residual", "residual_add", None])
def test_fused_update_stands_for_the_librarys_own_parts(name):
    from tributary_b200.encoder import KernelOps, _fuses
    derived = type("Derived", (KernelOps,), {} if name is None else {name: staticmethod(getattr(RefOps, name))})
    assert _fuses(derived()) == _fuses(derived) == (name is None)
    derived.residual_norm = FusedOps.residual_norm  # ops with a fused update of their own
    assert _fuses(derived()) and _fuses(FusedOps()) and not _fuses(RefOps())


def test_parts_replaced_on_the_librarys_ops_themselves(monkeypatch):
    from tributary_b200.encoder import KernelOps, _fuses
    assert _fuses(KernelOps())
    monkeypatch.setattr(KernelOps, "gate_residual", staticmethod(RefOps.gate_residual))
    assert not _fuses(KernelOps())
