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
