"""What autograd may ask of the operators beyond a first backward pass, as far
as it is decided without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad


def test_tangents_are_refused_where_nothing_is_recorded():
    from tributary_b200.layer_ops import _any_grad
    x, y = torch.zeros(3), torch.zeros(2)
    assert not _any_grad(x, None, y) and _any_grad(x, None, y.clone().requires_grad_())
    with forward_ad.dual_level():
        assert not _any_grad(x, None, y)
        dual = forward_ad.make_dual(x, torch.ones(3))
        for args in ((dual,), (y, None, dual[1:])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                _any_grad(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                _any_grad(*args)
    assert not _any_grad(dual)  # its level is closed, and its tangent gone


def test_functions_take_the_arguments_they_took():
    """The autograd functions are called by name elsewhere too: what came
    later has defaults."""
    import inspect
    from tributary_b200.attention import RTAttentionFunction
    from tributary_b200.layer_ops import ResidualNormFunction
    from tributary_b200.tokens import QKAttention
    for function, given in ((RTAttentionFunction, 5), (QKAttention, 7), (ResidualNormFunction, 7)):
        inspect.signature(function.forward).bind(None, *range(given))
