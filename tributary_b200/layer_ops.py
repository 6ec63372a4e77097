"""Autograd wrappers of the library's fused encoder-layer kernels (the
training step's non-attention work): ZeroCenteredRMSNorm
(confluence/confluence/layers.py:16-30), the gated residual of the attention
sublayer (layers.py:170-174), the SwiGLU activation (layers.py:177-200), the
FFN's residual, and a block's residual update fused with the norms before and
after it.
CUDA tensors only; each forward and backward is one kernel of
libtributary_b200.so (a second, small one sums norm gradients)."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _any_grad, _first_order, _once, _ptr, _stream_ptr


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, eps):
        x = x.float().contiguous()
        d = x.shape[-1]
        rows = x.numel() // d
        y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        g = gamma.float().contiguous()
        _lib.check(_lib.load().rt_rms_norm(_p(x), _p(g), rows, d, float(eps), _p(y), _p(rstd),
                                           _stream_ptr(x.device)), "rt_rms_norm")
        ctx.save_for_backward(x, g, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, g, rstd = ctx.saved_tensors
        lib = _lib.load()
        d = x.shape[-1]
        rows = x.numel() // d
        dy = dy.to(torch.bfloat16).contiguous()
        dx = torch.empty_like(x)
        dgamma = torch.empty_like(g)
        ws = torch.empty(lib.rt_rms_norm_bwd_workspace_bytes(rows, d), dtype=torch.uint8, device=x.device)
        _lib.check(lib.rt_rms_norm_bwd(_p(dy), _p(x), _p(g), _p(rstd), rows, d, _p(dx), _p(dgamma), _p(ws),
                                       ws.numel(), _stream_ptr(x.device)), "rt_rms_norm_bwd")
        return dx, dgamma, None


class GateResidualFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, out, gate, scale):
        x = x.float().contiguous()
        out = out.to(torch.bfloat16).contiguous()
        gate = gate.to(torch.bfloat16).contiguous()
        y = torch.empty_like(x)
        _lib.check(_lib.load().rt_gate_residual(_p(x), _p(out), _p(gate), x.numel(), float(scale), _p(y),
                                                _stream_ptr(x.device)), "rt_gate_residual")
        ctx.save_for_backward(out, gate)
        ctx.scale = scale
        return y

    @staticmethod
    def backward(ctx, dy):
        out, gate = ctx.saved_tensors
        dy = dy.float().contiguous()
        d_out = torch.empty_like(out)
        d_gate = torch.empty_like(gate)
        _lib.check(_lib.load().rt_gate_residual_bwd(_p(dy), _p(out), _p(gate), dy.numel(), float(ctx.scale),
                                                    _p(d_out), _p(d_gate), _stream_ptr(dy.device)),
                   "rt_gate_residual_bwd")
        return dy, d_out, d_gate, None


class ResidualAddFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, scale):
        x = x.float().contiguous()
        h = h.to(torch.bfloat16).contiguous()
        y = torch.empty_like(x)
        _lib.check(_lib.load().rt_residual_add(_p(x), _p(h), x.numel(), float(scale), _p(y), _stream_ptr(x.device)),
                   "rt_residual_add")
        ctx.scale = scale
        return y

    @staticmethod
    def backward(ctx, dy):
        dy = dy.float().contiguous()
        dh = torch.empty(dy.shape, dtype=torch.bfloat16, device=dy.device)
        _lib.check(_lib.load().rt_residual_add_bwd(_p(dy), dy.numel(), float(ctx.scale), _p(dh),
                                                   _stream_ptr(dy.device)), "rt_residual_add_bwd")
        return dy, dh, None


class SwiGLUFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u):
        u = u.to(torch.bfloat16).contiguous()
        f = u.shape[-1] // 2
        rows = u.numel() // u.shape[-1]
        h = torch.empty(u.shape[:-1] + (f,), dtype=torch.bfloat16, device=u.device)
        _lib.check(_lib.load().rt_swiglu(_p(u), rows, f, _p(h), _stream_ptr(u.device)), "rt_swiglu")
        ctx.save_for_backward(u)
        return h

    @staticmethod
    def backward(ctx, dh):
        (u,) = ctx.saved_tensors
        f = u.shape[-1] // 2
        rows = u.numel() // u.shape[-1]
        dh = dh.to(torch.bfloat16).contiguous()
        du = torch.empty_like(u)
        _lib.check(_lib.load().rt_swiglu_bwd(_p(dh), _p(u), rows, f, _p(du), _stream_ptr(u.device)), "rt_swiglu_bwd")
        return du


def _as(t, dtype):
    """``t`` as the kernels take it: of ``dtype``, contiguous and on a 16-byte
    boundary (itself where it is all that)."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _residual_norm(x, out, gate, gamma, post_gamma, scale, eps):
    """rt_residual_norm: y, n and what its backward takes."""
    x, out, gamma = _as(x, torch.float32), _as(out, torch.bfloat16), _as(gamma, torch.float32)
    gate = None if gate is None else _as(gate, torch.bfloat16)
    post_gamma = None if post_gamma is None else _as(post_gamma, torch.float32)
    d = x.shape[-1]
    rows = x.numel() // d
    y, n = torch.empty_like(x), torch.empty_like(out)
    rstd = gamma.new_empty(rows if post_gamma is None else 2 * rows)
    _lib.check(_lib.load().rt_residual_norm(
        x.data_ptr(), out.data_ptr(), _ptr(gate), gamma.data_ptr(), _ptr(post_gamma), rows, d, scale, eps,
        y.data_ptr(), n.data_ptr(), rstd.data_ptr(), _stream_ptr(x.device)), "rt_residual_norm")
    return y, n, (y, out, gate, gamma, post_gamma, rstd), (rows, d, scale)


class ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, out, gate, gamma, post_gamma, scale, eps, create_graph=False):
        ctx.set_materialize_grads(False)
        ctx.create_graph = create_graph
        y, n, saved, ctx.sizes = _residual_norm(x, out, gate, gamma, post_gamma, scale, eps)
        ctx.save_for_backward(*saved)
        return y, n

    @staticmethod
    def backward(ctx, dy, dn):
        if not ctx.create_graph:
            _first_order()
        y, out, gate, gamma, post_gamma, rstd = ctx.saved_tensors
        ups = dy, dn
        lib = _lib.load()
        rows, d, scale = ctx.sizes
        dy = None if dy is None else _as(dy, torch.float32)
        dn = torch.zeros_like(out) if dn is None else _as(dn, torch.bfloat16)
        dx, d_out, dgamma = torch.empty_like(y), torch.empty_like(out), torch.empty_like(gamma)
        d_gate = None if gate is None else torch.empty_like(gate)
        dpost = None if post_gamma is None else torch.empty_like(post_gamma)
        size = lib.rt_residual_norm_bwd_workspace_bytes(rows, d)
        ws = gamma.new_empty(size // 4)
        _lib.check(lib.rt_residual_norm_bwd(
            _ptr(dy), dn.data_ptr(), y.data_ptr(), out.data_ptr(), _ptr(gate), gamma.data_ptr(), _ptr(post_gamma),
            rstd.data_ptr(), rows, d, scale, dx.data_ptr(), d_out.data_ptr(), _ptr(d_gate), dgamma.data_ptr(),
            _ptr(dpost), ws.data_ptr(), size, _stream_ptr(y.device)), "rt_residual_norm_bwd")
        grads = _once((dx, d_out, d_gate, dgamma, dpost), y, gamma, post_gamma, *ups)
        return grads + (None, None, None)


def residual_norm(x, out, gamma, eps: float, scale: float, gate=None, post_gamma=None, *, create_graph: bool = False):
    """(y, n) of a block's residual update and the norm before the next block:

        z = out, or with ``post_gamma`` (1 + post_gamma) * out / sqrt(mean(out^2) + eps)
        y = x + scale * z * sigmoid(gate)        (fp32; no factor without ``gate``)
        n = (1 + gamma) * y / sqrt(mean(y^2) + eps)                         (bf16)

    x fp32, out and gate bf16, all [..., d]; gamma and post_gamma fp32 [d], d
    from 1 to 8192. Differentiable once: a backward pass with create_graph is
    refused, or with ``create_graph`` given here runs and gives gradients that
    raise when they are differentiated. Without ``post_gamma`` y and n are those of
    ``gate_residual`` (or ``residual_add``) followed by ``rms_norm``."""
    if not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    shape, device = x.shape, x.device
    if not shape or not 1 <= shape[-1] <= 8192:
        raise ValueError(f"x must be [..., d] with d from 1 to 8192, got {tuple(shape)}")
    for name, t, want in (("out", out, shape), ("gate", gate, shape), ("gamma", gamma, shape[-1:]),
                          ("post_gamma", post_gamma, shape[-1:])):
        if t is None and (name == "gate" or name == "post_gamma"):
            continue
        if t.shape != want or t.device != device:
            raise ValueError(f"{name} must be {tuple(want)} on {device}, got {tuple(t.shape)} on {t.device}")
    scale, eps = float(scale), float(eps)
    if not _any_grad(x, out, gate, gamma, post_gamma):
        return _residual_norm(x, out, gate, gamma, post_gamma, scale, eps)[:2]
    return ResidualNormFunction.apply(x, out, gate, gamma, post_gamma, scale, eps, create_graph)


def rms_norm(x, gamma, eps: float):
    """bf16 (1 + gamma) * x / sqrt(mean(x^2) + eps) of an fp32 [..., d] tensor."""
    return RMSNormFunction.apply(x, gamma, eps)


def gate_residual(x, out, gate, scale: float):
    """fp32 x + scale * out * sigmoid(gate) (out, gate: the bf16 W_O and W_gate outputs)."""
    return GateResidualFunction.apply(x, out, gate, scale)


def residual_add(x, h, scale: float):
    """fp32 x + scale * h (h: the bf16 W_down output)."""
    return ResidualAddFunction.apply(x, h, scale)


def swiglu(u):
    """bf16 silu(u[..., :f]) * u[..., f:] of the fused [..., 2f] gate / up projection."""
    return SwiGLUFunction.apply(u)
