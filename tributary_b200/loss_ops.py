"""Autograd wrapper of the library's categorical loss with distillation: the
cross-entropy and z-loss of the categorical head
(confluence/confluence/loss.py:33-170) and the Kullback-Leibler divergence
from a teacher's top logits, one kernel each way over the student's logits.
CUDA tensors only."""
from __future__ import annotations

import torch

from . import _lib
from .attention import _any_grad, _first_order, _no_tangents, _ptr, _stream_ptr
from .layer_ops import _as

_DTYPES = {torch.float32: _lib.RT_FP32, torch.bfloat16: _lib.RT_BF16, torch.float16: _lib.RT_FP16}
_MOST = 2 ** 31 - 1  # columns and entries reach the library as int32


def _ids32(t, vocab: int):
    """int32 ids; wider ones are cut to [-1, vocab] first, so that an id no
    int32 holds stays one that names no column."""
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    return (t.clamp(-1, vocab) if t.dtype == torch.int64 else t).to(torch.int32).contiguous()


def _distill_loss(logits, target, teacher_ids, teacher_logits, *weights):
    """rt_distill_loss: the loss rows and what its backward takes."""
    logits = _as(logits, logits.dtype)
    vocab = logits.shape[-1]
    entries = 0 if teacher_ids is None else teacher_ids.shape[-1]
    loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    rows = loss.numel()
    stats = loss.new_empty(5 * rows)
    head, tail = (_DTYPES[logits.dtype], rows, vocab), (entries,) + weights
    _lib.check(_lib.load().rt_distill_loss(
        logits.data_ptr(), *head, _ptr(target), _ptr(teacher_ids), _ptr(teacher_logits), *tail, loss.data_ptr(),
        stats.data_ptr(), _stream_ptr(logits.device)), "rt_distill_loss")
    return loss, (logits, target, teacher_ids, teacher_logits, stats), (head, tail)


class DistillLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, teacher_ids, teacher_logits, *weights):
        loss, saved, ctx.args = _distill_loss(logits, target, teacher_ids, teacher_logits, *weights)
        ctx.save_for_backward(*saved)
        return loss

    @staticmethod
    def backward(ctx, grad):
        _first_order()
        logits, target, teacher_ids, teacher_logits, stats = ctx.saved_tensors
        head, tail = ctx.args
        grad = _as(grad, torch.float32)
        dlogits = torch.empty_like(logits)
        _lib.check(_lib.load().rt_distill_loss_bwd(
            logits.data_ptr(), *head, _ptr(target), _ptr(teacher_ids), _ptr(teacher_logits), *tail,
            stats.data_ptr(), grad.data_ptr(), dlogits.data_ptr(), _stream_ptr(logits.device)), "rt_distill_loss_bwd")
        return (dlogits,) + (None,) * 7


def distill_loss(logits, target=None, teacher_ids=None, teacher_logits=None, temperature: float = 1.0,
                 ce_weight: float = 1.0, z_weight: float = 0.0, kd_weight: float = 1.0):
    """fp32 loss [...] per row of ``logits`` [..., V] (fp32, bf16 or fp16):

        [target valid]  ce_weight * (l1 - logits[target]) + z_weight * l1^2
      + [a valid entry] kd_weight * T^2 * sum_e p_e * (ln p_e - logits[id_e] / T + lT)

    with l1 = logsumexp(logits), lT = logsumexp(logits / T), T = temperature
    (2^-63 <= T < 2^64) and p = softmax(teacher_logits / T) over the row's valid
    entries. ``target`` [...] and ``teacher_ids`` [..., K] are integers,
    ``teacher_logits`` [..., K] floats (K <= 128); an id outside [0, V) is not
    valid: -1 marks rows without target and pads entries. Equal ids in a row
    count each; an entry whose teacher logit is -inf is none. Rows with
    neither target nor entry have loss and gradient 0. The gradient is the
    logits', once differentiable; teacher logits are data."""
    if not logits.is_cuda or logits.dtype not in _DTYPES:
        raise TypeError("logits must be a CUDA tensor of float32, bfloat16 or float16")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., V], got {tuple(logits.shape)}")
    if logits.shape[-1] > _MOST:
        raise ValueError(f"V up to {_MOST}, got {tuple(logits.shape)}")
    if (teacher_ids is None) != (teacher_logits is None):
        raise ValueError("teacher_ids and teacher_logits come together")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    ints = (torch.int16, torch.int32, torch.int64)
    if target is not None:
        if target.dtype not in ints or target.shape != lead or target.device != logits.device:
            raise ValueError(f"target must be integers {tuple(lead)} on {logits.device}")
        target = _ids32(target, vocab)
    if teacher_ids is not None:
        if (teacher_ids.dtype not in ints or teacher_ids.shape[:-1] != lead or teacher_ids.dim() != logits.dim() or
                teacher_ids.device != logits.device):
            raise ValueError(f"teacher_ids must be integers {tuple(lead)} + (K,) on {logits.device}")
        if teacher_logits.shape != teacher_ids.shape or teacher_logits.device != logits.device:
            raise ValueError(f"teacher_logits must be {tuple(teacher_ids.shape)} on {logits.device}")
        if teacher_ids.shape[-1] > _MOST:
            raise ValueError(f"K up to {_MOST}, got {tuple(teacher_ids.shape)}")
        _no_tangents(teacher_logits)
        teacher_ids, teacher_logits = _ids32(teacher_ids, vocab), _as(teacher_logits.detach(), torch.float32)
    args = (logits, target, teacher_ids, teacher_logits, float(temperature), float(ce_weight), float(z_weight),
            float(kd_weight))
    if not _any_grad(logits):
        return _distill_loss(*args)[0]
    return DistillLossFunction.apply(*args)
