"""Distillation from a teacher's best alternatives on the B200 CUDA library: the loss of a student whose targets are
short lists of tokens with log probabilities, as `token_logprobs(..., top_k=k)` gives them.
"""
import os

import torch
import torch.nn as nn

from . import _cabi
from .logprobs import check_temperature


def _prep(logits, top_tokens, top_logprobs, temperature):
    dev = _cabi.require_cuda(logits, top_tokens, top_logprobs)
    if top_tokens.dtype != torch.int64 or top_logprobs.dtype != torch.float32:
        raise RuntimeError("the alternatives must be int64 tokens and float32 log probabilities, got %s and %s"
                           % (top_tokens.dtype, top_logprobs.dtype))
    if logits.dim() < 1 or top_tokens.shape != top_logprobs.shape or top_tokens.dim() != logits.dim() or \
            top_tokens.shape[:-1] != logits.shape[:-1]:
        raise RuntimeError("alternatives of shapes %s and %s do not match logits %s"
                           % (tuple(top_tokens.shape), tuple(top_logprobs.shape), tuple(logits.shape)))
    if not 1 <= top_tokens.shape[-1] <= 128:
        raise RuntimeError("lists of 1 to 128 alternatives, got %d" % top_tokens.shape[-1])
    check_temperature(temperature)
    return (dev, top_tokens.contiguous(), top_logprobs.contiguous()) + _cabi.as_rows(logits)


def _value(rec, reduction):
    """The loss out of its record; no view in autograd's eyes, which would refuse `loss += other`.  (The record's
    count, which backward reads, lies elsewhere in it.)"""
    return rec[4 if reduction == 'mean' else 5].data


# (allocations by new_empty: half the host time of torch.empty with a device)
def _scratch(lib, q, rows, k):
    return q.new_empty(lib.b200_top_distill_scratch_bytes(rows, k) // 4)


def _two_pass(logits, top_tokens, top_logprobs, temperature, reduction):
    """Losses or the reduction record, and what the backward kernel needs."""
    dev, tok, q, flat, rows, v, stride = _prep(logits, top_tokens, top_logprobs, temperature)
    lib, k = _cabi.load_library(), tok.shape[-1]
    scratch = _scratch(lib, q, rows, k)
    losses = rec = None
    if reduction in ('mean', 'sum'):
        rec = q.new_empty(8)
    else:
        losses = q.new_empty(logits.shape[:-1])
    with _cabi.on_device(dev):
        _cabi.check(lib.b200_top_distill_forward(
            flat.data_ptr(), tok.data_ptr(), q.data_ptr(), _cabi.ptr(losses), _cabi.ptr(rec), scratch.data_ptr(),
            4 * scratch.numel(), rows, v, stride, _cabi.dtype_code(flat), k, temperature, _cabi.stream_ptr(dev)))
    return losses, rec, scratch, flat, tok


def _two_pass_grad(flat, tok, scratch, d_loss, per_row, count, shape, temperature):
    flat, rows, v, stride = _cabi.as_rows(flat)
    dev = flat.device
    grad = flat.new_empty(shape)
    with _cabi.on_device(dev):
        _cabi.check(_cabi.load_library().b200_top_distill_backward(
            flat.data_ptr(), tok.data_ptr(), scratch.data_ptr(), 4 * scratch.numel(), d_loss.data_ptr(), int(per_row), count,
            grad.data_ptr(), rows, v, stride, _cabi.dtype_code(flat), tok.shape[-1], temperature, _cabi.stream_ptr(dev)))
    return grad


def _step(logits, top_tokens, top_logprobs, temperature, reduction):
    """(record, final gradient) from one read of the logits, or None when this layout has no such step."""
    dev, tok, q, flat, rows, v, stride = _prep(logits, top_tokens, top_logprobs, temperature)
    lib, k, dt = _cabi.load_library(), tok.shape[-1], _cabi.dtype_code(flat)
    # (asked before the gradient is allocated, whose address ends in zeros as 0 does)
    if not lib.b200_top_distill_step_path(flat.data_ptr(), None, rows, v, stride, dt):
        return None
    grad = flat.new_empty(logits.shape)
    scratch = _scratch(lib, q, rows, k)
    rec = q.new_empty(8)
    with _cabi.on_device(dev):
        _cabi.check(lib.b200_top_distill_step(
            flat.data_ptr(), tok.data_ptr(), q.data_ptr(), grad.data_ptr(), rec.data_ptr(), scratch.data_ptr(),
            4 * scratch.numel(), rows, v, stride, dt, k, temperature, int(reduction == 'mean'), _cabi.stream_ptr(dev)))
    return rec, grad


class TopTokenDistillFunc(torch.autograd.Function):
    """(logits, top_tokens, top_logprobs, temperature, reduction) -> loss.  'mean' / 'sum' of float32 and bfloat16
    logits that need a gradient: loss and gradient come from one read of the logits, backward only applies the
    upstream gradient (a kernel that leaves at once when that is 1).  float16 logits take the two-pass form, in
    which the upstream gradient -- a loss scale as a rule -- is applied before the one rounding."""

    @staticmethod
    def forward(ctx, logits, top_tokens, top_logprobs, temperature, reduction):
        ctx.temperature, ctx.reduction, ctx.shape = temperature, reduction, logits.shape
        ctx.grad = ctx.kept = None
        if ctx.needs_input_grad[0] and reduction in ('mean', 'sum') and os.environ.get("B200_SOFTMAX_FUSED", "1") != "0":
            step = _step(logits, top_tokens, top_logprobs, temperature, reduction)
            if step is not None:
                rec, ctx.grad = step
                ctx.save_for_backward(logits, top_tokens, top_logprobs)
                return _value(rec, reduction)
        losses, rec, scratch, flat, tok = _two_pass(logits, top_tokens, top_logprobs, temperature, reduction)
        if ctx.needs_input_grad[0]:
            shared = flat.data_ptr() == logits.data_ptr()
            ctx.kept = scratch, rec
            ctx.save_for_backward(logits if shared else flat, tok)
        if reduction in ('mean', 'sum'):
            return _value(rec, reduction)
        return losses

    @staticmethod
    @_cabi.once_differentiable
    def backward(ctx, grad_output):
        if ctx.grad is not None:              # first trip through the graph: the gradient is there
            grad, ctx.grad = ctx.grad, None
            g = _cabi.scalar_gradient(grad_output)
            with _cabi.on_device(grad.device):
                _cabi.check(_cabi.load_library().b200_rescale_gradient(
                    grad.data_ptr(), g.data_ptr(), None, grad.numel(), _cabi.dtype_code(grad),
                    _cabi.stream_ptr(grad.device)))
            return grad, None, None, None, None
        if ctx.kept is not None:
            logits, tok = ctx.saved_tensors
            scratch, rec = ctx.kept
        else:                                 # a second trip: the first one scaled the gradient in place
            _, rec, scratch, logits, tok = _two_pass(*ctx.saved_tensors, ctx.temperature, ctx.reduction)
        per_row = ctx.reduction not in ('mean', 'sum')
        g = grad_output.to(torch.float32).contiguous() if per_row else _cabi.scalar_gradient(grad_output)
        count = rec.data_ptr() + _cabi.RECORD_COUNT if ctx.reduction == 'mean' else None
        return _two_pass_grad(logits, tok, scratch, g, per_row, count, ctx.shape, ctx.temperature), None, None, None, None


class TopTokenDistillLoss(nn.Module):
    """Kullback-Leibler divergence of the student from a teacher that is known by its best alternatives:

        >>> best = token_logprobs(teacher_logits, tokens, top_k=64)
        >>> criteria = TopTokenDistillLoss()
        >>> loss = criteria(student_logits, best.top_tokens, best.top_logprobs)     # [..., V], [..., K], [..., K]

    The teacher's probabilities are made to sum to one over each list; the student's are softmax(logits /
    temperature).  Entries with a negative token do not exist (lists of any length in one tensor), the same token
    twice adds up, a token beyond the vocabulary gives NaN.  A row without any entry -- or with log probabilities of
    -inf only -- costs nothing, has no gradient and does not count in the 'mean' (NaN if there is none that counts).
    'mean' and 'sum' give a float32 scalar, anything else the rows' losses.  The teacher's side has no gradient.
    """

    def __init__(self, temperature=1.0, reduction='mean'):
        super().__init__()
        check_temperature(temperature)
        self.temperature = temperature
        self.reduction = reduction

    def forward(self, logits, top_tokens, top_logprobs):
        if _cabi.tracked(logits):
            return TopTokenDistillFunc.apply(logits, top_tokens, top_logprobs, float(self.temperature), self.reduction)
        losses, rec, _, _, _ = _two_pass(logits, top_tokens, top_logprobs, float(self.temperature), self.reduction)
        return losses if rec is None else _value(rec, self.reduction)
