"""Distillation from a teacher's best alternatives on the B200 CUDA library: the loss of a student whose targets are
short lists of tokens with log probabilities, as `token_logprobs(..., top_k=k)` gives them.
"""
import os

import torch
import torch.nn as nn

from . import _cabi
from .logprobs import check_temperature


def _prep(logits, top_tokens, top_logprobs, temperature):
    """What a call works on: (device, tokens, log probabilities, logits as read, rows, V, stride, K, type, scratch)."""
    dev = _cabi.require_cuda(logits, top_tokens, top_logprobs)
    if top_tokens.dtype != torch.int64 or top_logprobs.dtype != torch.float32:
        raise RuntimeError("the alternatives must be int64 tokens and float32 log probabilities, got %s and %s"
                           % (top_tokens.dtype, top_logprobs.dtype))
    shape, lists = logits.shape, top_tokens.shape
    if len(shape) < 1 or lists != top_logprobs.shape or len(lists) != len(shape) or lists[:-1] != shape[:-1]:
        raise RuntimeError("alternatives of shapes %s and %s do not match logits %s"
                           % (tuple(lists), tuple(top_logprobs.shape), tuple(shape)))
    k = lists[-1]
    if not 1 <= k <= 128:
        raise RuntimeError("lists of 1 to 128 alternatives, got %d" % k)
    check_temperature(temperature)
    flat, rows, v, stride = _cabi.as_rows(logits)
    q = top_logprobs.contiguous()
    # (allocations by new_empty: half the host time of torch.empty with a device)
    scratch = q.new_empty(_cabi.load_library().b200_top_distill_scratch_bytes(rows, k) // 4)
    return dev, top_tokens.contiguous(), q, flat, rows, v, stride, k, _cabi.dtype_code(flat), scratch


def _value(rec, reduction):
    """The loss out of its record; no view in autograd's eyes, which would refuse `loss += other`.  (The record's
    count, which backward reads, lies elsewhere in it.)"""
    return rec[4 if reduction == 'mean' else 5].data


def _two_pass(call, shape, temperature, reduction):
    """Losses of that shape or the reduction record; leaves in scratch what the backward kernel needs."""
    dev, tok, q, flat, rows, v, stride, k, dt, scratch = call
    losses = rec = None
    if reduction in ('mean', 'sum'):
        rec = q.new_empty(8)
    else:
        losses = q.new_empty(shape)
    with _cabi.on_device(dev):
        _cabi.check(_cabi.load_library().b200_top_distill_forward(
            flat.data_ptr(), tok.data_ptr(), q.data_ptr(), _cabi.ptr(losses), _cabi.ptr(rec), scratch.data_ptr(),
            4 * scratch.numel(), rows, v, stride, dt, k, temperature, _cabi.stream_ptr(dev)))
    return losses, rec


def _step(call, shape, temperature, reduction):
    """(record, final gradient) from one read of the logits, or None when this layout has no such step."""
    dev, tok, q, flat, rows, v, stride, k, dt, scratch = call
    lib = _cabi.load_library()
    # (asked before the gradient is allocated, whose address ends in zeros as 0 does)
    if not lib.b200_top_distill_step_path(flat.data_ptr(), None, rows, v, stride, dt):
        return None
    grad, rec = flat.new_empty(shape), q.new_empty(8)
    with _cabi.on_device(dev):
        _cabi.check(lib.b200_top_distill_step(
            flat.data_ptr(), tok.data_ptr(), q.data_ptr(), grad.data_ptr(), rec.data_ptr(), scratch.data_ptr(),
            4 * scratch.numel(), rows, v, stride, dt, k, temperature, int(reduction == 'mean'), _cabi.stream_ptr(dev)))
    return rec, grad


class TopTokenDistillFunc(torch.autograd.Function):
    """(logits, top_tokens, top_logprobs, temperature, reduction) -> loss.  'mean' / 'sum' of float32 and bfloat16
    logits that need a gradient: loss and gradient come from one read of the logits.  Backward is a kernel that leaves
    at once when the upstream gradient is 1; otherwise it scales a float32 gradient (a second rounding, in 32 bits) and
    writes a bfloat16 one again from the logits, for as many bytes: scaled, it would be off by a whole step.  float16
    logits take the two-pass form: their upstream gradient -- a loss scale as a rule -- is not 1."""

    @staticmethod
    def forward(ctx, logits, top_tokens, top_logprobs, temperature, reduction):
        call = _prep(logits, top_tokens, top_logprobs, temperature)
        _, tok, _, flat, _, _, _, _, _, scratch = call
        shape, reduced, need = logits.shape, reduction in ('mean', 'sum'), ctx.needs_input_grad[0]
        step = losses = grad = None
        if need and reduced and os.environ.get("B200_SOFTMAX_FUSED", "1") != "0":
            step = _step(call, shape, temperature, reduction)
        if step is not None:
            rec, grad = step
        else:
            losses, rec = _two_pass(call, shape[:-1], temperature, reduction)
        if need:
            ctx.grad, ctx.info = grad, (scratch, rec, temperature, reduction, shape)
            # (the input itself where the kernel read it, so that a change in place is noticed)
            ctx.save_for_backward(logits if flat.data_ptr() == logits.data_ptr() else flat, tok)
        return _value(rec, reduction) if reduced else losses

    @staticmethod
    @_cabi.once_differentiable
    def backward(ctx, grad_output):
        scratch, rec, temperature, reduction, shape = ctx.info
        per_row = reduction not in ('mean', 'sum')
        g = grad_output.to(torch.float32).contiguous() if per_row else _cabi.scalar_gradient(grad_output)
        lib = _cabi.load_library()
        grad, ctx.grad = ctx.grad, None       # (there on the first trip through the graph of a step)
        if grad is not None and grad.dtype is torch.float32:
            with _cabi.on_device(grad.device):
                _cabi.check(lib.b200_rescale_gradient(grad.data_ptr(), g.data_ptr(), None, grad.numel(), _cabi.F32,
                                                      _cabi.stream_ptr(grad.device)))
            return grad, None, None, None, None
        logits, tok = ctx.saved_tensors
        count = rec.data_ptr() + _cabi.RECORD_COUNT if reduction == 'mean' else None
        flat, rows, v, stride = _cabi.as_rows(logits)
        dev, k, dt = flat.device, tok.shape[-1], _cabi.dtype_code(flat)
        with _cabi.on_device(dev):
            if grad is not None:
                _cabi.check(lib.b200_top_distill_step_backward(
                    flat.data_ptr(), tok.data_ptr(), scratch.data_ptr(), 4 * scratch.numel(), g.data_ptr(), count,
                    grad.data_ptr(), rows, v, stride, dt, k, temperature, _cabi.stream_ptr(dev)))
            else:
                grad = flat.new_empty(shape)
                _cabi.check(lib.b200_top_distill_backward(
                    flat.data_ptr(), tok.data_ptr(), scratch.data_ptr(), 4 * scratch.numel(), g.data_ptr(), int(per_row),
                    count, grad.data_ptr(), rows, v, stride, dt, k, temperature, _cabi.stream_ptr(dev)))
        return grad, None, None, None, None


class TopTokenDistillLoss(nn.Module):
    """Kullback-Leibler divergence of the student from a teacher that is known by its best alternatives:

        >>> best = token_logprobs(teacher_logits, tokens, top_k=64)
        >>> criteria = TopTokenDistillLoss()
        >>> loss = criteria(student_logits, best.top_tokens, best.top_logprobs)     # [..., V], [..., K], [..., K]

    The teacher's probabilities are made to sum to one over each list; the student's are softmax(logits /
    temperature).  The temperature is the student's alone: lists are taken as they are (for both sides at T take them by
    `token_logprobs(..., temperature=T)`), and losses are not multiplied by T^2.  Entries with a negative token do not
    exist (lists of any length in one tensor); of a token that stands in a list twice both terms count in the loss, and
    its weight in the gradient is the sum; a token beyond the vocabulary gives NaN.  A row without any entry -- or with log probabilities of
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
        temperature = float(self.temperature)
        call = _prep(logits, top_tokens, top_logprobs, temperature)
        losses, rec = _two_pass(call, logits.shape[:-1], temperature, self.reduction)
        return losses if rec is None else _value(rec, self.reduction)
