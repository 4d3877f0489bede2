"""Log probabilities of given tokens, with the entropy and the best alternatives of every row, on the B200 CUDA
library: what scoring, sampling and policy training read off a language model's logits.  One pass over the logits
forward, one more with the gradient's write backward; nothing of the vocabulary's size is kept in between.
"""
from typing import NamedTuple, Optional

import torch

from . import _cabi


class TokenLogProbs(NamedTuple):
    """What `token_logprobs` returns; the last two are None unless alternatives were asked for."""
    logprobs: torch.Tensor                  # float32, the tokens' shape
    entropy: torch.Tensor                   # float32, the tokens' shape, in nats
    top_logprobs: Optional[torch.Tensor]    # float32 [..., top_k], largest first
    top_tokens: Optional[torch.Tensor]      # int64 [..., top_k]


def _check(logits, tokens, top_k, temperature):
    dev = _cabi.require_cuda(logits, tokens)
    if tokens.dtype != torch.int64:
        raise RuntimeError("tokens must be int64, got %s" % tokens.dtype)
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise RuntimeError("tokens shape %s does not match logits %s (expected %s)"
                           % (tuple(tokens.shape), tuple(logits.shape), tuple(logits.shape[:-1])))
    if not 0 <= top_k <= min(128, logits.shape[-1]):
        raise ValueError("top_k must lie between 0 and 128 and not exceed the vocabulary, got %s" % (top_k,))
    check_temperature(temperature)
    return dev


def check_temperature(temperature):
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError("temperature must lie between 1e-4 and 1e4, got %s" % (temperature,))


def _forward(dev, logits, tokens, top_k, temperature, ignore_index, want_stats):
    flat, rows, v, stride = _cabi.as_rows(logits)
    dt = _cabi.dtype_code(flat)
    shape = tokens.shape
    tokens = tokens.contiguous()
    # (allocations by *_like and new_empty: half the host time of torch.empty with a device)
    logprobs = tokens.new_empty(shape, dtype=torch.float32)
    entropy = torch.empty_like(logprobs)
    top_lp = top_tok = stats = None
    if top_k:
        top_lp = logprobs.new_empty(shape + (top_k,))
        top_tok = tokens.new_empty(shape + (top_k,))
    if want_stats:
        stats = logprobs.new_empty((rows, 4))
    lib = _cabi.load_library()
    with _cabi.on_device(dev):
        _cabi.check(lib.b200_token_logprobs(
            flat.data_ptr(), tokens.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(), _cabi.ptr(stats),
            _cabi.ptr(top_lp), _cabi.ptr(top_tok), rows, v, stride, dt, top_k, temperature, ignore_index,
            _cabi.stream_ptr(dev)))
    return flat, tokens, logprobs, entropy, top_lp, top_tok, stats


class TokenLogProbsFunc(torch.autograd.Function):
    """(logits, tokens, top_k, temperature, ignore_index) -> logprobs, entropy, top_logprobs, top_tokens.  The
    alternatives carry no gradient."""

    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        dev = _check(logits, tokens, top_k, temperature)
        flat, tok, logprobs, entropy, top_lp, top_tok, stats = _forward(
            dev, logits, tokens, top_k, temperature, ignore_index, ctx.needs_input_grad[0])
        if ctx.needs_input_grad[0]:
            # (the input itself where the kernel read it, so that a change in place is noticed)
            shared = flat.data_ptr() == logits.data_ptr()
            ctx.save_for_backward(logits if shared else flat, tok, stats)
            ctx.info = logits.shape, temperature, ignore_index
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top_lp, top_tok)
        return logprobs, entropy, top_lp, top_tok

    @staticmethod
    @_cabi.once_differentiable
    def backward(ctx, d_logprobs, d_entropy, _top_logprobs, _top_tokens):
        if d_logprobs is None and d_entropy is None:
            return None, None, None, None, None
        logits, tokens, stats = ctx.saved_tensors
        flat, rows, v, stride = _cabi.as_rows(logits)
        dev = flat.device
        if d_logprobs is not None:
            d_logprobs = d_logprobs.contiguous()
        if d_entropy is not None:
            d_entropy = d_entropy.contiguous()
        grad = flat.new_empty(ctx.info[0])
        with _cabi.on_device(dev):
            _cabi.check(_cabi.load_library().b200_token_logprobs_backward(
                flat.data_ptr(), tokens.data_ptr(), stats.data_ptr(), _cabi.ptr(d_logprobs), _cabi.ptr(d_entropy),
                grad.data_ptr(), rows, v, stride, _cabi.dtype_code(flat), ctx.info[1], ctx.info[2],
                _cabi.stream_ptr(dev)))
        return grad, None, None, None, None


def token_logprobs(logits, tokens, top_k=0, temperature=1.0, ignore_index=-100):
    """Log probability of one given token per row, entropy and the `top_k` best alternatives:

        >>> out = token_logprobs(logits, tokens, top_k=20)      # logits [..., V] float/half/bfloat16, tokens [...] int64
        >>> (out.logprobs * advantage - 0.01 * out.entropy).sum().backward()

    of softmax(logits / temperature).  Log probabilities and entropies are float32 and have gradients; alternatives
    (at most 128, largest first, equal logits by index) have none.  Rows whose token is `ignore_index` are not read:
    0, 0, and for the alternatives 0 and -1.  A token outside the vocabulary gives NaN, a row of -inf alone -inf and
    entropy 0 with a zero gradient.  Masked logits (-inf or the type's lowest value) are fine; a NaN makes its row
    NaN.  Rows may lie apart in memory (`logits[..., :vocabulary]` of a padded head).
    """
    top_k, temperature, ignore_index = int(top_k), float(temperature), int(ignore_index)
    if _cabi.tracked(logits):
        return TokenLogProbs(*TokenLogProbsFunc.apply(logits, tokens, top_k, temperature, ignore_index))
    dev = _check(logits, tokens, top_k, temperature)
    return TokenLogProbs(*_forward(dev, logits, tokens, top_k, temperature, ignore_index, False)[2:6])
