"""The operators at a language model's output end from their definitions, in 64 bits: layer norm, log probabilities of
given tokens with entropy and alternatives, and distillation from lists of alternatives.  Test infrastructure."""
import math

import torch


def layer_norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    std = ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    y = (x - mean) / std
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def layer_norm_grads(x, weight, eps, dy):
    """dx, dweight, dbias"""
    x, dy = x.double(), dy.double()
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    std = ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) / std
    g = dy if weight is None else dy * weight.double()
    dx = (n * g - g.sum(-1, keepdim=True) - h * (g * h).sum(-1, keepdim=True)) / (n * std)
    return dx, (dy * h).reshape(-1, n).sum(0), dy.reshape(-1, n).sum(0)


def softmax_parts(logits, temperature):
    """(log p, p) of rows; a row of -inf alone has log p -inf and p 0."""
    z = logits.double() / temperature
    m = z.amax(-1, keepdim=True)
    z = z - torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = z.exp().sum(-1, keepdim=True)
    logp = torch.where(s == 0, torch.full_like(z, -math.inf), z - s.log())
    return logp, logp.exp()


def entropy_of(logp, p):
    return -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)


def token_logprobs(logits, tokens, temperature=1.0, ignore_index=-100):
    """(logprobs, entropy) [rows]"""
    logp, p = softmax_parts(logits, temperature)
    v = logits.shape[-1]
    inside = (tokens >= 0) & (tokens < v)
    lp = logp.gather(-1, tokens.clamp(0, v - 1).unsqueeze(-1)).squeeze(-1)
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    valid = tokens != ignore_index
    return torch.where(valid, lp, torch.zeros_like(lp)), torch.where(valid, entropy_of(logp, p), torch.zeros_like(lp))


def token_logprobs_grad(logits, tokens, d_logprobs, d_entropy, temperature=1.0, ignore_index=-100):
    logp, p = softmax_parts(logits, temperature)
    h = entropy_of(logp, p).unsqueeze(-1)
    dl, dh = d_logprobs.double().unsqueeze(-1), d_entropy.double().unsqueeze(-1)
    v = logits.shape[-1]
    hot = torch.zeros_like(p).scatter_(-1, tokens.clamp(0, v - 1).unsqueeze(-1), 1.0)
    g = dl * (hot - p) - dh * torch.where(p == 0, torch.zeros_like(p), p * (logp + h))
    g = torch.where(((tokens < 0) | (tokens >= v)).unsqueeze(-1), torch.full_like(g, math.nan), g / temperature)
    empty = (logits == -math.inf).all(-1) & (tokens >= 0) & (tokens < v)
    return torch.where(((tokens == ignore_index) | empty).unsqueeze(-1), torch.zeros_like(g), g)


def alternatives(logits, k):
    """Indices of the k largest logits of each row: NaN in front, then by value, equal values by index."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, math.inf).add(0), x)
    first = torch.sort(x, dim=-1, descending=True, stable=True).indices
    nan = logits.isnan().gather(-1, first).to(torch.int8)
    order = torch.sort(nan, dim=-1, descending=True, stable=True).indices
    return first.gather(-1, order)[..., :k]


def list_weights(tokens, logprobs):
    """(weights that sum to one over each list, whether the row has any)."""
    q = torch.where(tokens >= 0, logprobs.double(), torch.full_like(logprobs, -math.inf, dtype=torch.float64))
    m = q.amax(-1, keepdim=True)
    some = (m != -math.inf).squeeze(-1)
    w = (q - torch.where(m == -math.inf, torch.zeros_like(m), m)).exp()
    return torch.where(some.unsqueeze(-1), w / w.sum(-1, keepdim=True), torch.zeros_like(w)), some


def distill(logits, tokens, logprobs, temperature=1.0):
    """(losses [rows], gradient of their sum, counted rows)"""
    w, some = list_weights(tokens, logprobs)
    logp, p = softmax_parts(logits, temperature)
    v = logits.shape[-1]
    at = tokens.clamp(0, v - 1)
    bad = (tokens >= v).any(-1) | w.isnan().any(-1)          # (a NaN in the list makes its row NaN)
    term = torch.where(w > 0, w * (w.log() - logp.gather(-1, at)), torch.zeros_like(w))
    loss = term.sum(-1)
    grad = (p.clone().scatter_add_(-1, at, -w)) / temperature
    empty = (logits == -math.inf).all(-1)
    grad = torch.where((empty | ~some).unsqueeze(-1), torch.zeros_like(grad), grad)
    nan = torch.full_like(loss, math.nan)
    loss = torch.where(bad, nan, torch.where(some, loss, torch.zeros_like(loss)))
    grad = torch.where((bad & ~empty).unsqueeze(-1), torch.full_like(grad, math.nan), grad)
    return loss, grad, some | bad
