"""What the operators at the output end of a language model are measured on: the layer norm in front of the head, log
probabilities of given tokens with entropy and the best alternatives, and the loss of a student that learns from such
alternatives.

A case is a dict of plain values: `op` ("logprobs", "distill", "norm"), `dtype`, `rows` and

  logprobs  `vocab`, `pad` (columns of the storage behind the vocabulary: rows of a padded head), `k` (alternatives),
            `temperature`, `train` (gradients of the log probabilities and the entropies follow), `ignored` (share of
            rows that are padding)
  distill   `vocab`, `k` (length of the longest list of alternatives), `ragged` (lists of any length, some empty),
            `temperature`, `reduction`, `weight` (the factor of this loss in a sum of losses)
  norm      `width`, `param` (type of weight and bias), `train`
"""
import math
import os
import sys

import torch

own = False        # False: the operators' plain forms; True: the calls that a user makes of pytorch_loss

IGNORE = -100
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def _logprobs(rows, vocab, dtype, **more):
    case = {"op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "pad": 0, "k": 0, "temperature": 1.0,
            "train": False, "ignored": 0.0}
    case.update(more)
    return case


def _distill(rows, vocab, dtype, k, **more):
    case = {"op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "ragged": False, "temperature": 1.0,
            "reduction": "mean", "weight": 1.0}
    case.update(more)
    return case


def _norm(rows, width, dtype, **more):
    case = {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "param": dtype, "train": True}
    case.update(more)
    return case


def listed():
    return [
        # one request of a server, one new token: a single row over a large vocabulary, latency alone
        _logprobs(1, 131072, "bf16", k=20, name="logprobs_one"),
        # one step of a batch of requests: float32 logits of a head whose odd vocabulary is padded to whole 64s
        _logprobs(64, 50001, "f32", pad=47, k=5, temperature=0.8, name="logprobs_batch"),
        # scoring whole prompts, alternatives stored for a student
        _logprobs(4096, 32768, "f16", k=20, name="logprobs_prompt"),
        # policy training: gradients of log probability and entropy, a padded batch
        _logprobs(16384, 32768, "bf16", train=True, ignored=0.1, name="logprobs_train"),
        # the same over an odd vocabulary: float32 rows that start at any multiple of four bytes
        _logprobs(3000, 50001, "f32", train=True, temperature=0.8, name="logprobs_train_odd"),
        # a student's small batch
        _distill(256, 32768, "f32", 20, name="distill_small"),
        # a student over a large vocabulary, long lists of alternatives
        _distill(8192, 65536, "bf16", 64, name="distill_vocab"),
        # an odd vocabulary in half precision, lists of any length, one of several losses
        _distill(2047, 100003, "f16", 32, ragged=True, temperature=1.5, reduction="sum", weight=0.4,
                 name="distill_odd"),
        # the norm of one decode step
        _norm(32, 4096, "bf16", train=False, name="norm_decode"),
        # the norm of a training step
        _norm(16384, 4096, "bf16", param="f32", name="norm_train"),
        # an odd width
        _norm(6001, 1003, "f32", name="norm_odd"),
        # a wide model in half precision
        _norm(16384, 8192, "f16", name="norm_wide"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of these ranges: rows, vocabularies and widths over their logarithm, odd ones among them."""
    op = rng.choice(["logprobs", "logprobs", "distill", "norm"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        train = rng.random() < 0.75
        width = rng.choice([64, 256, 768, 1024, 4096, 8192, _log_int(rng, 33, 16384), _log_int(rng, 33, 16384)])
        rows = _log_int(rng, 1, min(65536, (1 << 27) // width))
        return _norm(rows, width, dtype, param=rng.choice([dtype, "f32"]), train=train)
    vocab = rng.choice([1024, 32768, 65536, 131072, _log_int(rng, 500, 160000), _log_int(rng, 500, 160000)])
    rows = _log_int(rng, 1, min(16384, (1 << 28) // vocab))
    temperature = rng.choice([1.0, 1.0, 0.7, 1.5])
    if op == "distill":
        return _distill(rows, vocab, dtype, _log_int(rng, 1, 128), ragged=rng.random() < 0.5, temperature=temperature,
                        reduction="sum" if dtype == "f16" else rng.choice(["mean", "sum"]),
                        weight=rng.choice([1.0, 1.0, 0.4]))
    if rng.random() < 0.5:
        return _logprobs(rows, vocab, dtype, train=True, temperature=temperature, ignored=rng.choice([0.0, 0.1, 0.5]))
    return _logprobs(rows, vocab, dtype, pad=rng.choice([0, 0, -vocab % 64, 7]), k=rng.choice([0, 1, 5, 20, 64, 128]),
                     temperature=temperature, ignored=rng.choice([0.0, 0.0, 0.1]))


# ---- inputs

def _logits(case, g):
    """Logits as a head gives them: noise, one token ahead by up to 12 in most rows, and the last percent of the
    vocabulary masked out."""
    rows, vocab, pad = case["rows"], case["vocab"], case.get("pad", 0)
    x = torch.randn(rows, vocab + pad, generator=g, device="cuda").mul_(2.0)
    best = torch.randint(0, vocab - vocab // 100, (rows, 1), generator=g, device="cuda")
    x.scatter_add_(1, best, torch.rand(rows, 1, generator=g, device="cuda").mul_(12.0))
    x[:, vocab - vocab // 100:vocab] = -math.inf
    return x.to(DTYPES[case["dtype"]])[:, :vocab], best


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    rows, state = case["rows"], {"case": case}
    if case["op"] == "norm":
        width, par = case["width"], DTYPES[case["param"]]
        x = torch.randn(rows, width, generator=g, device="cuda") * (torch.rand(rows, 1, generator=g, device="cuda") + 0.5)
        x += torch.randn(rows, 1, generator=g, device="cuda")
        state["x"] = x.to(DTYPES[case["dtype"]])
        state["weight"] = (torch.randn(width, generator=g, device="cuda") * 0.2 + 1.0).to(par)
        state["bias"] = (torch.randn(width, generator=g, device="cuda") * 0.2).to(par)
        if case["train"]:
            state["dy"] = torch.randn(rows, width, generator=g, device="cuda").to(DTYPES[case["dtype"]])
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_(True)
        return state
    x, best = _logits(case, g)
    live = case["vocab"] - case["vocab"] // 100
    if case["op"] == "logprobs":
        # half the tokens are the best one, the others any
        other = torch.randint(0, live, (rows, 1), generator=g, device="cuda")
        tokens = torch.where(torch.rand(rows, 1, generator=g, device="cuda") < 0.5, best, other).squeeze(1)
        gone = torch.randperm(rows, generator=g, device="cuda")[:int(case["ignored"] * rows)]
        tokens[gone] = IGNORE
        state["tokens"] = tokens
        if case["train"]:
            state["d_logprobs"] = torch.randn(rows, generator=g, device="cuda")
            state["d_entropy"] = torch.randn(rows, generator=g, device="cuda") * 0.1
    else:
        # the teacher saw logits that the student's resemble
        k = case["k"]
        teacher = x.float().mul_(0.8)
        teacher += torch.randn(teacher.shape, generator=g, device="cuda")
        state["top_logprobs"], state["top_tokens"] = torch.topk(torch.log_softmax(teacher, 1), k, dim=1)
        if case["ragged"]:
            length = torch.randint(0, k + 1, (rows, 1), generator=g, device="cuda")
            past = torch.arange(k, device="cuda") >= length
            state["top_tokens"].masked_fill_(past, -1)
            state["top_logprobs"].masked_fill_(past, -math.inf)
        if case["weight"] != 1.0:
            state["upstream"] = torch.tensor(case["weight"], device="cuda")
    state["logits"] = x.requires_grad_(True) if case["op"] == "distill" or case["train"] else x
    return state


# ---- one pass

def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-loss_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import pytorch_loss
    return pytorch_loss


def _own_logprobs(case, state):
    out = _package().token_logprobs(state["logits"], state["tokens"], top_k=case["k"], temperature=case["temperature"],
                                    ignore_index=IGNORE)
    got = {"logprobs": out.logprobs.detach(), "entropy": out.entropy.detach()}
    if case["train"]:
        got["grad"], = torch.autograd.grad((out.logprobs, out.entropy), (state["logits"],),
                                           (state["d_logprobs"], state["d_entropy"]))
    if case["k"]:
        got["top_logprobs"], got["top_tokens"] = out.top_logprobs, out.top_tokens
    return got


def _plain_logprobs(case, state):
    x, tokens = state["logits"].detach(), state["tokens"]
    valid = tokens != IGNORE
    z = x.float() / case["temperature"]
    z -= z.amax(1, keepdim=True)
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    z -= torch.log(total)                                   # log probabilities
    p /= total
    masked = p == 0                                         # (0 log 0 counts nothing)
    entropy = -(p * z.masked_fill(masked, 0.0)).sum(1)
    logprobs = z.gather(1, tokens.clamp(min=0).unsqueeze(1)).squeeze(1)
    got = {"logprobs": logprobs.masked_fill(~valid, 0.0), "entropy": entropy.masked_fill(~valid, 0.0)}
    if case["train"]:
        dl = (state["d_logprobs"] * valid).unsqueeze(1)
        dh = (state["d_entropy"] * valid).unsqueeze(1)
        grad = -p * (dl + dh * (z.masked_fill(masked, 0.0) + entropy.unsqueeze(1)))
        at = tokens.clamp(min=0).unsqueeze(1)
        grad.scatter_add_(1, at, dl)
        got["grad"] = (grad / case["temperature"]).to(x.dtype)
    if case["k"]:
        # (a stable order: equal logits go by their index)
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        got["top_logprobs"] = z.gather(1, best).masked_fill(~valid.unsqueeze(1), 0.0)
        got["top_tokens"] = best.masked_fill(~valid.unsqueeze(1), -1)
    return got


def _own_distill(case, state):
    loss = _package().TopTokenDistillLoss(temperature=case["temperature"], reduction=case["reduction"])(
        state["logits"], state["top_tokens"], state["top_logprobs"])
    grad, = torch.autograd.grad(loss, state["logits"], state.get("upstream"))
    return {"loss": loss.detach(), "grad": grad}


def _targets(tokens, logprobs):
    """A teacher's probabilities, made to sum to one over each list, and which rows have any."""
    there = tokens >= 0
    q = logprobs.masked_fill(~there, -math.inf)
    best = q.amax(1, keepdim=True)
    valid = best > -math.inf
    t = torch.exp(q - best.masked_fill(~valid, 0.0))
    return t / t.sum(1, keepdim=True).masked_fill(~valid, 1.0), valid


def _plain_distill(case, state):
    x, tokens = state["logits"].detach(), state["top_tokens"]
    t, valid = _targets(tokens, state["top_logprobs"])
    z = x.float() / case["temperature"]
    z -= z.amax(1, keepdim=True)
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    z -= torch.log(total)
    p /= total
    at = tokens.clamp(min=0)
    diff = torch.log(t.masked_fill(t == 0, 1.0)) - z.gather(1, at)
    loss = (t * diff.masked_fill(t == 0, 0.0)).sum()
    scale = 1.0
    if case["reduction"] == "mean":
        loss, scale = loss / valid.sum(), 1.0 / valid.sum()
    grad = (p * valid).scatter_add_(1, at, -t)
    return {"loss": loss, "grad": (grad * (scale * case["weight"] / case["temperature"])).to(x.dtype)}


def _own_norm(case, state):
    y = _package().layer_norm(state["x"], state["weight"], state["bias"], EPS)
    got = {"y": y.detach()}
    if case["train"]:
        got["dx"], got["dweight"], got["dbias"] = torch.autograd.grad(
            y, (state["x"], state["weight"], state["bias"]), state["dy"])
    return got


def _plain_norm(case, state):
    x, w, b = (state[name].detach() for name in ("x", "weight", "bias"))
    mean = x.float().mean(1, keepdim=True)
    xc = x.float() - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xc *= rstd
    got = {"y": (xc * w.float() + b.float()).to(x.dtype)}
    if case["train"]:
        dy = state["dy"].float()
        g = dy * w.float()
        got["dx"] = ((g - g.mean(1, keepdim=True) - xc * (g * xc).mean(1, keepdim=True)) * rstd).to(x.dtype)
        got["dweight"] = (dy * xc).sum(0).to(w.dtype)
        got["dbias"] = dy.sum(0).to(b.dtype)
    return got


def run(state):
    case = state["case"]
    if own:
        return {"logprobs": _own_logprobs, "distill": _own_distill, "norm": _own_norm}[case["op"]](case, state)
    return {"logprobs": _plain_logprobs, "distill": _plain_distill, "norm": _plain_norm}[case["op"]](case, state)


# ---- what a pass cannot do without

def work(case):
    """Inputs read once, outputs written once.  Rows that are padding, or whose list is empty, need not be read; a
    gradient is zero there, but written."""
    rows, s = case["rows"], SIZES[case["dtype"]]
    if case["op"] == "norm":
        e, par = rows * case["width"], case["width"] * SIZES[case["param"]]
        if case["train"]:
            return {"bytes": 4 * s * e + 4 * par, "flops": 20 * e}       # x and dy in, y and dx out
        return {"bytes": 2 * s * e + 2 * par, "flops": 9 * e}
    e, k = rows * case["vocab"], case["k"]
    if case["op"] == "logprobs":
        live = e - int(case["ignored"] * rows) * case["vocab"]
        b = s * live + 16 * rows + 12 * k * rows
        if case["train"]:
            return {"bytes": b + s * e + 8 * rows, "flops": 14 * e}
        return {"bytes": b, "flops": 8 * e}
    live = e * k // (k + 1) if case["ragged"] else e                     # (one list in k + 1 is empty)
    return {"bytes": s * live + s * e + 12 * k * rows, "flops": 10 * e}


# ---- the same in 64 bits, from the definitions

def _exact_norm(case, state):
    x, w = state["x"].detach().double(), state["weight"].detach().double()
    n = case["width"]
    mean = x.sum(1, keepdim=True) / n
    var = ((x - mean) ** 2).sum(1, keepdim=True) / n
    std = torch.sqrt(var + EPS)
    xn = (x - mean) / std
    got = {"y": w * xn + state["bias"].detach().double()}
    if case["train"]:
        dy = state["dy"].double()
        u = w * dy
        got["dx"] = (n * u - u.sum(1, keepdim=True) - xn * (xn * u).sum(1, keepdim=True)) / (n * std)
        got["dweight"], got["dbias"] = torch.einsum("ij,ij->j", dy, xn), dy.sum(0)
    return got


def _exact_logprobs(case, state):
    t, parts = case["temperature"], []
    step = max(1, (1 << 27) // case["vocab"])
    for i in range(0, case["rows"], step):
        logits, tokens = state["logits"].detach()[i:i + step], state["tokens"][i:i + step]
        x = logits.double() / t
        valid = (tokens != IGNORE).double()
        lse = torch.logsumexp(x, 1)
        p = torch.softmax(x, 1)
        xp = torch.where(p > 0, x, torch.zeros_like(x))
        mean = (p * xp).sum(1)
        at = torch.where(tokens == IGNORE, torch.zeros_like(tokens), tokens)
        row = torch.arange(len(tokens), device=x.device)
        part = {"logprobs": (x[row, at] - lse) * valid, "entropy": (lse - mean) * valid}
        if case["train"]:
            # d entropy / dx_j = -p_j (x_j - mean), over the temperature
            dl, dh = state["d_logprobs"][i:i + step].double(), state["d_entropy"][i:i + step].double()
            grad = p * (-dl[:, None] - dh[:, None] * (xp - mean[:, None]))
            grad[row, at] += dl
            part["grad"] = grad * (valid / t)[:, None]
        if case["k"]:
            top = torch.topk(x, case["k"], dim=1).values - lse[:, None]
            part["top_logprobs"] = top * valid[:, None]
        parts.append(part)
    got = {name: torch.cat([q[name] for q in parts]) for name in parts[0]}
    if case["k"]:
        got["top_tokens"] = None
    return got


def _exact_distill(case, state):
    temp, k = case["temperature"], case["k"]
    tokens, q = state["top_tokens"], state["top_logprobs"].double()
    length = (tokens >= 0).sum(1)                       # (what is there stands in front)
    t = torch.where(tokens >= 0, torch.exp(q), torch.zeros_like(q))
    t = t / t.sum(1, keepdim=True).clamp(min=1e-300)
    count = float((length > 0).sum()) if case["reduction"] == "mean" else 1.0
    step, loss, grads = max(1, (1 << 27) // case["vocab"]), 0.0, []
    for i in range(0, case["rows"], step):
        x = state["logits"].detach()[i:i + step].double() / temp
        there, ti = length[i:i + step] > 0, t[i:i + step]
        at = torch.where(tokens[i:i + step] >= 0, tokens[i:i + step], torch.zeros_like(tokens[i:i + step]))
        logp = x.gather(1, at) - torch.logsumexp(x, 1, keepdim=True)
        loss = loss + torch.where(ti > 0, ti * (torch.log(ti) - logp), torch.zeros_like(ti)).sum()
        grad = torch.softmax(x, 1)
        for j in range(k):
            grad[torch.arange(len(at), device=x.device), at[:, j]] -= ti[:, j]
        grads.append(grad * (there.double() * (case["weight"] / (count * temp)))[:, None])
    return {"loss": loss / count, "grad": torch.cat(grads)}


def exact(case, seed):
    state = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "distill": _exact_distill, "norm": _exact_norm}[case["op"]](case, state)
