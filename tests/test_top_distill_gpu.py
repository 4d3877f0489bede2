"""Distillation from lists of alternatives against 64 bits.

Tolerances (u = 2^-24): a row's loss is sum w (log w - log p): log p as in test_token_logprobs_gpu.py, log w and w carry
about 10 u of their size and the list's sum (at most 4 + 5 additions).  The gradient p - w: p's relative error
(104 + 4 log2 V + 8 |log p|) u, w's 24 u, and half a step of its type (float32 / bfloat16 step: the mean's divisor is in)."""
import math

import pytest
import torch

from oracle import language_head as O
from test_token_logprobs_gpu import DTYPES, TINY, U, close

pytestmark = pytest.mark.gpu


def inputs(rows, v, k, dtype, seed=0, pad=0, ragged=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, v + pad, generator=g, device="cuda") * 2).to(dtype)[:, :v]
    teacher = x.float() * 0.8 + torch.randn(rows, v, generator=g, device="cuda")
    q, tok = torch.topk(torch.log_softmax(teacher, 1), k, dim=1)
    if ragged:
        past = torch.arange(k, device="cuda") >= torch.randint(0, k + 1, (rows, 1), generator=g, device="cuda")
        tok, q = tok.masked_fill(past, -1), q.masked_fill(past, -math.inf)
    return x, tok, q.contiguous()


def expected(x, tok, q, t):
    loss, grad, counted = O.distill(x, tok, q, t)
    w, _ = O.list_weights(tok, q)
    logp, p = O.softmax_parts(x, t)
    v = x.shape[-1]
    at = tok.clamp(0, v - 1)
    lp = torch.where(w > 0, logp.gather(-1, at), torch.zeros_like(w)).nan_to_num(0.0, 0.0, 0.0)
    lw = torch.where(w > 0, w.log(), torch.zeros_like(w)).nan_to_num()
    span = torch.where(tok >= 0, q, torch.zeros_like(q)).nan_to_num(0.0, 0.0, 0.0).double().abs().amax(-1, keepdim=True)
    wrel = 24 + 2 * span                                             # (q - max q and its exponential)
    ltol = ((104 + 4 * math.log2(v + 1)) * U + 4 * U * lp.abs() + (lw.abs() + lp.abs()) * wrel * U + 10 * U) * w.nan_to_num()
    ltol = ltol.sum(-1)
    clipped = torch.where(p == 0, torch.zeros_like(p), logp)
    gtol = (p * (104 + 4 * math.log2(v + 1) + 8 * clipped.abs()) * U).scatter_add_(-1, at, w.nan_to_num() * wrel * U)
    gtol = (gtol + 2.0 ** -126 * 400) / t
    return loss, grad, counted, ltol, gtol


def check(x, tok, q, t=1.0, up=1.0):
    import pytorch_loss as P
    eps, tiny = torch.finfo(x.dtype).eps / 2, TINY[x.dtype]
    loss, grad, counted, ltol, gtol = expected(x, tok, q, t)
    n = int(counted.sum())
    # rows' losses, with an upstream gradient of their own
    leaf = x.detach().requires_grad_(True)
    got = P.TopTokenDistillLoss(t, 'none')(leaf, tok, q)
    close(got.detach(), loss, ltol, "losses")
    g = torch.Generator(device="cuda").manual_seed(4)
    d = torch.randn(loss.shape, generator=g, device="cuda")
    have, = torch.autograd.grad(got, leaf, d)
    want = grad * d.double().unsqueeze(-1)
    close(have, want, gtol * d.double().abs().unsqueeze(-1) + want.nan_to_num().abs() * (eps + 4 * U) + tiny, "gradient, per row")
    for red in ("mean", "sum"):
        scale = 1.0 / n if red == "mean" and n else 1.0
        leaf = x.detach().requires_grad_(True)
        crit = P.TopTokenDistillLoss(t, red)
        got = crit(leaf, tok, q)
        want = loss.sum() * (scale if n or red == "sum" else math.nan)
        close(got.detach(), want, (ltol.nan_to_num().sum() + 2 * U * loss.abs().nan_to_num(0.0, 0.0, 0.0).sum()) * scale, red)
        have, = torch.autograd.grad(got, leaf, torch.tensor(up, device="cuda"), retain_graph=True)
        again, = torch.autograd.grad(got, leaf, torch.tensor(up, device="cuda"))
        wantg = grad * (scale * up)
        # (a second rounding where the step's gradient is multiplied by the upstream gradient)
        tol = gtol * scale * up + wantg.nan_to_num().abs() * ((2.01 if up != 1 else 1) * eps + 8 * U) + tiny * (1 + up)
        close(have, wantg, tol, "gradient, " + red)
        close(again, wantg, tol, "gradient again, " + red)
        with torch.no_grad():
            close(crit(x, tok, q), want, (ltol.nan_to_num().sum() + 2 * U * loss.abs().nan_to_num(0.0, 0.0, 0.0).sum()) * scale, red)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v, k", [(1, 1), (3, 2), (9, 9), (100, 5), (1000, 20), (1025, 33), (2049, 128), (8192, 64),
                                  (32768, 20), (50001, 7), (100003, 32), (131072, 128)])
def test_losses_and_gradients(v, k, dtype):
    for rows in (1, 6, 40):
        x, tok, q = inputs(rows, v, k, dtype, seed=v)
        check(x, tok, q)
    x, tok, q = inputs(17, v, k, dtype, seed=v + 1, ragged=True)
    check(x, tok, q, t=1.5, up=0.4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v, pad", [(1000, 24), (1001, 23), (5001, 1), (40000, 8)])
def test_rows_apart(v, pad, dtype):
    x, tok, q = inputs(9, v, 11, dtype, pad=pad)
    check(x, tok, q)


def test_many_rows():
    x, tok, q = inputs(5000, 700, 12, torch.bfloat16, ragged=True)
    check(x, tok, q)
    x, tok, q = inputs(900, 20001, 12, torch.float32, ragged=True)
    check(x, tok, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [60, 6000, 90000])
def test_lists_and_rows_at_the_edge(v, dtype):
    low = torch.finfo(dtype).min
    x, tok, q = inputs(16, v, 8, dtype)
    tok[0] = -1                                                      # no list
    q[1] = -math.inf                                                 # no mass
    tok[2] = tok[2, 0]                                               # one token eight times
    tok[3, 4:] = tok[3, :4]                                          # each twice
    tok[4, 2:] = -7
    tok[5, 3], q[5, 3] = -1, math.nan                                # an entry that does not exist is not looked at
    x[6] = -math.inf                                                 # nothing left: infinite loss, no gradient
    x[7] = low
    x[8, tok[8, 0]] = -math.inf                                      # a masked token that the teacher wants
    q[9] = torch.tensor([-1e30, -2.0, -3.0, -1e30, -4.0, -5.0, -math.inf, -1.0], device="cuda")
    x[10, : v // 2] = -math.inf
    check(x, tok, q)
    x[11, 0] = math.nan
    check(x, tok, q)
    x[11, 0] = 0.0
    tok[12, 1] = v                                                   # beyond the vocabulary
    tok[13, 7] = 1 << 40
    check(x, tok, q)
    tok[12, 1] = tok[13, 7] = 0
    q[14, 0] = math.nan
    check(x, tok, q)


def test_nothing_counts():
    import pytorch_loss as P
    x, tok, q = inputs(5, 3000, 4, torch.float32)
    tok[:] = -1
    check(x, tok, q)
    for v in (30, 3000):
        e = torch.zeros(0, v, device="cuda", requires_grad=True)
        lists = torch.zeros(0, 4, dtype=torch.int64, device="cuda"), torch.zeros(0, 4, device="cuda")
        assert math.isnan(float(P.TopTokenDistillLoss()(e, *lists).detach()))
        s = P.TopTokenDistillLoss(reduction='sum')(e, *lists)
        s.backward()
        assert float(s.detach()) == 0.0 and e.grad.shape == (0, v)


@pytest.mark.parametrize("v", [500, 33000])
def test_one_pass_step_agrees_with_two_passes(v, monkeypatch):
    import pytorch_loss as P
    x, tok, q = inputs(30, v, 9, torch.float32, ragged=True)
    got = []
    for fused in ("1", "0"):
        monkeypatch.setenv("B200_SOFTMAX_FUSED", fused)
        leaf = x.detach().requires_grad_(True)
        loss = P.TopTokenDistillLoss()(leaf, tok, q)
        loss.backward()
        got.append((loss.detach(), leaf.grad))
    _, _, _, _, gtol = expected(x, tok, q, 1.0)
    assert abs(float(got[0][0]) - float(got[1][0])) <= 2e-6 * abs(float(got[1][0]))
    close(got[0][1], got[1][1], 2 * gtol + got[1][1].abs().double() * 16 * U, "two ways")


def test_half_gradients_survive_loss_scaling():
    """A mean over many rows in float16: the loss scale is applied before the rounding."""
    import pytorch_loss as P
    x, tok, q = inputs(2000, 300, 5, torch.float16)
    leaf = x.detach().requires_grad_(True)
    P.TopTokenDistillLoss()(leaf, tok, q).mul(65536.0).backward()
    _, grad, _, _, gtol = expected(x, tok, q, 1.0)
    want = grad * (65536.0 / 2000)
    close(leaf.grad, want, gtol * 33 + want.abs() * (2.0 ** -11 + 8 * U) + 2.0 ** -25, "scaled")


def test_leading_dimensions():
    import pytorch_loss as P
    x, tok, q = inputs(12, 700, 6, torch.float32)
    want = P.TopTokenDistillLoss(reduction='none')(x, tok, q)
    got = P.TopTokenDistillLoss(reduction='none')(x.view(3, 4, 700), tok.view(3, 4, 6), q.view(3, 4, 6))
    assert got.shape == (3, 4) and torch.equal(got.view(-1), want)
    a = P.TopTokenDistillLoss(reduction='none')(x.t().contiguous().t(), tok.t().contiguous().t(), q)
    assert torch.equal(a, want)
    one = P.TopTokenDistillLoss(reduction='none')(x[0], tok[0], q[0])
    assert one.shape == ()


def test_results_repeat_bit_for_bit():
    import pytorch_loss as P
    for rows, v, dtype in ((300, 32768, torch.bfloat16), (20, 131072, torch.float32), (700, 900, torch.float16)):
        x, tok, q = inputs(rows, v, 20, dtype)
        first = None
        for _ in range(4):
            leaf = x.detach().requires_grad_(True)
            loss = P.TopTokenDistillLoss()(leaf, tok, q)
            loss.backward()
            if first is None:
                first = loss.detach(), leaf.grad
            assert torch.equal(loss.detach(), first[0]) and torch.equal(leaf.grad, first[1])


def test_refusals_on_the_gpu():
    import pytorch_loss as P
    x, tok, q = inputs(4, 50, 3, torch.float32)
    crit = P.TopTokenDistillLoss()
    for a in ((x.double(), tok, q), (x, tok.int(), q), (x, tok, q.half()), (x, tok[:3], q[:3]), (x, tok, q[:, :2]),
              (x, tok[:, 0], q[:, 0]), (x, tok[:, :0], q[:, :0]), (x[:, :0], tok, q),
              (x, tok.repeat(1, 43), q.repeat(1, 43))):
        with pytest.raises(RuntimeError):
            crit(*a)
    crit.temperature = -1.0
    with pytest.raises(ValueError):
        crit(x, tok, q)
