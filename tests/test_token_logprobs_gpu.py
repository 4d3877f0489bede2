"""Log probabilities of given tokens, entropies and alternatives against 64 bits.

Tolerances, with u = 2^-24 (half a float32 step) and z the distance to the row's maximum in log2 units:
z carries 3 roundings (3 u |z|), 2^z another 2^-22, and a sum over a row at most 60 additions one after the other (16
pairs of a batch, the batches of a thread, the joins).  sum p |z| <= log2 V, sum p z^2 <= (log2 V)^2 or so.  Hence
   log p      (4 + 60 + 4 log2 V + 40) u + 4 u |log p|
   entropy    the same + 3 (log2 V)^2 u
   gradient   (the same sum + 4 |z|) u of p (|dl| + |dh| (|log p| + H)), plus half a step of its type."""
import math

import pytest
import torch

from oracle import language_head as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def lp_tol(v, logp):
    return (104 + 4 * math.log2(v + 1)) * U + 4 * U * logp.abs().nan_to_num(0.0, 0.0, 0.0)


def h_tol(v):
    return (104 + 4 * math.log2(v + 1) + 3 * math.log2(v + 1) ** 2) * U


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what + ": NaN elsewhere"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what + ": infinities"
    assert not bool((got.isinf() & ~inf).any()), what + ": infinities"
    off = ((got - want).abs() - tol.nan_to_num(0.0)).masked_fill(inf | want.isnan(), -1.0)
    assert bool((off <= 0).all()), "%s: off by %g more than allowed" % (what, float(off.max()))


def grad_tol(x, tokens, dl, dh, t, ignore=-100):
    logp, p = O.softmax_parts(x, t)
    v = x.shape[-1]
    h = O.entropy_of(logp, p)
    lp = torch.where(p == 0, torch.zeros_like(p), logp)
    size = p * (dl.double().abs().unsqueeze(-1) + dh.double().abs().unsqueeze(-1) * (lp.abs() + h.unsqueeze(-1)))
    hot = torch.zeros_like(p).scatter_(-1, tokens.clamp(0, v - 1).unsqueeze(-1), 1.0)
    tol = size * (104 + 4 * math.log2(v + 1) + 3 * math.log2(v + 1) ** 2 + 8 * lp.abs()) * U
    tol = tol + hot * dl.double().abs().unsqueeze(-1) * 4 * U
    want = O.token_logprobs_grad(x, tokens, dl, dh, t, ignore)
    # (2^z below 2^-126 is 0: what such an element would have added)
    return want, (tol + 2.0 ** -126 * 400) / t + want.nan_to_num().abs() * torch.finfo(x.dtype).eps / 2 + TINY[x.dtype]


def inputs(rows, v, dtype, seed=0, pad=0, sigma=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, v + pad, generator=g, device="cuda") * sigma
    best = torch.randint(0, v, (rows, 1), generator=g, device="cuda")
    x.scatter_add_(1, best, torch.rand(rows, 1, generator=g, device="cuda") * 12)
    tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, best.squeeze(1),
                         torch.randint(0, v, (rows,), generator=g, device="cuda"))
    return x.to(dtype)[:, :v], tokens, torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")


def check(x, tokens, dl=None, dh=None, k=0, t=1.0, ignore=-100):
    import pytorch_loss as P
    v = x.shape[-1]
    train = dl is not None
    leaf = x.detach().requires_grad_(True) if train else x
    out = P.token_logprobs(leaf, tokens, top_k=k, temperature=t, ignore_index=ignore)
    lp, h = O.token_logprobs(x, tokens, t, ignore)
    close(out.logprobs.detach(), lp, lp_tol(v, lp), "log probabilities")
    close(out.entropy.detach(), h, torch.full_like(h, h_tol(v)), "entropies")
    if k:
        valid = (tokens != ignore).unsqueeze(-1)
        want = O.alternatives(x, k).masked_fill(~valid, -1)
        assert torch.equal(out.top_tokens, want)
        logp, _ = O.softmax_parts(x, t)
        wlp = logp.gather(-1, want.clamp(min=0)).masked_fill(~valid, 0.0)
        close(out.top_logprobs, wlp, lp_tol(v, wlp), "alternatives")
    else:
        assert out.top_tokens is None and out.top_logprobs is None
    if train:
        grad, = torch.autograd.grad((out.logprobs, out.entropy), leaf, (dl, dh))
        want, tol = grad_tol(x, tokens, dl, dh, t, ignore)
        assert grad.dtype == x.dtype and grad.is_contiguous()
        close(grad, want, tol, "gradient")
    return out


# one logit; rows below, at and above a vector, a warp's row, a block's batch; odd sizes; several blocks to a row
SIZES = [1, 2, 3, 7, 8, 9, 31, 64, 100, 257, 1000, 1023, 1024, 2047, 2048, 2049, 4099, 8192, 32768, 50001, 131072, 160001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", SIZES)
def test_values_and_gradients(v, dtype):
    for rows in ((1, 5, 33) if v <= 8192 else (1, 5)):
        x, tokens, dl, dh = inputs(rows, v, dtype, seed=v)
        check(x, tokens, dl, dh)
        for k in {1, min(5, v), min(20, v), min(32, v), min(33, v), min(128, v)}:
            check(x, tokens, k=k, t=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, v", [(1024, 1000), (700, 2500), (1500, 4100), (600, 16384)])
def test_many_rows(rows, v, dtype):
    x, tokens, dl, dh = inputs(rows, v, dtype, seed=5)
    tokens[::7] = -100
    check(x, tokens, dl, dh, t=1.5)
    check(x, tokens, k=20, t=1.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v, pad", [(50, 3), (1000, 24), (1001, 23), (5001, 1), (32000, 768)])
def test_rows_apart_and_shifted(v, pad, dtype):
    """Rows of a padded storage, and a storage that starts off a 16-byte boundary."""
    x, tokens, dl, dh = inputs(9, v, dtype, seed=v, pad=pad)
    check(x, tokens, dl, dh)
    check(x, tokens, k=min(20, v))
    flat = torch.empty(9 * v + 1, device="cuda", dtype=dtype)[1:]
    moved = flat.view(9, v).copy_(x)
    check(moved, tokens, dl, dh)
    check(moved, tokens, k=min(20, v))


def test_leading_dimensions_and_copies():
    import pytorch_loss as P
    x, tokens, _, _ = inputs(12, 300, torch.float32, seed=3)
    want = P.token_logprobs(x, tokens, top_k=4)
    views = [x.view(3, 4, 300), x.view(3, 4, 300).transpose(0, 1).contiguous().transpose(0, 1), x.t().contiguous().t().view(3, 4, 300)
             if False else x.t().contiguous().t().reshape(3, 4, 300)]
    for y in views:
        got = P.token_logprobs(y, tokens.view(3, 4), top_k=4)
        assert got.logprobs.shape == (3, 4) and got.top_tokens.shape == (3, 4, 4)
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(b.shape), b)
    one = P.token_logprobs(x[0], tokens[0], top_k=4)
    assert one.logprobs.shape == () and one.top_tokens.shape == (4,)
    close(one.logprobs, want.logprobs[0], lp_tol(300, want.logprobs[0]), "one row")
    y = x.t().contiguous().t()                                     # logits across memory: copied, the gradient too
    leaf = y.detach().requires_grad_(True)
    g, = torch.autograd.grad(P.token_logprobs(leaf, tokens).logprobs.sum(), leaf)
    leaf2 = x.detach().requires_grad_(True)
    g2, = torch.autograd.grad(P.token_logprobs(leaf2, tokens).logprobs.sum(), leaf2)
    assert torch.equal(g, g2)
    e = x[:1].expand(6, 300).detach().requires_grad_(True)         # the same row for all tokens
    g, = torch.autograd.grad(P.token_logprobs(e, tokens[:6]).logprobs.sum(), e)
    want, tol = grad_tol(x[:1].expand(6, 300), tokens[:6], torch.ones(6, device="cuda"), torch.zeros(6, device="cuda"), 1.0)
    close(g, want, tol, "gradient of a broadcast row")


@pytest.mark.parametrize("v", [40, 1500, 9000, 140000])
def test_empty_inputs(v):
    import pytorch_loss as P
    x = torch.zeros(0, v, device="cuda", requires_grad=True)
    out = P.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top_k=3)
    assert out.logprobs.shape == (0,) and out.top_tokens.shape == (0, 3)
    (out.logprobs.sum() + out.entropy.sum()).backward()
    assert x.grad.shape == (0, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 1500, 9000, 140000])
def test_masked_rows(v, dtype):
    """-inf and the type's lowest value in all or most places, infinities, NaN, equal logits, far apart logits."""
    low = torch.finfo(dtype).min
    rows = [torch.randn(v) for _ in range(14)]
    rows[0][:] = -math.inf                                          # nothing left
    rows[1][:] = low                                                # nothing left, as masks that add the lowest value do
    rows[2][1:] = -math.inf                                         # one left
    rows[3][: v // 2] = low
    rows[4][: v - 3] = -math.inf                                    # fewer than the alternatives
    rows[5][v // 3] = math.nan
    rows[6][v // 2] = math.inf
    rows[7][:] = 0.0                                                # all equal
    rows[8][:] = 0.0
    rows[8][::2] = -0.0                                             # -0 and 0 are equal
    rows[9] = torch.linspace(-60, 60, v)                            # ascending
    rows[10][: v // 2] = -math.inf
    rows[10][v // 2:] = low                                         # -inf and the lowest
    rows[11][3] = torch.finfo(dtype).max
    rows[12][0] = math.nan
    rows[12][v - 1] = -math.nan
    rows[13] = rows[13].sort(descending=True).values
    x = torch.stack(rows).to(dtype).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, v, (14,), generator=g, device="cuda")
    tokens[2] = 0
    dl, dh = torch.randn(14, generator=g, device="cuda"), torch.randn(14, generator=g, device="cuda")
    for tok in (tokens, torch.full_like(tokens, v - 1), torch.zeros_like(tokens)):
        check(x, tok, dl, dh)
        check(x, tok, k=20)
    check(x, tokens, k=32, t=3.0)
    many = x.repeat(100, 1)                                         # (a block to a row, whatever the size)
    check(many, tokens.repeat(100), k=20)
    check(many, tokens.repeat(100), dl.repeat(100), dh.repeat(100))


def test_tokens_that_do_not_count_or_exist():
    x, tokens, dl, dh = inputs(12, 5000, torch.float32)
    tokens[0], tokens[1], tokens[2], tokens[3] = -100, -1, 5000, 1 << 40
    check(x, tokens, dl, dh)
    check(x, tokens, k=3)
    tokens[4] = 7
    check(x, tokens, dl, dh, ignore=7)
    check(x, tokens, k=3, ignore=-1)
    x[0] = math.nan                                                 # not read
    check(x, tokens, dl, dh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits_where_few_threads_see_them(dtype):
    """The largest logits lie 2048 apart, or fill one stretch, or agree at thousands of places: the candidates of the
    first bound do not fit."""
    g = torch.Generator(device="cuda").manual_seed(2)
    v = 1 << 17
    x = torch.randn(4, v, generator=g, device="cuda")
    x[0, ::2048] += 50
    x[0, 1::2048] += 50
    x[1, 5000:9000] += 50
    x[2] = (x[2] * 2).round()                                       # about twenty values
    x[3, : v // 2] = 7.0
    x = x.to(dtype)
    tokens = torch.randint(0, v, (4,), generator=g, device="cuda")
    for k in (1, 20, 128):
        check(x, tokens, k=k)
        check(x.repeat(300, 1), tokens.repeat(300), k=k)            # (one block to a row)


def test_logits_below_the_normal_range():
    """Denormal logits keep their order among the alternatives (their log probabilities cannot tell them apart)."""
    import pytorch_loss as P
    for v in (200, 3000, 20000):
        x = torch.zeros(4, v)
        x[:, ::3] = torch.rand(4, len(range(0, v, 3))) * 1e-38
        x[:, 5] = -1e-40
        x[1] -= 1e-39
        x[2] = x[2].sort().values
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype).cuda()
            for k in (5, 30, 100):
                got = P.token_logprobs(y, torch.zeros(4, dtype=torch.int64, device="cuda"), top_k=k)
                assert torch.equal(got.top_tokens.cpu(), O.alternatives(y.cpu(), k))


@pytest.mark.parametrize("t", [1e-4, 0.05, 20.0, 1e4])
def test_temperatures(t):
    x, tokens, dl, dh = inputs(6, 3000, torch.float32)
    check(x, tokens, dl * t, dh * t, t=t)
    check(x, tokens, k=10, t=t)


def test_upstream_gradients():
    """One output alone, none, broadcast ones; the alternatives carry none."""
    import pytorch_loss as P
    x, tokens, dl, dh = inputs(10, 2100, torch.float32)
    zero = torch.zeros_like(dl)
    for use, a, b in (((True, False), dl, zero), ((False, True), zero, dh)):
        leaf = x.detach().requires_grad_(True)
        out = P.token_logprobs(leaf, tokens, top_k=3)
        got, = torch.autograd.grad(out.logprobs if use[0] else out.entropy, leaf, dl if use[0] else dh)
        want, tol = grad_tol(x, tokens, a, b, 1.0)
        close(got, want, tol, "gradient of one output")
        assert not out.top_logprobs.requires_grad
    leaf = x.detach().requires_grad_(True)
    out = P.token_logprobs(leaf, tokens)
    got, = torch.autograd.grad(out.logprobs.mean() + out.entropy.sum(), leaf)
    want, tol = grad_tol(x, tokens, torch.full_like(dl, 0.1), torch.ones_like(dl), 1.0)
    close(got, want, tol, "broadcast upstream gradients")
    with torch.no_grad():
        assert not P.token_logprobs(leaf, tokens).logprobs.requires_grad


def test_gradient_against_differences():
    """Central differences of the 64-bit value: the step's own error is (1e-4)^2 times third derivatives below 1."""
    x, tokens, dl, dh = inputs(3, 37, torch.float32, sigma=1.0)
    import pytorch_loss as P
    leaf = x.detach().requires_grad_(True)
    out = P.token_logprobs(leaf, tokens, temperature=0.8)
    got, = torch.autograd.grad((out.logprobs, out.entropy), leaf, (dl, dh))

    def value(y):
        lp, h = O.token_logprobs(y, tokens, 0.8)
        return (lp * dl.double()).sum() + (h * dh.double()).sum()
    want, x64, step = torch.zeros(3, 37, dtype=torch.float64, device="cuda"), x.double(), 1e-4
    for i in range(3):
        for j in range(37):
            d = torch.zeros_like(x64)
            d[i, j] = step
            want[i, j] = (value(x64 + d) - value(x64 - d)) / (2 * step)
    _, tol = grad_tol(x, tokens, dl, dh, 0.8)
    close(got, want, tol + 1e-7, "differences")


def test_second_backward_and_changes_in_place():
    import pytorch_loss as P
    x, tokens, dl, dh = inputs(5, 600, torch.bfloat16)
    leaf = x.detach().requires_grad_(True)
    out = P.token_logprobs(leaf, tokens)
    a, = torch.autograd.grad(out.logprobs.sum(), leaf, retain_graph=True)
    b, = torch.autograd.grad(out.logprobs.sum(), leaf)
    assert torch.equal(a, b)
    y = leaf * 1
    out = P.token_logprobs(y, tokens)
    y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.logprobs.sum().backward()


def test_results_repeat_bit_for_bit():
    import pytorch_loss as P
    for rows, v in ((1, 131072), (40, 50001), (500, 32768), (900, 1000)):
        x, tokens, dl, dh = inputs(rows, v, torch.bfloat16)
        leaf = x.detach().requires_grad_(True)
        first = P.token_logprobs(leaf, tokens, top_k=20)
        g, = torch.autograd.grad((first.logprobs, first.entropy), leaf, (dl, dh))
        for _ in range(3):
            again = P.token_logprobs(leaf, tokens, top_k=20)
            g2, = torch.autograd.grad((again.logprobs, again.entropy), leaf, (dl, dh))
            assert all(torch.equal(a, b) for a, b in zip(first, again)) and torch.equal(g, g2)


def test_offsets_past_32_bits():
    """70000 rows of 32768 float16 logits: 4.6 GB, 2.3e9 elements; the last rows against 64 bits."""
    import pytorch_loss as P
    rows, v = 70000, 32768
    x = torch.zeros(rows, v, dtype=torch.float16, device="cuda")
    tail, tokens, dl, dh = inputs(8, v, torch.float16, seed=9)
    x[-8:] = tail
    tok = torch.zeros(rows, dtype=torch.int64, device="cuda")
    tok[-8:] = tokens
    tok[100:-8] = -100
    leaf = x.requires_grad_(True)
    out = P.token_logprobs(leaf, tok, top_k=5)
    lp, h = O.token_logprobs(tail, tokens)
    close(out.logprobs[-8:].detach(), lp, lp_tol(v, lp), "last rows")
    assert torch.equal(out.top_tokens[-8:], O.alternatives(tail, 5))
    up = torch.zeros(rows, device="cuda")
    up[-8:] = dl
    g, = torch.autograd.grad(out.logprobs, leaf, up)
    want, tol = grad_tol(tail, tokens, dl, torch.zeros_like(dl), 1.0)
    close(g[-8:], want, tol, "last rows' gradient")
    assert float(g[:-8].abs().max()) == 0.0


def test_refusals_on_the_gpu():
    import pytorch_loss as P
    x, tokens, _, _ = inputs(4, 50, torch.float32)
    for bad in (dict(logits=x.double()), dict(tokens=tokens.int()), dict(tokens=tokens[:3]), dict(tokens=tokens.unsqueeze(1))):
        with pytest.raises(RuntimeError):
            P.token_logprobs(**{"logits": x, "tokens": tokens, **bad})
    for bad in (dict(top_k=51), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            P.token_logprobs(x, tokens, **bad)
    with pytest.raises(RuntimeError):
        P.token_logprobs(x[:, :0], tokens)
    with pytest.raises(ValueError):
        P.token_logprobs(torch.randn(2, 500, device="cuda"), tokens[:2], top_k=129)
