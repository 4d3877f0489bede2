"""Layer norm forward and backward against 64 bits.

Tolerances (u = 2^-24, S = rms(x) / std(x) of the row, including eps): a row's sums take at most 64 additions one after
the other, so the mean is off by 64 u rms(x) at most and h = (x - mean) / std by e = (66 S + 70 |h| + 4) u.
   y    |w| e + 2 u (|w h| + |b|)
   dx   the terms |g|, mean|g|, |h| mean|g h| over std, each 80 u of its size, and h's error e times mean|g h| + mean|g|
   dw   (rows a block + 40) u of the sum of |dy h|, and the sum of |dy| e;  db  the same without h's part
plus half a step of the type."""
import math

import pytest
import torch

from oracle import language_head as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
PAIRS = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


def close(got, want, tol, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, (what, got.dtype, got.shape, want.shape)
    off = (got.double() - want).abs() - tol - want.abs() * (torch.finfo(dtype).eps / 2) - torch.finfo(dtype).tiny
    assert torch.equal(got.isnan(), want.isnan()), what
    off = off.nan_to_num(-1.0)
    assert bool((off <= 0).all()), "%s: off by %g more than allowed" % (what, float(off.max()))


def inputs(rows, d, dtype, par, seed=0, mean=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, d, generator=g, device="cuda") * (torch.rand(rows, 1, generator=g, device="cuda") + 0.5)
    x = (x + mean * torch.randn(rows, 1, generator=g, device="cuda")).to(dtype)
    w = (torch.randn(d, generator=g, device="cuda") * 0.3 + 1).to(par)
    b = (torch.randn(d, generator=g, device="cuda") * 0.3).to(par)
    return x, w, b, torch.randn(rows, d, generator=g, device="cuda").to(dtype)


def check(x, w, b, dy, eps=1e-5):
    import pytorch_loss as P
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = P.layer_norm(*leaves, eps)
    x64 = x.double()
    n = x.shape[-1]
    std = ((x64 - x64.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x64 - x64.mean(-1, keepdim=True)) / std
    e = (66 * x64.square().mean(-1, keepdim=True).sqrt() / std + 70 * h.abs() + 4) * U
    w64 = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    close(y.detach(), O.layer_norm(x, w, b, eps), w64.abs() * e + 2 * U * ((w64 * h).abs() + b64.abs()), x.dtype, "y")
    with torch.no_grad():
        assert torch.equal(P.layer_norm(x, w, b, eps), y.detach())
    there = [t for t in leaves if t is not None]
    got = list(torch.autograd.grad(y, there, dy))
    dx, dw, db = O.layer_norm_grads(x, w, eps, dy)
    d64 = dy.double()
    g = (d64 * w64).abs()
    mg, mgh = g.mean(-1, keepdim=True), (g * h.abs()).mean(-1, keepdim=True)
    he = e * (mg + mgh) + h.abs() * (g * e).mean(-1, keepdim=True)
    close(got.pop(0), dx, (80 * U * (g + mg + h.abs() * mgh) + he) / std, x.dtype, "dx")
    rows = x[..., 0].numel()
    per = (math.ceil(rows / 64) + 60) * U
    flat = lambda t: t.reshape(-1, n).sum(0)
    if w is not None:
        close(got.pop(0), dw, per * flat((d64 * h).abs()) + flat(d64.abs() * e), w.dtype, "dweight")
    if b is not None:
        close(got.pop(0), db, per * flat(d64.abs()), b.dtype, "dbias")


# below, at and above a vector, a warp's row, the blocks' rows; odd widths; beyond what registers hold
WIDTHS = [1, 2, 5, 8, 31, 64, 255, 256, 512, 513, 1000, 1003, 1024, 2048, 2056, 4096, 4100, 8192, 8193, 16384, 16392, 32768, 40001]


@pytest.mark.parametrize("dtype, par", PAIRS)
@pytest.mark.parametrize("d", WIDTHS)
def test_values_and_gradients(d, dtype, par):
    for rows in ((1, 7, 300) if d <= 4100 else (1, 19)):
        check(*inputs(rows, d, dtype, par, seed=d), eps=1e-5)


@pytest.mark.parametrize("dtype, par", PAIRS)
@pytest.mark.parametrize("rows, d", [(5000, 512), (3001, 1003), (2500, 4096), (20000, 64), (1200, 8192)])
def test_many_rows(rows, d, dtype, par):
    check(*inputs(rows, d, dtype, par, seed=d))


@pytest.mark.parametrize("d", [64, 1003, 4096, 40001])
def test_without_weight_or_bias(d):
    x, w, b, dy = inputs(11, d, torch.bfloat16, torch.float32)
    check(x, None, None, dy)
    check(x, w, None, dy)
    check(x, None, b, dy)


@pytest.mark.parametrize("d", [8, 300, 2048, 5000])
def test_rows_far_from_zero_and_constant_rows(d):
    """A mean 1000 times the spread loses no variance; a constant row has h = 0."""
    x, w, b, dy = inputs(9, d, torch.float32, torch.float32, mean=1000.0)
    x[3] = 5.0
    check(x, w, b, dy)
    x, w, b, dy = inputs(9, d, torch.float32, torch.float32)
    check(x * 1e-3, w, b, dy, eps=1e-12)


def test_eps_zero_and_one_column():
    import pytorch_loss as P
    x = torch.randn(5, 100, device="cuda")
    check(x, None, None, torch.randn_like(x), eps=0.0)
    one = torch.randn(5, 1, device="cuda")
    b = torch.randn(1, device="cuda")
    assert torch.equal(P.layer_norm(one, torch.ones(1, device="cuda"), b), b.expand(5, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_and_infinities_stay_in_their_rows(dtype):
    import pytorch_loss as P
    for d in (60, 1500, 6000, 50000):
        x, w, b, dy = inputs(6, d, dtype, dtype)
        want = P.layer_norm(x, w, b)
        y = x.clone()
        y[2, d // 2], y[4, 0] = math.nan, math.inf
        got = P.layer_norm(y, w, b)
        assert bool(got[2].isnan().all()) and bool(got[4].isnan().any())
        keep = [0, 1, 3, 5]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_layouts(dtype):
    """Leading dimensions, rows apart, rows off a 16-byte boundary, permuted images, an upstream gradient of any layout."""
    import pytorch_loss as P
    x, w, b, dy = inputs(24, 136, dtype, torch.float32)
    check(x.view(2, 3, 4, 136), w, b, dy.view(2, 3, 4, 136))
    wide = torch.randn(24, 200, device="cuda").to(dtype)
    check(wide[:, :136], w, b, dy)
    check(wide[:, 1:137], w, b, dy)
    check(wide[:, 64:], w, b, wide[:, :136])
    check(x, w, b, dy.t().contiguous().t())
    check(x, w, b, dy[:1].expand(24, 136))
    check(x.t().contiguous().t(), w, b, dy)
    check(x[:1].expand(24, 136), w, b, dy)
    image = torch.randn(2, 136, 5, 7, device="cuda").to(dtype).contiguous(memory_format=torch.channels_last)
    check(image.permute(0, 2, 3, 1), w, b, torch.randn(2, 5, 7, 136, device="cuda").to(dtype))
    off = torch.empty(137, device="cuda")[1:].copy_(w)
    check(x, off, b, dy)
    check(x, w.repeat_interleave(2)[::2], b, dy)


def test_which_gradients_are_made():
    import pytorch_loss as P
    x, w, b, dy = inputs(50, 640, torch.float32, torch.float32)
    full = torch.autograd.grad(P.layer_norm(*(l := [t.detach().requires_grad_(True) for t in (x, w, b)])), l, dy)
    for mask in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        leaves = [t.detach().requires_grad_(bool(m)) for t, m in zip((x, w, b), mask)]
        got = torch.autograd.grad(P.layer_norm(*leaves), [t for t, m in zip(leaves, mask) if m], dy)
        for a, e in zip(got, [f for f, m in zip(full, mask) if m]):
            assert torch.equal(a, e)


@pytest.mark.parametrize("d", [40, 3000, 40000])
def test_no_rows(d):
    import pytorch_loss as P
    m = P.LayerNorm(d).cuda()
    x = torch.zeros(0, d, device="cuda", requires_grad=True)
    m(x).sum().backward()
    assert x.grad.shape == (0, d) and float(m.weight.grad.abs().sum()) == 0.0 and float(m.bias.grad.abs().sum()) == 0.0


def test_gradient_against_differences():
    """Central differences of the 64-bit value, step 1e-4: error below 1e-7 for third derivatives of this size."""
    import pytorch_loss as P
    x, w, b, dy = inputs(3, 13, torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(P.layer_norm(*leaves), leaves, dy)
    value = lambda *a: (O.layer_norm(*a, 1e-5) * dy.double()).sum()
    base = [t.double() for t in (x, w, b)]
    for i, t in enumerate(base):
        want = torch.zeros_like(t)
        for j in range(t.numel()):
            d = torch.zeros_like(t)
            d.view(-1)[j] = 1e-4
            up, down = list(base), list(base)
            up[i], down[i] = t + d, t - d
            want.view(-1)[j] = (value(*up) - value(*down)) / 2e-4
        assert float((got[i].double() - want).abs().max()) < 2e-5 * float(want.abs().max() + 1)


def test_results_repeat_bit_for_bit():
    import pytorch_loss as P
    for rows, d in ((3000, 1024), (700, 4096), (333, 1003), (50, 40000)):
        x, w, b, dy = inputs(rows, d, torch.bfloat16, torch.float32)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        first = torch.autograd.grad(P.layer_norm(*leaves), leaves, dy)
        for _ in range(3):
            again = torch.autograd.grad(P.layer_norm(*leaves), leaves, dy)
            assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_offsets_past_32_bits():
    import pytorch_loss as P
    rows, d = 280000, 8192                                           # 2.3e9 elements, 4.6 GB
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    tail, w, b, dy = inputs(6, d, torch.bfloat16, torch.bfloat16)
    x[-6:] = tail
    up = torch.zeros_like(x)
    up[-6:] = dy
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = P.layer_norm(*leaves)
    small = [t.detach().requires_grad_(True) for t in (tail, w, b)]
    assert torch.equal(y[-6:].detach(), P.layer_norm(*small).detach())
    got = torch.autograd.grad(y, leaves, up)
    want = torch.autograd.grad(P.layer_norm(*small), small, dy)
    assert torch.equal(got[0][-6:], want[0]) and float(got[0][:-6].abs().max()) == 0.0
    for a, e in zip(got[1:], want[1:]):                              # (six terms, in another order)
        assert float((a.double() - e.double()).abs().max()) <= 2.0 ** -7 * float(e.double().abs().max())


def test_refusals_on_the_gpu():
    import pytorch_loss as P
    x, w, b, _ = inputs(4, 50, torch.float16, torch.float16)
    for a in ((x.double(), w, b), (x, w[:49], b), (x, w.bfloat16(), b), (x, w, b.float()), (x, w.unsqueeze(0), b),
              (x, w.cpu(), b), (x[:, :0], None, None)):
        with pytest.raises(RuntimeError):
            P.layer_norm(*a)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            P.layer_norm(x, w, b, eps)
