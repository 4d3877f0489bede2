"""The operators at a language model's output end where a program goes beyond their plain use: losses changed in place,
forward-mode differentiation, batches without rows, what a call allocates, results that have to be exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _distill_inputs(rows=6, v=3000, k=4, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(rows, v, generator=g, device="cuda").to(dtype)
    tok = torch.randint(0, v, (rows, k), generator=g, device="cuda")
    return x, tok, torch.randn(rows, k, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_a_loss_may_be_changed_in_place(reduction, dtype):
    """`loss += other` and `loss *= w`, as programs with several losses do; v = 500 takes two passes in every type.
    Upstream gradients of 1 and 0.5 are powers of two: gradients are equal bit for bit."""
    import pytorch_loss as P
    crit = P.TopTokenDistillLoss(reduction=reduction)
    for v in (500, 3000):
        x, tok, q = _distill_inputs(v=v, dtype=dtype)
        other = torch.ones((), device="cuda", requires_grad=True)
        want_loss, want = [], []
        for w in (1.0, 0.5):
            leaf = x.clone().requires_grad_(True)
            loss = crit(leaf, tok, q)
            want_loss.append(loss.detach() * w + 1)
            want += torch.autograd.grad(loss * w, leaf)
        for w, wl, wg in zip((1.0, 0.5), want_loss, want):
            leaf = x.clone().requires_grad_(True)
            loss = crit(leaf, tok, q)
            if w != 1.0:
                loss *= w
            loss += other
            loss.backward()
            assert torch.equal(loss.detach(), wl) and torch.equal(leaf.grad, wg)
        assert float(other.grad) == 2.0
        with torch.no_grad():
            total = crit(x, tok, q)
        total += other                                       # a loss taken without a graph, in a sum that has one
        total.backward()
        assert float(other.grad) == 3.0 and torch.equal(total.detach(), want_loss[0])


def test_forward_mode_is_refused():
    """A tangent is never dropped in silence."""
    import torch.autograd.forward_ad as fwAD
    import pytorch_loss as P
    x, tok, q = _distill_inputs()
    w, b = torch.ones(3000, device="cuda"), torch.zeros(3000, device="cuda")
    crit = P.TopTokenDistillLoss()
    calls = [lambda d: P.token_logprobs(d(x), tok[:, 0]), lambda d: P.token_logprobs(d(x), tok[:, 0], top_k=3),
             lambda d: crit(d(x), tok, q), lambda d: P.TopTokenDistillLoss(reduction='none')(d(x), tok, q),
             lambda d: P.layer_norm(d(x), w, b), lambda d: P.layer_norm(x, d(w), b), lambda d: P.layer_norm(x, w, d(b)),
             lambda d: P.layer_norm(d(x))]
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            for call in calls:
                with pytest.raises(NotImplementedError):
                    call(lambda t: fwAD.make_dual(t, torch.ones_like(t)))
                call(lambda t: t)                            # (no tangent: nothing to refuse)


@pytest.mark.parametrize("dtype, par", [(torch.float32, torch.float32), (torch.float16, torch.float32),
                                        (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("d", [256, 1024, 4096, 8192, 16384])
def test_constant_rows_leave_the_weight_alone(d, dtype, par):
    """Rows of one value c, of few bits, and d a power of two: every partial sum is exact (a share of 2^k values of at
    most 24 - 14 bits), the mean is c and h = 0 exactly, so the weight's gradient is 0, y is the bias and a row's dx is
    r (g - mean g) -- in the forward kernel's sense and in the backward kernel's."""
    import pytorch_loss as P
    c = torch.tensor([1000.0, -1004.0, 0.5, 120.0, 5.0], device="cuda").to(dtype)
    x = c.unsqueeze(1).expand(5, d).contiguous().requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(d)
    w = torch.randn(d, generator=g, device="cuda").to(par).requires_grad_(True)
    b = torch.randn(d, generator=g, device="cuda").to(par).requires_grad_(True)
    dy = torch.randn(5, d, generator=g, device="cuda").to(dtype)
    y = P.layer_norm(x, w, b)
    assert torch.equal(y.detach(), b.detach().to(dtype).expand(5, d))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert float(dw.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [30, 3000])
def test_no_rows_give_no_losses(v, dtype):
    import pytorch_loss as P
    crit = P.TopTokenDistillLoss(reduction='none')
    for shape in ((0,), (0, 3), (3, 0)):
        x = torch.zeros(shape + (v,), device="cuda", dtype=dtype)
        lists = torch.zeros(shape + (4,), dtype=torch.int64, device="cuda"), torch.zeros(shape + (4,), device="cuda")
        assert crit(x, *lists).shape == shape
        x.requires_grad_(True)
        losses = crit(x, *lists)
        assert losses.shape == shape and losses.dtype == torch.float32
        losses.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("rows, v, pad, dtype", [(64, 131072, 0, torch.float32), (4000, 1000, 0, torch.float32),
                                                 (500, 20001, 47, torch.bfloat16)])
def test_a_layout_without_the_step_allocates_no_gradient_forward(rows, v, pad, dtype):
    """Rows above 320 KB or up to 4 KB, rows off the gradient's place: two passes.  Forward keeps 24 + 4 K bytes a row."""
    import pytorch_loss as P
    x, tok, q = _distill_inputs(rows, v + pad, 4, dtype)
    leaf = x[:, :v].requires_grad_(True)
    tok = tok.clamp(max=v - 1)
    crit = P.TopTokenDistillLoss()
    crit(leaf, tok, q)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = crit(leaf, tok, q)
    assert torch.cuda.max_memory_allocated() - before < leaf.numel() * leaf.element_size() // 4
    loss.backward()


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("v", [2056, 9000, 32768, 50001, 131072])
def test_a_scaled_gradient_is_rounded_once(v, reduction):
    """The one-pass step in bfloat16 under an upstream gradient that is no power of two: half a step of the type and what
    its float32 arithmetic loses, as without one.  The second trip through the graph gives the same bits."""
    import pytorch_loss as P
    from test_top_distill_gpu import U, close, expected, inputs
    x, tok, q = inputs(300, v, 20, torch.bfloat16, seed=v, ragged=True)
    _, grad, counted, _, gtol = expected(x, tok, q, 1.25)
    scale = 0.3 / (int(counted.sum()) if reduction == "mean" else 1)
    leaf = x.detach().requires_grad_(True)
    loss = P.TopTokenDistillLoss(1.25, reduction)(leaf, tok, q)
    up = torch.tensor(0.3, device="cuda")
    got, = torch.autograd.grad(loss, leaf, up, retain_graph=True)
    want = grad * scale
    close(got, want, gtol * scale + want.abs() * (torch.finfo(torch.bfloat16).eps / 2 + 8 * U) + 2.0 ** -126, "gradient")
    again, = torch.autograd.grad(loss, leaf, up)
    assert torch.equal(got, again)


@pytest.mark.parametrize("rows", [5, 4000])
def test_a_step_under_one_upstream_gradient_then_another(rows):
    """A captured backward pass is replayed with upstream gradients of 1, 0.3 and 1 again: each replay gives what an
    eager call gives."""
    import pytorch_loss as P
    x, tok, q = _distill_inputs(rows, 5001, 7, torch.bfloat16)
    crit, up = P.TopTokenDistillLoss(), torch.ones((), device="cuda")
    leaf = x.clone().requires_grad_(True)
    call = lambda: torch.autograd.grad(crit(leaf, tok, q), leaf, up)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for value in (1.0, 0.3, 1.0):
        up.fill_(value)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, call())


def test_steps_notice_changed_logits():
    """What a bfloat16 step's backward may have to read again must not have changed meanwhile."""
    import pytorch_loss as P
    x, tok, q = _distill_inputs(6, 5001, 4, torch.bfloat16)
    y = x.requires_grad_(True) * 1
    loss = P.TopTokenDistillLoss()(y, tok, q)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v, pad", [(3000, 8), (5001, 3), (700, 4)])
def test_saved_tensors_may_move(v, pad, dtype):
    """What backward reads comes from autograd's saved tensors, wherever hooks have put them and with whatever strides."""
    import pytorch_loss as P
    x, tok, q = _distill_inputs(50, v + pad, 6, dtype)
    tok, leaf = tok.clamp(max=v - 1), x.requires_grad_(True)
    w, b = torch.randn(v, device="cuda"), torch.randn(v, device="cuda")
    up, d, dy = torch.tensor(0.3, device="cuda"), torch.randn(50, device="cuda"), torch.randn(50, v, device="cuda").to(dtype)
    for call, g in ((lambda y: P.TopTokenDistillLoss()(y, tok, q), up), (lambda y: P.token_logprobs(y, tok[:, 0]).logprobs, d),
                    (lambda y: P.layer_norm(y, w, b), dy)):
        want, = torch.autograd.grad(call(leaf[:, :v]), leaf, g)
        with torch.autograd.graph.save_on_cpu():
            out = call(leaf[:, :v])
        got, = torch.autograd.grad(out, leaf, g)
        assert torch.equal(got, want)
