"""The operators at a language model's output end together, as a training step and a server use them: one after the
other, captured and replayed, on other streams and from several threads."""
import threading

import pytest
import torch

from oracle import language_head as O

pytestmark = pytest.mark.gpu


def _model(rows=96, width=256, vocab=2048, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return make(rows, width), make(vocab, width) * 0.2, make(vocab, width) * 0.2, torch.randint(0, vocab, (rows,), generator=g, device="cuda")


def test_a_student_learns_from_a_teacher():
    """norm -> head -> the teacher's alternatives -> the student's loss, back to hidden states, norm and head; then one
    policy step on log probabilities and entropies.  All in float32 against 64 bits: the longest sums on the way have
    2048 terms, so 2048 u of a tensor's norm bounds what they lose."""
    import pytorch_loss as P
    tol = 2048 * 2.0 ** -24
    hidden, head, teacher_head, tokens = _model()
    tokens[::9] = -100
    norm = P.LayerNorm(256).cuda()
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5)
        norm.bias.normal_()
    hidden.requires_grad_(True)
    head.requires_grad_(True)
    logits = norm(hidden) @ head.t()
    with torch.no_grad():
        best = P.token_logprobs(norm(hidden) @ teacher_head.t(), tokens, top_k=16)
    assert bool((best.top_tokens[::9] == -1).all())
    loss = P.TopTokenDistillLoss(temperature=1.25)(logits, best.top_tokens, best.top_logprobs)
    out = P.token_logprobs(logits, tokens)
    total = loss - (out.logprobs * 0.1).mean() - 0.01 * out.entropy.sum()
    got = torch.autograd.grad(total, [hidden, head, norm.weight, norm.bias])

    h64, w64, nw, nb = (t.detach().double().requires_grad_(True) for t in (hidden, head, norm.weight, norm.bias))
    z = O.layer_norm(h64, nw, nb, 1e-5) @ w64.t()
    w, some = O.list_weights(best.top_tokens, best.top_logprobs)
    logp = torch.log_softmax(z / 1.25, -1).gather(-1, best.top_tokens.clamp(min=0))
    kl = (torch.where(w > 0, w * (w.clamp(min=1e-300).log() - logp), torch.zeros_like(w)).sum(-1) * some).sum() / some.sum()
    lp = torch.log_softmax(z, -1)
    valid = tokens != -100
    chosen = lp.gather(-1, tokens.clamp(min=0).unsqueeze(-1)).squeeze(-1) * valid
    entropy = -(lp.exp() * lp).sum(-1) * valid
    want_total = kl - (chosen * 0.1).mean() - 0.01 * entropy.sum()
    want = torch.autograd.grad(want_total, [h64, w64, nw, nb])
    assert abs(float(total.detach()) - float(want_total)) <= tol * abs(float(want_total))
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= tol * float(b.norm())


def _operators():
    import pytorch_loss as P
    g = torch.Generator(device="cuda").manual_seed(7)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")
    ids = torch.randint(0, 5000, (40,), generator=g, device="cuda")
    lists = torch.randint(-1, 5000, (40, 12), generator=g, device="cuda"), make(40, 12)
    d1, d2, dy = make(40), make(40), make(300, 1000).bfloat16()
    crit, w, b = P.TopTokenDistillLoss(), make(1000).requires_grad_(True), make(1000).requires_grad_(True)
    one = torch.ones((), device="cuda")

    def logprobs(x):
        out = P.token_logprobs(x, ids, top_k=9)
        return torch.autograd.grad((out.logprobs, out.entropy), x, (d1, d2)) + tuple(t.detach() for t in out)

    def distill(x):
        loss = crit(x, *lists)
        return torch.autograd.grad(loss, x, one) + (loss.detach(),)

    def norm(x):
        y = P.layer_norm(x, w, b)
        return torch.autograd.grad(y, (x, w, b), dy) + (y.detach(),)
    return {"logprobs": (logprobs, lambda: make(40, 5000)), "distill": (distill, lambda: make(40, 5000)),
            "distill16": (distill, lambda: make(40, 5000).half()), "norm": (norm, lambda: make(300, 1000).bfloat16())}


@pytest.mark.parametrize("name", ["logprobs", "distill", "distill16", "norm"])
def test_captured_and_replayed(name):
    """Two graphs of the same call, replayed at once on two streams, each on inputs of its own: nothing is shared."""
    call, make = _operators()[name]
    x = [make().requires_grad_(True) for _ in range(2)]
    new = [[make() for _ in range(2)] for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in x:
            call(t)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for t in x:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(t))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for pair in new:
        for t, v in zip(x, pair):
            t.detach().copy_(v)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, gr in zip(streams, graphs):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for o, v in zip(got, pair):
            for a, b in zip(o, call(v.clone().requires_grad_(True))):
                assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["logprobs", "distill", "distill16", "norm"])
def test_other_streams_and_threads(name):
    call, make = _operators()[name]
    inputs = [make() for _ in range(4)]
    want = [call(v.clone().requires_grad_(True)) for v in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(v, expected):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = call(v.clone().requires_grad_(True))
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                    bad.append("results differ")
        except Exception as e:                                       # noqa: BLE001
            bad.append(repr(e))
    threads = [threading.Thread(target=work, args=(v, w)) for v, w in zip(inputs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_second_derivatives_are_refused():
    import pytorch_loss as P
    x = torch.randn(4, 60, device="cuda", requires_grad=True)
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    outs = [P.token_logprobs(x, tok).logprobs.sum(), P.layer_norm(x).square().sum(),
            P.TopTokenDistillLoss()(x, tok.unsqueeze(1), torch.zeros(4, 1, device="cuda"))]
    for out in outs:
        g, = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_changes_in_place_are_noticed():
    import pytorch_loss as P
    x = torch.randn(4, 60, device="cuda", requires_grad=True)
    y = x * 1
    out = P.layer_norm(y)
    y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_modules_move_and_save():
    import pytorch_loss as P
    m = P.LayerNorm(48).cuda().bfloat16()
    x = torch.randn(3, 5, 48, device="cuda").bfloat16()
    n = P.LayerNorm(48).cuda()
    n.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    assert torch.equal(m(x), n(x)) and m(x).shape == x.shape
    bare = P.LayerNorm(48, affine=False).cuda()
    assert torch.equal(bare(x), m(x))
