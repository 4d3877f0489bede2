"""What the operators at a language model's output end refuse, on the CPU: the C entries before they touch a device, the
Python side before it reaches the library."""
import ctypes

import pytest
import torch

A = ctypes.c_void_p(0x7f0000001000)         # (addresses are made up: every call here is refused before it uses them)
ODD = ctypes.c_void_p(0x7f0000001001)
F32, F16, BF16, F64 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    import build as b200_build
    b200_build.build()
    from pytorch_loss import _cabi
    return _cabi.load_library()


def _logprobs(lib, x=A, tokens=A, lp=A, h=A, stats=None, top=A, ids=A, rows=4, v=100, stride=100, dt=F32, k=5, t=1.0):
    return lib.b200_token_logprobs(x, tokens, lp, h, stats, top, ids, rows, v, stride, dt, k, t, -100, None)


@pytest.mark.parametrize("change, code, words", [
    ({"rows": -1}, 1, b"rows"), ({"v": 0}, 1, b"V >= 1"), ({"stride": -1}, 1, b"stride"), ({"dt": F64}, 1, b"dtype"),
    ({"t": 0.0}, 1, b"temperature"), ({"t": float("nan")}, 1, b"temperature"), ({"t": float("inf")}, 1, b"temperature"),
    ({"t": -1.0}, 1, b"temperature"), ({"k": 129, "v": 1000}, 1, b"top_k"), ({"k": 101}, 1, b"top_k"),
    ({"k": -1}, 1, b"top_k"), ({"x": None}, 1, b"null"), ({"x": ODD}, 1, b"aligned"), ({"tokens": None}, 1, b"null"),
    ({"lp": None}, 1, b"null"), ({"h": None}, 1, b"null"), ({"top": None}, 1, b"null"), ({"ids": None}, 1, b"null"),
    ({"stats": ODD}, 1, b"16 bytes"), ({"rows": 1 << 28}, 2, b"rows"), ({"v": (1 << 30) + 1}, 2, b"2^30"),
])
def test_token_logprobs_refuses(lib, change, code, words):
    assert _logprobs(lib, **change) == code
    assert words in lib.b200_last_error()


def test_token_logprobs_backward_refuses(lib):
    call = lambda x=A, tok=A, st=A, g=A, rows=4, dt=F16, t=1.0: lib.b200_token_logprobs_backward(
        x, tok, st, None, None, g, rows, 100, 100, dt, t, -100, None)
    for change in ({"x": None}, {"tok": None}, {"st": None}, {"st": ODD}, {"g": None}, {"g": ODD}, {"dt": 9}, {"t": 0.0}):
        assert call(**change) == 1, change
    assert call(rows=0) == 0                                     # nothing to do


def test_top_distill_refuses(lib):
    need = lib.b200_top_distill_scratch_bytes(4, 8)
    assert need >= 4 * (16 + 4 + 4 + 32) and lib.b200_top_distill_scratch_bytes(-1, 8) == 0

    def fwd(x=A, tok=A, q=A, losses=A, out=A, sc=A, n=need, rows=4, k=8, t=1.0, dt=F32):
        return lib.b200_top_distill_forward(x, tok, q, losses, out, sc, n, rows, 100, 100, dt, k, t, None)
    for change, code in (({"x": None}, 1), ({"tok": None}, 1), ({"q": None}, 1), ({"losses": None, "out": None}, 1),
                         ({"sc": None}, 5), ({"sc": ODD}, 5), ({"n": need - 1}, 5), ({"k": 0}, 1), ({"k": 129}, 1),
                         ({"t": 1e5}, 1), ({"dt": F64}, 1)):
        assert fwd(**change) == code, change

    def bwd(d=A, g=A, count=None, dt=F32):
        return lib.b200_top_distill_backward(A, A, A, need, d, 1, count, g, 4, 100, 100, dt, 8, 1.0, None)
    for change in ({"d": None}, {"g": None}, {"g": ODD}, {"count": ODD}):
        assert bwd(**change) == 1, change

    def step(g=A, out=A, dt=F32, v=100, stride=100, q=A):
        return lib.b200_top_distill_step(A, A, q, g, out, A, need, 4, v, stride, dt, 8, 1.0, 1, None)
    for change in ({"g": None}, {"out": None}, {"q": None}, {"dt": F16}, {"g": ctypes.c_void_p(0x7f0000001004)},
                   {"stride": 101}):
        assert step(**change) == 2, change


def test_which_layouts_have_the_one_pass_step(lib):
    q = lambda rows, v, stride, dt, g=A: lib.b200_top_distill_step_path(A, g, rows, v, stride, dt)
    assert q(4, 32768, 32768, F32) == 1 and q(4, 131072, 131072, BF16) == 1
    assert q(4, 50001, 50001, F32) == 1                          # odd rows: gradient rows lie like the logits'
    assert q(4, 50001, 50048, F32) == 0 and q(1, 50001, 50048, F32) == 1
    assert q(4, 81920, 81920, F32) == 1 and q(4, 81921, 81921, F32) == 0          # rows of more than 4 to 320 KB
    assert q(4, 1025, 1025, F32) == 1 and q(4, 1024, 1024, F32) == 0 and q(4, 2048, 2048, BF16) == 0
    assert q(4, 32768, 32768, F16) == 0 and q(0, 32768, 32768, F32) == 0
    assert q(4, 32768, 32768, F32, ctypes.c_void_p(0x7f0000001004)) == 0


def test_layer_norm_refuses(lib):
    def fwd(x=A, y=A, st=A, rows=4, d=64, stride=64, dt=F16, par=F16, eps=1e-5):
        return lib.b200_layer_norm(x, A, A, y, st, rows, d, stride, dt, par, eps, None)
    for change, code in (({"x": None}, 1), ({"y": None}, 1), ({"st": ctypes.c_void_p(0x7f0000001004)}, 1),
                         ({"rows": -1}, 1), ({"d": 0}, 1), ({"stride": -1}, 1), ({"dt": F64}, 1), ({"par": BF16}, 1),
                         ({"eps": -1.0}, 1), ({"eps": float("nan")}, 1), ({"rows": 1 << 31}, 2), ({"d": 1 << 31}, 2)):
        assert fwd(**change) == code, change
    need = lib.b200_layer_norm_scratch_bytes(4, 64)
    assert need > 0 and lib.b200_layer_norm_scratch_bytes(-1, 64) == 0

    def bwd(x=A, st=A, dy=A, dx=A, sc=A, n=need):
        return lib.b200_layer_norm_backward(x, A, st, dy, dx, A, A, sc, n, 4, 64, 64, 64, F16, F16, None)
    for change, code in (({"x": None}, 1), ({"st": None}, 1), ({"dy": None}, 1), ({"dx": None}, 1), ({"sc": None}, 5),
                         ({"sc": ODD}, 5), ({"n": need - 1}, 5)):
        assert bwd(**change) == code, change


def test_pointers_off_their_type_are_refused(lib):
    four, two = ctypes.c_void_p(0x7f0000001004), ctypes.c_void_p(0x7f0000001002)
    for change in ({"tokens": four}, {"ids": four}, {"lp": two}, {"h": two}, {"top": two}, {"x": two}):
        assert _logprobs(lib, **change) == 1, change
    back = lambda tok=A, dl=A, dh=A, g=A: lib.b200_token_logprobs_backward(A, tok, A, dl, dh, g, 4, 100, 100, F32, 1.0, -100, None)
    for change in ({"tok": four}, {"dl": two}, {"dh": two}, {"g": two}):
        assert back(**change) == 1, change
    need = lib.b200_top_distill_scratch_bytes(4, 8)
    fwd = lambda tok=A, q=A, losses=A, out=A: lib.b200_top_distill_forward(A, tok, q, losses, out, A, need, 4, 5000, 5000, F32, 8, 1.0, None)
    for change in ({"tok": four}, {"q": two}, {"losses": two}, {"out": four}):
        assert fwd(**change) == 1, change
    step = lambda tok=A, q=A, out=A: lib.b200_top_distill_step(A, tok, q, A, out, A, need, 4, 5000, 5000, F32, 8, 1.0, 1, None)
    for change in ({"tok": four}, {"q": two}, {"out": four}):
        assert step(**change) == 1, change
    norm = lambda x=A, w=A, b=A, y=A: lib.b200_layer_norm(x, w, b, y, A, 4, 64, 64, F16, F32, 1e-5, None)
    for change in ({"x": ODD}, {"y": ODD}, {"w": two}, {"b": two}):
        assert norm(**change) == 1, change
    n = lib.b200_layer_norm_scratch_bytes(4, 64)
    grad = lambda x=A, w=A, dy=A, dx=A, dw=A, db=A: lib.b200_layer_norm_backward(x, w, A, dy, dx, dw, db, A, n, 4, 64, 64, 64, F16, F32, None)
    for change in ({"x": ODD}, {"dy": ODD}, {"dx": ODD}, {"w": two}, {"dw": two}, {"db": two}):
        assert grad(**change) == 1, change


def test_cpu_tensors_are_refused():
    import pytorch_loss as P
    x, t = torch.randn(3, 10), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="gpu"):
        P.token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="gpu"):
        P.TopTokenDistillLoss()(x, t.unsqueeze(1), torch.zeros(3, 1))
    with pytest.raises(RuntimeError, match="gpu"):
        P.layer_norm(x)
    with pytest.raises(RuntimeError, match="16 elements"):
        P.LayerNorm(16)(x)
    with pytest.raises(ValueError, match="temperature"):
        P.TopTokenDistillLoss(temperature=0.0)


def test_rows_of_any_layout():
    """One stride describes the rows, or a copy is made."""
    from pytorch_loss import _cabi
    x = torch.arange(2 * 3 * 8.).reshape(2, 3, 8)
    for t, stride, same in ((x, 8, True), (x[..., :5], 8, True), (x[0], 8, True), (x[0, 0], 8, True),
                            (x[:, 0], 24, True), (x.transpose(0, 1), 8, False), (x.transpose(1, 2), 3, False),
                            (x[..., ::2], 4, False), (x[:, :0], 8, None), (x[..., :1], 8, True),
                            (x[:1, :1].expand(2, 3, 8), 0, None)):
        flat, rows, n, step = _cabi.as_rows(t)
        assert n == t.shape[-1] and rows == t.numel() // n
        assert torch.equal(flat, t.reshape(rows, n))
        if same is not None:
            assert (flat.data_ptr() == t.data_ptr()) == same and (rows < 2 or step == stride)
        if rows > 1:
            assert torch.equal(flat.as_strided((rows, n), (step, 1)), flat)
    with pytest.raises(RuntimeError):
        _cabi.as_rows(torch.zeros(()))
    with pytest.raises(RuntimeError):
        _cabi.as_rows(torch.zeros(3, 0))


def test_module_defaults():
    import pytorch_loss as P
    d, n = P.TopTokenDistillLoss(), P.LayerNorm(8)
    assert (d.temperature, d.reduction) == (1.0, 'mean') and len(d.state_dict()) == 0
    assert n.eps == 1e-5 and set(n.state_dict()) == {"weight", "bias"}
    assert set(P.LayerNorm(8, bias=False).state_dict()) == {"weight"} and not P.LayerNorm(8, affine=False).state_dict()
