"""The operators at a language model's output end: host logic of what lies beyond their plain use, on the CPU."""
import ctypes

import torch
import torch.autograd.forward_ad as fwAD


def test_which_calls_autograd_has_to_see():
    from pytorch_loss import _cabi
    x, w = torch.zeros(3), torch.zeros(3, requires_grad=True)
    assert not _cabi.tracked(x) and not _cabi.tracked(x, None) and not _cabi.tracked(None)
    assert _cabi.tracked(w) and _cabi.tracked(x, None, w)
    with torch.no_grad():
        assert not _cabi.tracked(x, w)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones(3))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                assert _cabi.tracked(dual) and _cabi.tracked(x, None, dual) and not _cabi.tracked(x)


def test_no_rows_need_no_address_for_their_losses():
    """An empty tensor's pointer is null: the losses of no rows are nothing to do, not an error."""
    import build as b200_build
    b200_build.build()
    from pytorch_loss import _cabi
    lib = _cabi.load_library()
    made_up = ctypes.c_void_p(0x7f0000001000)               # (never used: there is nothing to do)
    need = lib.b200_top_distill_scratch_bytes(0, 4)
    call = lambda rows: lib.b200_top_distill_forward(None if rows == 0 else made_up, None if rows == 0 else made_up,
                                                     None if rows == 0 else made_up, None, None, made_up, 1 << 20, rows,
                                                     100, 100, _cabi.F32, 4, 1.0, None)
    assert need <= 1 << 20 and call(0) == 0 and call(3) == 1


def test_step_backward_refuses():
    import build as b200_build
    b200_build.build()
    from pytorch_loss import _cabi
    lib = _cabi.load_library()
    at = lambda a: ctypes.c_void_p(0x7f0000001000 + a)      # (never used: every call is refused before it is)
    need = lib.b200_top_distill_scratch_bytes(4, 8)

    def call(x=at(0), tok=at(0), sc=at(0), n=need, d=at(0), count=at(0), g=at(0), v=5000, stride=5000, dt=_cabi.BF16, k=8, t=1.0):
        return lib.b200_top_distill_step_backward(x, tok, sc, n, d, count, g, 4, v, stride, dt, k, t, None)
    for change, code in (({"x": None}, 1), ({"tok": None}, 1), ({"tok": at(4)}, 1), ({"sc": None}, 5), ({"n": need - 1}, 5),
                         ({"d": None}, 1), ({"d": at(2)}, 1), ({"count": at(4)}, 1), ({"g": None}, 2), ({"g": at(4)}, 2),
                         ({"dt": _cabi.F32}, 2), ({"dt": _cabi.F16}, 2), ({"v": 2000, "stride": 2000}, 2), ({"stride": 5001}, 2),
                         ({"k": 0}, 1), ({"t": 0.0}, 1)):
        assert call(**change) == code, change
