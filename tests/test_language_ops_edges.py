"""The operators at a language model's output end: host logic of what lies beyond their plain use, on the CPU."""
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
