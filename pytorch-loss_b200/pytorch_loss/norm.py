"""Layer norm over the last dimension on the B200 CUDA library: forward in one read of the rows, backward in one read
of rows and upstream gradient that also leaves the sums for weight and bias.
"""
import torch
import torch.nn as nn

from . import _cabi


def _param_code(x, weight, bias):
    """Checks weight and bias; the code of their type (the rows' own where there are none)."""
    par = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or x.dim() < 1 or t.shape[0] != x.shape[-1]:
            raise RuntimeError("%s of shape %s does not match rows of %s" % (name, tuple(t.shape), tuple(x.shape)))
        if t.dtype is not par and (par is not None or t.dtype not in (x.dtype, torch.float32)):
            raise RuntimeError("weight and bias must both be float32 or both %s, got %s" % (x.dtype, t.dtype))
        par = t.dtype
    return _cabi.dtype_code(x) if par is None or par is x.dtype else _cabi.F32


# (allocations by *_like and new_empty: half the host time of torch.empty with a device)
def _forward(x, weight, bias, eps, want_stats):
    dev = _cabi.require_cuda(x, weight, bias)
    dt = _cabi.dtype_code(x)
    par = _param_code(x, weight, bias)
    if not 0.0 <= eps < float('inf'):
        raise ValueError("eps must be finite and not negative, got %s" % (eps,))
    flat, rows, d, stride = _cabi.as_rows(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    with _cabi.on_device(dev):
        _cabi.check(_cabi.load_library().b200_layer_norm(
            flat.data_ptr(), _cabi.ptr(weight), _cabi.ptr(bias), y.data_ptr(), _cabi.ptr(stats), rows, d, stride, dt, par,
            eps, _cabi.stream_ptr(dev)))
    return y, flat, weight, stats, par


class LayerNormFunc(torch.autograd.Function):
    """(x, weight or None, bias or None, eps) -> y."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, flat, w, stats, par = _forward(x, weight, bias, eps, True)
        # (the inputs themselves where the kernel read them, so that a change in place is noticed)
        ctx.save_for_backward(x if flat.data_ptr() == x.data_ptr() else flat,
                              weight if w is None or w.data_ptr() == weight.data_ptr() else w, stats)
        ctx.info = par, x.shape, None if bias is None else bias.dtype
        return y

    @staticmethod
    @_cabi.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        par, shape, bias_dtype = ctx.info
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        flat, rows, d, stride = _cabi.as_rows(x)
        dy, _, _, dy_stride = _cabi.as_rows(dy)
        dev = flat.device
        lib = _cabi.load_library()
        dx = flat.new_empty(shape)
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need_w else None
        db = flat.new_empty(d, dtype=bias_dtype) if need_b else None
        scratch, nbytes = None, 0
        if need_w or need_b:
            nbytes = lib.b200_layer_norm_scratch_bytes(rows, d)
            scratch = stats.new_empty(nbytes // 4)
        with _cabi.on_device(dev):
            _cabi.check(lib.b200_layer_norm_backward(
                flat.data_ptr(), _cabi.ptr(weight), stats.data_ptr(), dy.data_ptr(), dx.data_ptr(), _cabi.ptr(dw),
                _cabi.ptr(db), _cabi.ptr(scratch), nbytes, rows, d, stride, dy_stride, _cabi.dtype_code(flat), par,
                _cabi.stream_ptr(dev)))
        return dx if need_x else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x (float32, float16 or bfloat16); weight
    and bias, either of which may be missing, are float32 or of x's type.  Statistics and sums are float32, results
    have the type of what they belong to.  Rows may lie apart in memory (one stride between them); the result is
    contiguous."""
    eps = float(eps)
    if _cabi.tracked(x, weight, bias):
        return LayerNormFunc.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.Module):
    """Layer norm over rows of `size` elements (the last dimension), as in front of a language model's head:

        >>> norm = LayerNorm(4096).cuda()
        >>> logits = norm(hidden) @ head.t()        # hidden [..., 4096] float/half/bfloat16
    """

    def __init__(self, size, eps=1e-5, affine=True, bias=True):
        super().__init__()
        self.size, self.eps = int(size), float(eps)
        self.weight = nn.Parameter(torch.ones(self.size)) if affine else None
        self.bias = nn.Parameter(torch.zeros(self.size)) if affine and bias else None

    def forward(self, x):
        if x.dim() < 1 or x.shape[-1] != self.size:
            raise RuntimeError("rows of %d elements expected, got shape %s" % (self.size, tuple(x.shape)))
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%d, eps=%g, affine=%s, bias=%s" % (self.size, self.eps, self.weight is not None, self.bias is not None)
