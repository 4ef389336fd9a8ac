"""Root-mean-square norm with the residual's addition, and with its result in 8 bits.

    y = residual_rms_norm(x, weight)
    y, stream = residual_rms_norm(x, weight, residual=stream)        # stream + x, and its norm, in one pass
    q, scale = residual_rms_norm_quantized(x, weight, block=128)     # q.float() * scale (per 128 values) is the norm

    s = x + residual (in the residual's type),   y = s / sqrt(mean(s^2) + eps) * weight        over the last dimension D <= 16384

x: contiguous, float32 / float16 / bfloat16; residual: x's type or float32; weight: [D] (x's type or float32), None for ones, or
[NH, D] for an x of shape [B, NH, S, D]: a norm of its own for every head of a mixer's result, as ``mlstm_scan`` and
``mlstm_matmul`` return it.  What is normalised is the sum as it is returned, rounded to the stream's type, so that the gradients
are those of the values that the next layer sees.  ``out_dtype``: x's type by default; any type where the stream (x, or
the residual) is float32.  Squares are summed in float32, so magnitudes above 1e19 overflow.

Inputs that require gradients get them, through the norm and through the sum.  The quantized form has none: its result feeds an
8-bit product.  The reference has neither; they stand beside ``output_gate_forward`` in what follows a mixer.
"""
import torch

from . import _lib

__all__ = ["residual_rms_norm", "residual_rms_norm_backward", "residual_rms_norm_quantized"]


def _check(x, weight, residual, w_dtype=None):
    """(device, rows, D, groups, inner) of x with this weight; ``w_dtype``: a type that the weight may have beside x's and float32."""
    if x.dim() < 1 or x.numel() == 0:
        raise ValueError("x must have at least one row of at least one value")
    D = x.shape[-1]
    if D > 16384:
        raise ValueError("the last dimension of x must be at most 16384")
    groups, inner = 1, 1
    if weight is not None:
        if weight.shape != (D,):
            if x.dim() != 4 or weight.shape != (x.shape[1], D):
                raise ValueError("weight must have the shape [D], or [NH, D] for x [B, NH, S, D]")
            groups, inner = x.shape[1], x.shape[2]
        if weight.dtype not in (x.dtype, torch.float32, w_dtype):
            raise TypeError("weight must have x's element type or float32")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError("residual must have x's element type or float32")
    dev = _lib.require_one_cuda_device(x, weight, residual)
    for name, t in (("x", x), ("weight", weight), ("residual", residual)):
        if t is not None and not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    return dev, x.numel() // D, D, groups, inner


def _forward(checked, x, weight, residual, eps, out, scale, block):
    dev, rows, D, groups, inner = checked
    total = None if residual is None else torch.empty_like(residual)
    stream = x if residual is None else residual
    with _lib.device_guard(dev):
        rc = _lib.lib().mlstm_rms_fwd(x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), out.data_ptr(), _lib.ptr(total), _lib.ptr(scale), rows, D,
                                      groups, inner, block, eps, _lib.dtype_code(x), _lib.dtype_code(stream),
                                      0 if weight is None else _lib.dtype_code(weight), 0 if scale is not None else _lib.dtype_code(out),
                                      _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_rms_fwd")
    return total


def residual_rms_norm_backward(dy, s, weight=None, ds=None, eps=1e-6, x_dtype=None):
    """Gradients (dx, dresidual, dweight): ``s`` is the sum (x where there was no residual), ``ds`` the gradient that the sum gets
    from its later uses or None.  dx has ``x_dtype`` (default: that of s) and dresidual the type of s; where these are the same
    type they are one tensor."""
    return _backward(_check(s, weight, None, x_dtype), dy, s, weight, ds, eps, x_dtype)


def _backward(checked, dy, s, weight, ds, eps, x_dtype):
    dev, rows, D, groups, inner = checked
    if dy.shape != s.shape or (dy.dtype != s.dtype and s.dtype != torch.float32):
        raise ValueError("dy must have the shape of s, and its element type unless that is float32")
    if ds is not None and (ds.shape != s.shape or ds.dtype != s.dtype):
        raise ValueError("ds must match s in shape and element type")
    _lib.require_cuda(s, dy, *(() if ds is None else (ds,)), *(() if weight is None else (weight,)))
    x_dtype = s.dtype if x_dtype is None else x_dtype
    dx = torch.empty(s.shape, dtype=x_dtype, device=dev)
    dres = dx if x_dtype == s.dtype else torch.empty_like(s)
    dweight = None if weight is None else torch.empty_like(weight)
    L = _lib.lib()
    ws, at, nbytes = _lib.scratch(0 if weight is None else L.mlstm_rms_bwd_workspace(rows, D, groups, inner), dev)
    with _lib.device_guard(dev):
        rc = L.mlstm_rms_bwd(dy.data_ptr(), _lib.ptr(ds), s.data_ptr(), _lib.ptr(weight), dx.data_ptr(), None if dres is dx else dres.data_ptr(),
                             _lib.ptr(dweight), at, nbytes, rows, D, groups, inner, eps, _lib.dtype_code(dx), _lib.dtype_code(s),
                             0 if weight is None else _lib.dtype_code(weight), _lib.dtype_code(dy), _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_rms_bwd")
    return dx, dres, dweight


class _ResidualRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, out_dtype):
        ctx.checked = _check(x, weight, residual)
        y = torch.empty_like(x) if out_dtype is x.dtype else torch.empty_like(x, dtype=out_dtype)
        total = _forward(ctx.checked, x, weight, residual, eps, y, None, 0)
        ctx.save_for_backward(x if total is None else total, weight)
        ctx.eps, ctx.x_dtype, ctx.with_residual = eps, x.dtype, residual is not None
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        s, weight = ctx.saved_tensors
        if dy is None:          # only the sum was used
            return (None if ds is None else ds.to(ctx.x_dtype)), None, ds, None, None
        dx, dres, dweight = _backward(ctx.checked, dy.contiguous(), s, weight, None if ds is None else ds.contiguous(), ctx.eps,
                                      ctx.x_dtype)
        return dx, dweight, dres if ctx.with_residual else None, None, None


def residual_rms_norm(x, weight=None, residual=None, eps=1e-6, out_dtype=None):
    out_dtype = x.dtype if out_dtype is None else out_dtype
    stream = x if residual is None else residual
    if out_dtype not in (torch.float32, torch.float16, torch.bfloat16) or (out_dtype != stream.dtype and stream.dtype != torch.float32):
        raise TypeError("out_dtype must be the type of the stream (x, or the residual), or any where that is float32")
    if torch.is_grad_enabled() and any([t.requires_grad for t in (x, weight, residual) if t is not None]):
        return _ResidualRmsNorm.apply(x, weight, residual, float(eps), out_dtype)
    checked = _check(x, weight, residual)
    y = torch.empty_like(x) if out_dtype is x.dtype else torch.empty_like(x, dtype=out_dtype)
    total = _forward(checked, x, weight, residual, float(eps), y, None, 0)
    return y if total is None else (y, total)


def residual_rms_norm_quantized(x, weight=None, residual=None, eps=1e-6, block=None):
    """(q, scale), with a residual (q, scale, s).  q: float8_e4m3fn, x's shape; scale: float32, x's shape with the last dimension
    D / block: the largest magnitude of a row, or of each ``block`` (32, 64, 128) of its values, divided by 448 (1 where all are
    zero; rounded up below the normal numbers, so that the least of blocks has one that is not 0).  Values are the nearest to their
    quotients by that scale (ties to even); a block with an infinity or a NaN gets that as its scale."""
    if torch.is_grad_enabled() and any([t.requires_grad for t in (x, weight, residual) if t is not None]):
        raise ValueError("the quantized norm has no gradients")
    D = x.shape[-1] if x.dim() else 0
    if block is not None and (block not in (32, 64, 128) or D % block):
        raise ValueError("block must be None (one scale per row), 32, 64 or 128, and divide the last dimension")
    block = D if block is None else block
    checked = _check(x, weight, residual)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x.shape[:-1] + (D // block,), dtype=torch.float32, device=x.device)
    total = _forward(checked, x, weight, residual, float(eps), q, scale, block)
    return (q, scale) if total is None else (q, scale, total)
