"""Short causal convolution along the positions, channel by channel, in front of a recurrent mixer.

    y = short_convolution(x, weight, bias, "silu")                                          # a prompt, or training
    y, state = short_convolution(x, weight, bias, "silu", initial=state, return_state=True)   # what follows it

    pre[t] = bias + sum_k weight[:, k] * x[t - (W - 1) + k],    y = pre * sigmoid(pre)  or  pre

x: [B, S, C] float32 / float16 / bfloat16, the last dimension contiguous, any strides between positions and batch entries (a
slice of a wider projection needs no copy); weight: [C, W], W = 2, 3 or 4, and bias: [C] or None, of x's type or float32.
In front of position 0 stand ``initial`` ([B, W - 1, C], x's type) or zeros.  ``return_state`` gives the last W - 1 inputs, the
``initial`` of the next call; ``state_out`` names the tensor they are written to, which may be ``initial`` itself (a decoding
loop in a CUDA graph keeps one buffer).  The reference has no such operator.

Inputs that require gradients get them (no states in that case).
"""
import ctypes

import torch

from . import _lib

__all__ = ["short_convolution", "short_convolution_backward"]

_ACTIVATIONS = {None: 0, "silu": 1}


_Strides = ctypes.c_longlong * 2


def _check(x, weight, bias, activation):
    """(device, strides of x or None where it is contiguous)"""
    if x.dim() != 3 or not x.numel():
        raise ValueError("x must have the shape [B, S, C] with at least one of each")
    B, S, C = x.shape
    if B > 65535 or S > 1 << 23 or C > 1 << 24:      # (before they become 32 bits)
        raise ValueError("x must have at most 65535 batch entries, 2^23 positions and 2^24 channels")
    if weight.dim() != 2 or weight.shape[0] != C or not 2 <= weight.shape[1] <= 4:
        raise ValueError("weight must have the shape [C, W] with W = 2, 3 or 4")
    if activation not in _ACTIVATIONS:
        raise ValueError('activation must be None or "silu"')
    wdt = weight.dtype
    if wdt is not x.dtype and wdt is not torch.float32:
        raise TypeError("weight and bias must share one element type: x's or float32")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != C:
            raise ValueError("bias must have the shape [C]")
        if bias.dtype is not wdt:
            raise TypeError("weight and bias must share one element type: x's or float32")
    dev = _lib.require_one_cuda_device(x, weight, bias)
    if not weight.is_contiguous() or (bias is not None and not bias.is_contiguous()):
        raise RuntimeError("weight and bias must be contiguous")
    if x.is_contiguous():
        return dev, None
    s = x.stride()
    if s[2] != 1 and C != 1:
        raise RuntimeError("the last dimension of x must be contiguous")
    return dev, _Strides(s[0], s[1])


def _forward(checked, x, weight, bias, activation, initial=None, state_out=None):
    dev, strides = checked
    B, S, C = x.shape
    W = weight.shape[1]
    for name, t in (("initial", initial), ("state_out", state_out)):
        if t is not None and (t.shape != (B, W - 1, C) or t.dtype != x.dtype or not t.is_contiguous() or t.device != dev):
            raise ValueError(f"{name} must be a contiguous [B, W - 1, C] tensor of x's type and device")
    y = torch.empty_like(x) if strides is None else x.new_empty((B, S, C))
    with _lib.device_guard(dev):
        rc = _lib.lib().mlstm_conv_fwd(x.data_ptr(), weight.data_ptr(), _lib.ptr(bias), _lib.ptr(initial), strides, y.data_ptr(),
                                       _lib.ptr(state_out), B, S, C, W, _lib.dtype_code(x), _lib.dtype_code(weight),
                                       _ACTIVATIONS[activation], _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_conv_fwd")
    return y


def short_convolution_backward(dy, x, weight, bias=None, activation=None):
    """Gradients (dx, dweight, dbias) of ``short_convolution`` without states; dbias is None where there is no bias."""
    return _backward(_check(x, weight, bias, activation), dy, x, weight, bias, activation)


def _backward(checked, dy, x, weight, bias, activation):
    dev, strides = checked
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy must match x in shape and element type")
    _lib.require_cuda(dy, weight)
    B, S, C = x.shape
    W = weight.shape[1]
    dt = _lib.dtype_code(x)
    L = _lib.lib()
    dx = torch.empty_like(x) if strides is None else x.new_empty((B, S, C))
    dweight = torch.empty_like(weight)
    dbias = None if bias is None else torch.empty_like(bias)
    ws, at, nbytes = _lib.scratch(L.mlstm_conv_bwd_workspace(B, S, C, W, dt), dev)
    with _lib.device_guard(dev):
        rc = L.mlstm_conv_bwd(dy.data_ptr(), x.data_ptr(), weight.data_ptr(), _lib.ptr(bias), strides, dx.data_ptr(),
                              dweight.data_ptr(), _lib.ptr(dbias), at, nbytes, B, S, C, W, dt, _lib.dtype_code(weight),
                              _ACTIVATIONS[activation], _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_conv_bwd")
    return dx, dweight, dbias


class _ShortConvolution(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        ctx.save_for_backward(x, weight, bias)
        ctx.activation = activation
        return _forward(_check(x, weight, bias, activation), x, weight, bias, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        saved = ctx.saved_tensors       # (their strides may be others than the forward's: hooks may have moved them away and back)
        return _backward(_check(*saved, ctx.activation), dy.contiguous(), *saved, ctx.activation) + (None,)


def short_convolution(x, weight, bias=None, activation=None, initial=None, return_state=False, state_out=None):
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (initial is not None and initial.requires_grad)):
        if initial is not None or return_state or state_out is not None:
            raise ValueError("gradients are available for the plain call: no initial / return_state / state_out")
        return _ShortConvolution.apply(x, weight, bias, activation)
    if not return_state:
        if state_out is not None:
            raise ValueError("state_out needs return_state")
        return _forward(_check(x, weight, bias, activation), x, weight, bias, activation, initial)
    checked = _check(x, weight, bias, activation)
    if state_out is None:
        state_out = (torch.empty_like(initial) if initial is not None and initial.is_contiguous()
                     else x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])))
    return _forward(checked, x, weight, bias, activation, initial, state_out), state_out
