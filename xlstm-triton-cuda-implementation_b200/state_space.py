"""Selective state space scan: a recurrent mixer with N states per channel, each with a decay of its own.

    y = state_space_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus=True)                             # a prompt, or training
    y, state = state_space_scan(x, dt, A, B, C, D, z, dt_bias, True, initial=state, return_state=True)   # what follows it

    delta[t] = softplus(dt[t] + dt_bias)          (dt[t] + dt_bias without ``dt_softplus``)
    h[t][n]  = exp(delta[t] A[n]) h[t-1][n] + delta[t] x[t] B[t][n]
    y[t]     = (sum_n C[t][n] h[t][n] + D x[t]) * silu(z[t])

x, dt, z: [batch, S, channels]; B, C: [batch, S, N] or, with the channels in G groups, [batch, S, G, N]; float32 / float16 /
bfloat16, one type, the last dimension(s) contiguous, any strides between positions and batch entries.  A: [channels, N],
D, dt_bias: [channels], float32; N <= 64.  D, z and dt_bias may be None.  y has x's type; everything inside is float32.

``initial`` ([batch, channels, N] float32) continues an earlier call, ``return_state`` gives the state behind this one, and
``state_out`` names the tensor it is written to, which may be ``initial`` itself (a decoding loop in a CUDA graph keeps one
buffer).  Up to 8 positions take a kernel for decoding, as ``mlstm_chunkwise`` does for its mixer.  A position with delta = 0
(dt = -inf with ``dt_softplus``) and finite values in its other inputs leaves the state as it is and gets gradients of 0 for dt
and B: so a batch of different lengths is padded, on either side.

Inputs that require gradients get them (no states in that case): the forward then keeps the state in front of every 16
positions (N / 16 float32 values per element of x) and the backward recomputes what lies between.
The reference has no such operator; its own mixer with the same interface to states is ``mlstm_scan``.
"""
import ctypes

import torch

from . import _lib

__all__ = ["state_space_scan", "state_space_scan_forward", "state_space_scan_backward"]

_Strides = ctypes.c_longlong * 10


def _row_strides(t, name):
    s = t.stride()
    if s[2] != 1 and t.shape[2] != 1:
        raise RuntimeError(f"the last dimension of {name} must be contiguous")
    return s[0], s[1]


def _vector_strides(t, name):
    s = t.stride()
    n = t.shape[-1]
    if (s[-1] != 1 and n != 1) or (t.dim() == 4 and s[2] != n and t.shape[2] != 1):
        raise RuntimeError(f"a position's vectors in {name} must be contiguous")
    return s[0], s[1]


def _check(x, dt, A, B, C, D, z, dt_bias):
    """(device, strides or None where everything is contiguous, (batch, S, channels, G, N))"""
    shape = x.shape
    if len(shape) != 3 or not x.numel():
        raise ValueError("x must have the shape [batch, S, channels] with at least one of each")
    if dt.shape != shape or (z is not None and z.shape != shape):
        raise ValueError("x, dt and z must share the shape [batch, S, channels]")
    b, S, ch = shape
    if b > 65535 or S >= (1 << 31) - 32 or ch > 1 << 24:      # (before they become 32 bits)
        raise ValueError("x must have at most 65535 batch entries, 2^24 channels and fewer than 2^31 - 32 positions")
    vectors = B.shape
    if len(vectors) not in (3, 4) or C.shape != vectors or vectors[0] != b or vectors[1] != S:
        raise ValueError("B and C must share the shape [batch, S, N] or [batch, S, G, N]")
    G, N = (vectors[2] if len(vectors) == 4 else 1), vectors[-1]
    if G == 0 or ch % G:
        raise ValueError("the number of groups must divide the number of channels")
    if not 1 <= N <= 64:
        raise ValueError("N must be between 1 and 64")
    if A.shape != (ch, N):
        raise ValueError("A must have the shape [channels, N]")
    dtype = x.dtype
    if dt.dtype is not dtype or B.dtype is not dtype or C.dtype is not dtype or (z is not None and z.dtype is not dtype):
        raise TypeError("x, dt, B, C and z must share one element type")
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None:
            if t is not A and t.shape != (ch,):
                raise ValueError(f"{name} must have the shape [channels]")
            if t.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32")
            if not t.is_contiguous():
                raise RuntimeError(f"{name} must be contiguous")
    dev = _lib.require_one_cuda_device(x, dt, A, B, C, D, z, dt_bias)
    if x.is_contiguous() and dt.is_contiguous() and B.is_contiguous() and C.is_contiguous() and (z is None or z.is_contiguous()):
        return dev, None, (b, S, ch, G, N)
    strides = _Strides(*_row_strides(x, "x"), *_row_strides(dt, "dt"), *_vector_strides(B, "B"), *_vector_strides(C, "C"),
                       *((0, 0) if z is None else _row_strides(z, "z")))
    return dev, strides, (b, S, ch, G, N)


_STEP_TOKENS = None


def _step_tokens():
    global _STEP_TOKENS
    if _STEP_TOKENS is None:
        _STEP_TOKENS = _lib.lib().mlstm_ssm_step_max_tokens()
    return _STEP_TOKENS


def state_space_scan_forward(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial=None, state_out=None,
                             keep=False):
    """Run the forward; returns (y, checkpoints), with ``keep`` the states that the backward takes, else None."""
    return _forward(_check(x, dt, A, B, C, D, z, dt_bias), x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial, state_out, keep)


def _forward(checked, x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial=None, state_out=None, keep=False):
    dev, strides, dims = checked
    for name, t in (("initial", initial), ("state_out", state_out)):
        if t is not None and (t.shape != (dims[0], dims[2], dims[4]) or t.dtype != torch.float32 or not t.is_contiguous()
                              or t.device != dev):
            raise ValueError(f"{name} must be a contiguous float32 [batch, channels, N] tensor on x's device")
    L = _lib.lib()
    y = torch.empty_like(x) if strides is None else x.new_empty(x.shape)
    kept = torch.empty(L.mlstm_ssm_checkpoint_floats(*dims), dtype=torch.float32, device=dev) if keep else None
    # (a few tokens without anything to keep are a kernel that needs no scratch)
    ws, at, nbytes = _lib.scratch(0 if dims[1] <= _step_tokens() and not keep else L.mlstm_ssm_fwd_workspace(*dims), dev)
    with _lib.device_guard(dev):
        rc = L.mlstm_ssm_fwd(x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _lib.ptr(D), _lib.ptr(z), _lib.ptr(dt_bias),
                             _lib.ptr(initial), strides, y.data_ptr(), _lib.ptr(state_out), _lib.ptr(kept), at, nbytes, *dims,
                             _lib.dtype_code(x), 1 if dt_softplus else 0, _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_ssm_fwd")
    return y, kept


def state_space_scan_backward(dy, checkpoints, x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False):
    """Gradients (dx, ddt, dA, dB, dC, dD, dz, ddt_bias) of ``state_space_scan`` without states; None where the input is."""
    return _backward(_check(x, dt, A, B, C, D, z, dt_bias), dy, checkpoints, x, dt, A, B, C, D, z, dt_bias, dt_softplus)


def _backward(checked, dy, checkpoints, x, dt, A, B, C, D, z, dt_bias, dt_softplus):
    dev, strides, dims = checked
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy must match x in shape and element type")
    L = _lib.lib()
    if checkpoints.dtype != torch.float32 or checkpoints.numel() != L.mlstm_ssm_checkpoint_floats(*dims):
        raise ValueError("checkpoints must be what state_space_scan_forward(..., keep=True) gave for these inputs")
    _lib.require_cuda(dy, checkpoints, A)
    fresh = lambda t: None if t is None else torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)
    dx, ddt, dA, dB, dC, dD, dz, db = (fresh(t) for t in (x, dt, A, B, C, D, z, dt_bias))
    ws, at, nbytes = _lib.scratch(L.mlstm_ssm_bwd_workspace(*dims), dev)
    with _lib.device_guard(dev):
        rc = L.mlstm_ssm_bwd(dy.data_ptr(), x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _lib.ptr(D), _lib.ptr(z),
                             _lib.ptr(dt_bias), strides, checkpoints.data_ptr(), dx.data_ptr(), ddt.data_ptr(), dA.data_ptr(),
                             dB.data_ptr(), dC.data_ptr(), _lib.ptr(dD), _lib.ptr(dz), _lib.ptr(db), at, nbytes, *dims, _lib.dtype_code(x),
                             1 if dt_softplus else 0, _lib.stream_ptr(dev))
    _lib.check(rc, "mlstm_ssm_bwd")
    return dx, ddt, dA, dB, dC, dD, dz, db


class _StateSpaceScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, dt_softplus):
        y, kept = _forward(_check(x, dt, A, B, C, D, z, dt_bias), x, dt, A, B, C, D, z, dt_bias, dt_softplus, keep=True)
        ctx.save_for_backward(kept, x, dt, A, B, C, D, z, dt_bias)
        ctx.dt_softplus = dt_softplus
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        kept, *saved = ctx.saved_tensors    # (their strides may be others than the forward's: hooks may have moved them away and back)
        return _backward(_check(*saved), dy.contiguous(), kept, *saved, ctx.dt_softplus) + (None,)


def state_space_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial=None, return_state=False,
                     state_out=None):
    if torch.is_grad_enabled() and any([t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, initial) if t is not None]):
        if initial is not None or return_state or state_out is not None:
            raise ValueError("gradients are available for the plain call: no initial / return_state / state_out")
        return _StateSpaceScan.apply(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus))
    if not return_state:
        if state_out is not None:
            raise ValueError("state_out needs return_state")
        return state_space_scan_forward(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial)[0]
    checked = _check(x, dt, A, B, C, D, z, dt_bias)
    if state_out is None:
        state_out = (torch.empty_like(initial) if initial is not None and initial.is_contiguous()
                     else torch.empty((x.shape[0], x.shape[2], A.shape[1]), dtype=torch.float32, device=x.device))
    return _forward(checked, x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial, state_out)[0], state_out
