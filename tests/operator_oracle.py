"""The operators around the mixer in 64 bits on the CPU, straight from their definitions, for the parity tests."""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # of a value, relative to it


def conv(x, weight, bias=None, silu=False, initial=None):
    """(y, the last W - 1 inputs)"""
    x, weight = x.double(), weight.double()
    W, S = weight.shape[1], x.shape[1]
    before = x.new_zeros(x.shape[0], W - 1, x.shape[2]) if initial is None else initial.double()
    rows = torch.cat([before, x], 1)
    y = sum(rows[:, k:k + S] * weight[:, k] for k in range(W))
    if bias is not None:
        y = y + bias.double()
    return (y * torch.sigmoid(y) if silu else y), rows[:, S:]


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, initial=None):
    """(y, final state), position by position"""
    x, dt, A, B, C = (t.double() for t in (x, dt, A, B, C))
    b, S, ch = x.shape
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    B, C = (t.repeat_interleave(ch // t.shape[2], 2) for t in (B, C))
    delta = dt if dt_bias is None else dt + dt_bias.double()
    if softplus:
        delta = torch.logaddexp(delta, torch.zeros_like(delta))      # (its slope at 0 is 1/2, also by autograd)
    h = x.new_zeros(b, ch, A.shape[1]) if initial is None else initial.double()
    ys = []
    for t in range(S):
        d = delta[:, t, :, None]
        h = torch.exp(d * A) * h + d * x[:, t, :, None] * B[:, t]
        ys.append((h * C[:, t]).sum(-1))
    y = torch.stack(ys, 1)
    if D is not None:
        y = y + D.double() * x
    if z is not None:
        z = z.double()
        y = y * z * torch.sigmoid(z)
    return y, h


def norm(x, weight=None, residual=None, eps=1e-6):
    """(y, sum); the sum is rounded to the residual's type, as the operator says, and y is taken from it"""
    s = x.double()
    if residual is not None:
        total = s + residual.double()
        s = total + (total.detach().to(residual.dtype).double() - total.detach())
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        w = weight.double()
        y = y * (w if w.dim() == 1 else w[:, None])
    return y, s


def leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)
