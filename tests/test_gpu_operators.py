"""GPU parity of the operators around the mixer (short convolution, state space scan, residual norm) with their definitions in
64 bits.

Tolerances.  A result is off by half a step of its own type (operator_oracle.HALF_STEP, relative to the value) and by what fp32
arithmetic loses on the way.  The latter is bounded by a count of roundings times 2^-24 times the same formula with every term
taken in absolute value (``mag`` below), so that cancellation is accounted for."""
import importlib

import pytest
import torch

from tests import operator_oracle as oo

pytestmark = pytest.mark.gpu
PKG = "xlstm-triton-cuda-implementation_b200"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def pk():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return importlib.import_module(PKG)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def off(got, want, half, lost, what):
    """Every element: |got - want| <= half |want| + lost (both steps of the type's subnormals included)."""
    got = got.detach().cpu()
    tiny = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}.get(got.dtype, 0.0)
    g, w = got.double(), want.detach().double()
    lost = lost.detach().double() if isinstance(lost, torch.Tensor) else torch.full_like(w, lost)
    excess = (g - w).abs() - (half * (w.abs() + lost) + lost + tiny)
    assert torch.isfinite(g).all() and float(excess.max()) <= 0, (what, float((g - w).abs().max()), float(excess.max()))


# ---------------------------------------------------------------------------------------------- short convolution
def conv_inputs(dtype, B, S, C, W, bias, initial, seed, w32=False, wide=0):
    g = gen(seed)
    full = torch.randn(B, S, C + wide, generator=g).to(dtype)
    x = full[:, :, wide:] if wide else full
    wdt = F32 if w32 else dtype
    weight = (torch.randn(C, W, generator=g) * W ** -0.5).to(wdt)
    b = (0.5 * torch.randn(C, generator=g)).to(wdt) if bias else None
    init = torch.randn(B, W - 1, C, generator=g).to(dtype) if initial else None
    dy = torch.randn(B, S, C, generator=g).to(dtype)
    return x, weight, b, init, dy


def cu(t):
    """The tensor on the GPU with the strides it has here."""
    if t is None:
        return None
    if t.is_contiguous():
        return t.cuda()
    base = t._base
    return base.cuda().as_strided(t.shape, t.stride(), t.storage_offset())


CONV = [
    # dtype, B, S, C, W, bias, silu, initial, weight in fp32, columns of a wider tensor in front
    (BF16, 2, 1, 64, 4, True, True, True, False, 0),
    (BF16, 3, 2, 72, 4, True, True, True, False, 0),
    (F16, 1, 3, 8, 3, False, True, True, False, 0),
    (F32, 2, 5, 7, 2, True, False, False, False, 0),
    (F32, 1, 130, 36, 4, True, True, False, False, 0),
    (BF16, 2, 777, 200, 4, True, True, False, True, 0),
    (F16, 2, 333, 1, 4, True, True, True, True, 0),
    (BF16, 1, 1000, 129, 3, False, True, False, False, 0),
    (BF16, 2, 300, 128, 4, True, True, True, False, 8),      # a slice of a projection, aligned
    (BF16, 2, 300, 128, 4, True, False, False, False, 3),    # ... and not aligned
    (F32, 2, 70, 64, 2, True, True, True, False, 1),
]


@pytest.mark.parametrize("dtype,B,S,C,W,bias,silu,initial,w32,wide", CONV)
def test_convolution(pk, dtype, B, S, C, W, bias, silu, initial, w32, wide):
    x, weight, b, init, dy = conv_inputs(dtype, B, S, C, W, bias, initial, 7 * S + C, w32, wide)
    act = "silu" if silu else None
    y, state = pk.short_convolution(cu(x), cu(weight), cu(b), act, initial=cu(init), return_state=True)
    want, rows = oo.conv(x, weight, b, silu, init)
    assert y.dtype == dtype and y.is_contiguous()
    # W products and the bias, each a rounding of a partial sum; silu: an exponential and a division of a few units, at most
    # 1.1 times as steep as its argument
    mag = oo.conv(x.abs(), weight.abs(), None if b is None else b.abs(), False, None if init is None else init.abs())[0]
    off(y, want, oo.HALF_STEP[dtype], 1.1 * (W + 1) * U * mag + (16 * U * want.abs() if silu else 0), "y")
    assert torch.equal(state.cpu(), rows.to(dtype))


@pytest.mark.parametrize("dtype,B,S,C,W,bias,silu,initial,w32,wide", [c for c in CONV if not c[7]] + [
    (BF16, 2, 1, 64, 4, True, True, False, False, 0), (F16, 3, 2, 40, 4, True, True, False, False, 0),
    (BF16, 3, 600, 264, 4, True, True, False, False, 0)])
def test_convolution_gradients(pk, dtype, B, S, C, W, bias, silu, initial, w32, wide):
    x, weight, b, _, dy = conv_inputs(dtype, B, S, C, W, bias, False, 11 * S + C, w32, wide)
    leaves = [cu(t).requires_grad_(True) for t in (x, weight, b) if t is not None]
    y = pk.short_convolution(*leaves[:2], leaves[2] if bias else None, "silu" if silu else None)
    got = torch.autograd.grad(y, leaves, cu(dy))
    ref = [oo.leaf(t) for t in (x, weight, b) if t is not None]
    want = torch.autograd.grad(oo.conv(*ref[:2], ref[2] if bias else None, silu)[0], ref, dy.double())
    # d = dy act'(pre): |act'| <= 1.1, and its error is 1.1 |dy| times that of pre and a few units; then sums of W, resp. of
    # B S terms (a run of at most 32 by one thread, then in trees and short runs: fewer than 32 + 8 + 32 + B S / 256 in a row)
    pre = oo.conv(x.abs(), weight.abs(), None if b is None else b.abs())[0]
    d = 1.1 * dy.double().abs()
    loss = d * ((W + 1) * U * pre * (1.0 if silu else 0.0) + 16 * U)
    fold = lambda t: oo.conv(t.flip(1), weight.abs())[0].flip(1)
    xa = torch.cat([x.new_zeros(B, W - 1, C), x], 1).double().abs()
    n = (80 + B * S / 256) * U
    lost = [fold(loss) + W * U * fold(d),
            torch.stack([((loss + n * d) * xa[:, k:k + S]).sum((0, 1)) for k in range(W)], 1), (loss + n * d).sum((0, 1))]
    for name, gv, wv, lv in zip(("dx", "dweight", "dbias"), got, want, lost):
        off(gv, wv, oo.HALF_STEP[gv.dtype], lv, name)


def test_convolution_piece_by_piece(pk):
    """A prompt in pieces, then tokens, the state carried in one buffer: the same bits as in one call."""
    x, weight, b, init, _ = conv_inputs(BF16, 2, 50, 96, 4, True, True, 3)
    x, weight, b = cu(x), cu(weight), cu(b)
    whole, end = pk.short_convolution(x, weight, b, "silu", initial=cu(init), return_state=True)
    state, parts, at = cu(init), [], 0
    for n in (1, 1, 2, 30, 3, 1, 12):
        y, out = pk.short_convolution(x[:, at:at + n], weight, b, "silu", initial=state, return_state=True, state_out=state)
        assert out is state
        parts.append(y)
        at += n
    assert at == 50 and torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, end)


# ---------------------------------------------------------------------------------------------- state space scan
def scan_inputs(dtype, b, S, ch, N, G, seed, softplus=True, skip=True, gated=True, bias=True, initial=False, wide=0):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    fat = lambda: r(b, S, ch + wide).to(dtype)[:, :, wide:] if wide else r(b, S, ch).to(dtype)
    x, dt = fat(), (fat() if softplus else (0.02 + 0.1 * torch.rand(b, S, ch, generator=g)).to(dtype))
    A = -torch.exp(r(ch, N))
    B, C = (r(b, S, G, N).to(dtype) for _ in range(2))
    if G == 1:
        B, C = B[:, :, 0], C[:, :, 0]
    return dict(x=x, dt=dt, A=A, B=B, C=C, D=r(ch) if skip else None, z=fat() if gated else None,
                dt_bias=(r(ch) - 2.0) if bias else None, initial=r(b, ch, N) if initial else None), softplus


def scan_mag(a, softplus):
    """The formula with every term in absolute value (the decays as they are)."""
    m = {k: (v if v is None or k in ("dt", "A", "dt_bias", "z") else v.abs()) for k, v in a.items()}
    z = m.pop("z")
    y, h = oo.scan(**m, softplus=softplus)
    return (y if z is None else y * (z.double() * torch.sigmoid(z.double())).abs()), h


def scan_loss(S, N):
    """Roundings: a decay is off by 2^-22 (the hardware's exponential) and its exponent's two roundings (at most 2^-24 of
    itself after the exponential each), a product of up to S of them by as often; delta by some 2^-21 (softplus), its product with
    x and B by two more, the sum over N states by N, D x, the gate by 16."""
    return (S * 6 + N + 48) * U


SCAN = [
    # dtype, batch, S, channels, N, G, softplus, skip, gated, bias, initial, columns of a wider tensor in front
    (BF16, 2, 1, 64, 16, 1, True, True, True, True, True, 0),
    (F32, 1, 1, 3, 5, 1, True, True, True, True, True, 0),
    (F16, 3, 5, 24, 4, 2, True, False, True, True, True, 0),
    (F32, 2, 8, 65, 64, 1, False, True, False, False, True, 0),
    (BF16, 2, 7, 33, 33, 1, True, True, True, True, False, 1),
    (F32, 2, 9, 64, 16, 1, True, True, True, True, True, 0),
    (BF16, 1, 100, 128, 16, 1, True, True, True, True, True, 0),
    (F16, 2, 130, 96, 8, 2, True, True, True, True, True, 0),       # 48 channels in each group
    (F32, 1, 67, 63, 24, 3, True, True, True, True, True, 0),       # 21 channels in each group: nothing is aligned for pairs
    (BF16, 2, 300, 130, 1, 1, True, True, True, True, True, 3),
    (F32, 1, 257, 66, 32, 1, False, False, False, False, False, 2),
    (BF16, 1, 97, 64, 64, 1, True, True, True, True, True, 0),
    (BF16, 1, 1500, 70, 16, 1, True, True, True, True, True, 0),    # cut into segments
    (F32, 1, 1111, 40, 50, 2, True, True, True, True, True, 0),
    (BF16, 2, 90, 128, 24, 1, True, True, True, True, False, 0),    # 24 and 48 states, and numbers next to them
    (F32, 1, 70, 66, 17, 1, True, True, True, True, False, 0),
    (F16, 1, 1300, 64, 23, 2, True, True, True, True, False, 0),
    (BF16, 1, 61, 65, 25, 1, True, True, True, True, False, 0),
    (F32, 2, 66, 64, 48, 1, True, True, True, True, False, 0),
    (BF16, 1, 1400, 64, 40, 1, True, True, True, True, False, 0),
    (F16, 1, 40, 62, 49, 1, True, True, False, True, False, 0),
]


def on_gpu(a):
    return {k: cu(v) for k, v in a.items()}


@pytest.mark.parametrize("dtype,b,S,ch,N,G,softplus,skip,gated,bias,initial,wide", SCAN)
def test_scan(pk, dtype, b, S, ch, N, G, softplus, skip, gated, bias, initial, wide):
    a, sp = scan_inputs(dtype, b, S, ch, N, G, S + ch + N, softplus, skip, gated, bias, initial, wide)
    y, state = pk.state_space_scan(**on_gpu(a), dt_softplus=sp, return_state=True)
    want, end = oo.scan(**a, softplus=sp)
    ym, hm = scan_mag(a, sp)
    assert y.dtype == dtype and state.dtype == F32
    off(state, end, oo.HALF_STEP[F32], scan_loss(S, N) * hm, "state")
    off(y, want, oo.HALF_STEP[dtype], scan_loss(S, N) * ym, "y")


GRADS = [c for c in SCAN if not c[10]] + [
    (BF16, 2, 1, 64, 16, 1, True, True, True, True, False, 0),
    (F16, 3, 5, 24, 4, 2, True, False, True, True, False, 0),
    (F32, 2, 9, 64, 16, 1, True, True, False, True, False, 0),
    (BF16, 2, 100, 128, 16, 1, True, True, True, True, False, 0),
    (F32, 1, 67, 63, 24, 3, True, True, True, True, False, 0),
    (F16, 2, 130, 96, 8, 2, True, True, True, True, False, 0),
    (BF16, 1, 97, 64, 64, 1, True, True, True, True, False, 0),
    (BF16, 1, 1500, 70, 16, 1, True, True, True, True, False, 0),
    (F32, 1, 1111, 40, 50, 2, True, True, True, True, False, 0),
    (F32, 3, 64, 130, 2, 1, False, True, True, False, False, 0),
]
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


@pytest.mark.parametrize("dtype,b,S,ch,N,G,softplus,skip,gated,bias,initial,wide", GRADS)
def test_scan_gradients(pk, dtype, b, S, ch, N, G, softplus, skip, gated, bias, initial, wide):
    a, sp = scan_inputs(dtype, b, S, ch, N, G, 2 * S + ch + N, softplus, skip, gated, bias, False, wide)
    dy = torch.randn(b, S, ch, generator=gen(S)).to(dtype)
    names = [n for n in NAMES if a[n] is not None]
    d = {k: None if v is None else v.requires_grad_(True) for k, v in on_gpu(a).items() if k != "initial"}
    y = pk.state_space_scan(**d, dt_softplus=sp)
    got = torch.autograd.grad(y, [d[n] for n in names], cu(dy))
    ref = {k: oo.leaf(v) for k, v in a.items() if k != "initial"}
    want = torch.autograd.grad(oo.scan(**ref, softplus=sp)[0], [ref[n] for n in names], dy.double())
    mag = gradient_mag(a, dy, sp)
    # the forward's count for the states and once more on the way back; then sums over positions and batch (at most
    # S + b segments in a row), over the channels (a tree, then ch / 64 CTAs) or over the states
    loss = 2 * scan_loss(S, N) + (2 * S + b + ch / 64 + 64) * U
    for n, gv, wv in zip(names, got, want):
        assert gv.dtype == a[n].dtype and gv.shape == a[n].shape
        off(gv, wv, oo.HALF_STEP[gv.dtype], loss * mag[n], "d" + n)


def test_scan_gradients_where_softplus_bends(pk):
    """dt of exactly 0 of either sign (slope 1/2), far out on both sides, and of -inf (slope 0)."""
    a, _ = scan_inputs(F32, 2, 50, 70, 8, 1, 21, bias=False)
    for at, v in ((0, 0.0), (7, -0.0), (16, 40.0), (17, -40.0), (30, -200.0), (49, -float("inf"))):
        a["dt"][:, at] = v
    dy = torch.randn(2, 50, 70, generator=gen(22))
    names = [n for n in NAMES if a[n] is not None]
    d = {k: None if v is None else v.requires_grad_(True) for k, v in on_gpu(a).items() if k != "initial"}
    got = torch.autograd.grad(pk.state_space_scan(**d, dt_softplus=True), [d[n] for n in names], dy.cuda())
    ref = {k: oo.leaf(v) for k, v in a.items() if k != "initial"}
    want = torch.autograd.grad(oo.scan(**ref, softplus=True)[0], [ref[n] for n in names], dy.double())
    mag = gradient_mag(a, dy, True)
    for n, gv, wv in zip(names, got, want):
        off(gv, wv, U, (2 * scan_loss(50, 8) + (2 * 50 + 2 + 70 / 64 + 64) * U) * mag[n], "d" + n)


def gradient_mag(a, dy, softplus):
    """Every gradient's formula with all of its terms in absolute value."""
    a = {k: (None if v is None else v.detach().double()) for k, v in a.items()}
    b, S, ch = a["x"].shape
    G = a["B"].shape[2] if a["B"].dim() == 4 else 1
    Bv, Cv = (t.reshape(b, S, G, -1).repeat_interleave(ch // G, 2).abs() for t in (a["B"], a["C"]))
    raw = a["dt"] if a["dt_bias"] is None else a["dt"] + a["dt_bias"]
    delta = torch.nn.functional.softplus(raw, threshold=700.0) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    keep = torch.exp(delta[..., None] * a["A"])
    x, e, d = a["x"].abs(), dy.double().abs(), delta.abs()
    gate = torch.ones_like(x) if a["z"] is None else (a["z"] * torch.sigmoid(a["z"])).abs()
    D = torch.zeros(ch).double() if a["D"] is None else a["D"].abs()
    hs, h = [], torch.zeros(b, ch, keep.shape[-1]).double()
    before = []
    for t in range(S):
        before.append(keep[:, t] * h)
        h = before[-1] + (d[:, t] * x[:, t])[..., None] * Bv[:, t]
        hs.append(h)
    h, u = torch.stack(hs, 1), torch.stack(before, 1)
    y = (h * Cv).sum(-1) + D * x
    eg = e * gate
    g, carry = [None] * S, torch.zeros_like(h[:, 0])
    for t in reversed(range(S)):
        g[t] = eg[:, t, :, None] * Cv[:, t] + carry
        carry = keep[:, t] * g[t]
    g = torch.stack(g, 1)
    into = (g * Bv).sum(-1)
    dd = (x * into + (g * u * a["A"].abs()).sum(-1)) * slope
    group = lambda t: t.reshape(b, S, G, ch // G, -1).sum(3).reshape(a["B"].shape)
    return dict(x=d * into + D * eg, dt=dd, A=(g * u * d[..., None]).sum((0, 1)), B=group(g * (d * x)[..., None]),
                C=group(h * eg[..., None]), D=(eg * x).sum((0, 1)), z=1.1 * e * y, dt_bias=dd.sum((0, 1)))


def test_scan_gradients_against_differences(pk):
    """A step along a random direction of all inputs at once: the change of <dy, y> in fp32 against <gradient, direction>."""
    a, sp = scan_inputs(F32, 2, 40, 70, 16, 1, 5)
    d = {k: cu(v) for k, v in a.items() if v is not None}
    dy = torch.randn(2, 40, 70, generator=gen(1)).cuda()
    for t in d.values():
        t.requires_grad_(True)
    grads = torch.autograd.grad(pk.state_space_scan(**d, dt_softplus=True), list(d.values()), dy)
    step, g = 2.0 ** -8, gen(2)
    dirs = {k: torch.randn(v.shape, generator=g).cuda() for k, v in d.items()}
    with torch.no_grad():
        at = lambda s: (pk.state_space_scan(**{k: v + s * dirs[k] for k, v in d.items()}, dt_softplus=True).double() * dy).sum()
        slope = (at(step) - at(-step)) / (2 * step)
        want = sum((gv.double() * dirs[k]).sum() for k, gv in zip(d, grads))
        size = sum((gv.double() * dirs[k]).abs().sum() for k, gv in zip(d, grads)) ** 0.5
    # the third derivative's part is step^2 of the slope's terms; the roundings of y are 2^-20 of it over the step
    assert abs(float(slope - want)) <= 0.02 * (abs(float(want)) + float(size)), (float(slope), float(want))


def test_scan_piece_by_piece(pk):
    """Pieces of a prompt and single tokens behind it, the state in one buffer, against the definition of the whole."""
    a, sp = scan_inputs(BF16, 2, 141, 130, 16, 1, 6, initial=True)
    d = on_gpu(a)
    state, parts, at = d["initial"].clone(), [], 0
    for n in (1, 30, 8, 2, 99, 1):
        cut = {k: (v[:, at:at + n] if k in ("x", "dt", "B", "C", "z") else v) for k, v in d.items() if k != "initial"}
        y, out = pk.state_space_scan(**cut, dt_softplus=sp, initial=state, return_state=True, state_out=state)
        assert out is state
        parts.append(y)
        at += n
    want, end = oo.scan(**a, softplus=sp)
    ym, hm = scan_mag(a, sp)
    off(state, end, U, scan_loss(141, 16) * hm, "state")
    off(torch.cat(parts, 1), want, oo.HALF_STEP[BF16], scan_loss(141, 16) * ym, "y")


def test_scan_state_in_place_when_cut_into_segments(pk):
    a, sp = scan_inputs(BF16, 1, 2000, 64, 16, 1, 8, initial=True)
    d = on_gpu(a)
    y0, s0 = pk.state_space_scan(**d, dt_softplus=sp, return_state=True)
    for _ in range(3):
        state = d["initial"].clone()
        y1, _ = pk.state_space_scan(**{**d, "initial": state}, dt_softplus=sp, return_state=True, state_out=state)
        assert torch.equal(y0, y1) and torch.equal(s0, state)


@pytest.mark.parametrize("S", [5, 40, 1500])
def test_scan_steps_of_zero_leave_the_state(pk, S):
    """Left padding: delta = 0 passes the state on unchanged, also behind decays of -inf."""
    a, _ = scan_inputs(F32, 2, S, 64, 16, 1, 9, softplus=False, bias=False, initial=True)
    a["dt"].zero_()
    a["A"][3, 2] = -float("inf")
    y, state = pk.state_space_scan(**on_gpu(a), return_state=True)
    assert torch.equal(state.cpu(), a["initial"]) and bool(torch.isfinite(y).all())


@pytest.mark.parametrize("S", [4, 200])
def test_scan_keeps_bad_values_where_they_are(pk, S):
    """A NaN or an infinity in one channel at one position: no other channel and no earlier position changes."""
    a, sp = scan_inputs(F32, 2, S, 70, 13, 1, 10, initial=True)
    clean, _ = pk.state_space_scan(**on_gpu(a), dt_softplus=sp, return_state=True)
    t = S // 2
    a["x"][1, t, 5] = float("inf")
    a["x"][0, t, 64] = float("nan")
    y, state = pk.state_space_scan(**on_gpu(a), dt_softplus=sp, return_state=True)
    bad = torch.zeros(2, S, 70, dtype=torch.bool)
    bad[1, t:, 5] = True
    bad[0, t:, 64] = True
    y, clean = y.cpu(), clean.cpu()
    assert torch.equal(y[~bad], clean[~bad]) and not torch.isfinite(y[bad]).any()
    assert torch.isnan(state[0, 64]).all() and not torch.isfinite(state[1, 5]).any() and torch.isfinite(state[1, 6:]).all()


def test_scan_extremes(pk):
    """Steps so long that nothing is kept, growing states (A > 0), softplus far out on both sides."""
    a, _ = scan_inputs(F32, 1, 60, 64, 16, 1, 12, initial=True)
    a["dt"][0, :, 0] = 3.0e4
    a["dt"][0, :, 1] = -80.0
    a["dt_bias"][:2] = 0.0
    a["A"][2] = 0.0
    a["A"][3] = 0.01
    y, state = pk.state_space_scan(**on_gpu(a), dt_softplus=True, return_state=True)
    want, end = oo.scan(**a, softplus=True)
    ym, hm = scan_mag(a, True)
    off(state, end, U, scan_loss(60, 16) * hm, "state")
    off(y, want, U, scan_loss(60, 16) * ym, "y")


def test_scan_broadcast_inputs(pk):
    """Inputs that repeat along the batch or the positions (strides of 0) are read as they are; their gradients are sums."""
    a, sp = scan_inputs(F32, 1, 50, 64, 16, 1, 13)
    d = {k: v.cuda().requires_grad_(True) for k, v in a.items() if v is not None}
    wide = {k: v.expand(3, -1, -1) if k in ("x", "dt", "B", "C", "z") else v for k, v in d.items()}
    dy = torch.randn(3, 50, 64, generator=gen(14)).cuda()
    y = pk.state_space_scan(**wide, dt_softplus=sp)
    got = torch.autograd.grad(y, list(d.values()), dy)
    ref = {k: oo.leaf(v) for k, v in a.items() if v is not None}
    want = torch.autograd.grad(oo.scan(**ref, softplus=sp)[0], list(ref.values()), dy.cpu().double().sum(0, keepdim=True))
    mag = gradient_mag(a, dy.cpu().abs().sum(0, keepdim=True), sp)
    for n, gv, wv in zip(d, got, want):
        off(gv, wv, U, (2 * scan_loss(50, 16) + 300 * U) * mag[n], n)


# ---------------------------------------------------------------------------------------------- residual norm
NORM = [
    # dtype, residual type (None: none), weight: "x" of x's type, "f" float32, None; shape
    (BF16, BF16, "x", (5, 64)), (BF16, F32, "f", (3, 7, 200)), (F16, None, "x", (4, 257)), (F32, F32, "x", (2, 1)),
    (F32, None, None, (130, 36)), (BF16, BF16, "f", (9, 1000)), (F16, F16, "x", (3, 1024)), (BF16, None, "x", (2, 2048)),
    (BF16, BF16, "x", (700, 520)), (F32, F32, "f", (3, 4104)), (BF16, F32, "x", (2, 8200)), (F16, None, None, (2, 16384)),
    (F32, None, "x", (1, 16383)), (BF16, BF16, "x", (1, 5001)), (F32, F32, None, (3, 600)),
]


def norm_inputs(dtype, rdt, w, shape, seed):
    g = gen(seed)
    x = (torch.randn(*shape, generator=g) * 2).to(dtype)
    res = None if rdt is None else (torch.randn(*shape, generator=g) * 3).to(rdt)
    weight = None if w is None else (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(dtype if w == "x" else F32)
    return x, weight, res


@pytest.mark.parametrize("dtype,rdt,w,shape", NORM)
def test_norm(pk, dtype, rdt, w, shape):
    x, weight, res = norm_inputs(dtype, rdt, w, shape, sum(shape))
    got = pk.residual_rms_norm(cu(x), cu(weight), residual=cu(res))
    y, s = got if res is not None else (got, None)
    want, total = oo.norm(x, weight, res)
    if res is not None:
        assert s.dtype == rdt
        # x + residual in fp32, then to the stream's type: where that is no fp32 sum, to the nearest but for ties of the fp32 rounding
        off(s, x.double() + res.double(), oo.HALF_STEP[rdt], U * (x.double().abs() + res.double().abs()), "sum")
        want = oo.norm(s.cpu(), weight)[0]
    # the sum of squares: at most 32 in a row and a tree (relative 45 U, halved by the root), root and products
    off(y, want, oo.HALF_STEP[y.dtype], 32 * U * want.abs(), "y")


@pytest.mark.parametrize("dtype,rdt,w,shape", NORM)
def test_norm_gradients(pk, dtype, rdt, w, shape):
    x, weight, res = norm_inputs(dtype, rdt, w, shape, 3 + sum(shape))
    g = gen(4)
    dy = torch.randn(*shape, generator=g).to(dtype)
    leaves = [cu(t).requires_grad_(True) for t in (x, weight, res) if t is not None]
    args = iter(leaves)
    xs, ws, rs = (None if t is None else next(args) for t in (x, weight, res))
    out = pk.residual_rms_norm(xs, ws, residual=rs)
    ds = None if res is None else torch.randn(*shape, generator=g).to(rdt)
    got = list(torch.autograd.grad(out, leaves, (cu(dy), cu(ds)) if res is not None else cu(dy)))
    s = out[1].detach().cpu() if res is not None else x
    v, wl = oo.leaf(s), oo.leaf(weight)
    y = oo.norm(v, wl)[0]
    want = torch.autograd.grad(y, [v] + ([wl] if weight is not None else []), dy.double())
    dv = want[0] + (0 if ds is None else ds.double())
    r = 1 / torch.sqrt(v.detach().square().mean(-1, keepdim=True) + 1e-6)
    u = dy.double().abs() * (1.0 if weight is None else weight.double().abs())
    mag = r * (u + v.detach().abs() * r * r * (u * v.detach().abs()).mean(-1, keepdim=True)) + (0 if ds is None else ds.double().abs())
    off(got[0], dv, oo.HALF_STEP[x.dtype], 64 * U * mag, "dx")
    if weight is not None:
        rows = s.numel() // shape[-1]
        # a sum over the rows: at most rows / 148 + 40 and the blocks' partial sums (148 x 8 / 8 + 8) in a row
        lost = (rows / 100 + 300) * U * (dy.double() * v.detach() * r).abs().reshape(-1, shape[-1]).sum(0)
        off(got[1], want[1], oo.HALF_STEP[weight.dtype], lost, "dweight")
    if res is not None:
        off(got[-1], dv, oo.HALF_STEP[rdt], 64 * U * mag, "dresidual")


@pytest.mark.parametrize("B,NH,S,D,out", [(2, 4, 65, 64, BF16), (1, 8, 33, 128, F32), (3, 2, 7, 100, F16), (2, 3, 300, 256, BF16)])
def test_norm_of_every_head(pk, B, NH, S, D, out):
    """A mixer's float32 result, with a weight for every head, to 16 bits, and back."""
    g = gen(B + S)
    h, w, dy = torch.randn(B, NH, S, D, generator=g) * 5, 1 + 0.3 * torch.randn(NH, D, generator=g), torch.randn(B, NH, S, D, generator=g).to(out)
    hc, wc = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = pk.residual_rms_norm(hc, wc, out_dtype=out)
    assert y.dtype == out
    hl, wl = oo.leaf(h), oo.leaf(w)
    want = oo.norm(hl, wl)[0]
    off(y, want, oo.HALF_STEP[out], 32 * U * want.abs(), "y")
    got, ref = torch.autograd.grad(y, (hc, wc), dy.cuda()), torch.autograd.grad(want, (hl, wl), dy.double())
    r = 1 / torch.sqrt(hl.detach().square().mean(-1, keepdim=True) + 1e-6)
    u = dy.double().abs() * wl.detach().abs()[:, None]
    mag = r * (u + hl.detach().abs() * r * r * (u * hl.detach().abs()).mean(-1, keepdim=True))
    off(got[0], ref[0], U, 64 * U * mag, "dx")
    off(got[1], ref[1], U, (B * S + 300) * U * (dy.double() * hl.detach() * r).abs().sum((0, 2)), "dweight")


def test_norm_gradient_of_the_sum_alone(pk):
    """Only the stream is used further, or only the norm."""
    x, weight, res = norm_inputs(BF16, F32, "x", (6, 96), 1)
    xs, ws, rs = (cu(t).requires_grad_(True) for t in (x, weight, res))
    _, s = pk.residual_rms_norm(xs, ws, residual=rs)
    ds = torch.randn(6, 96, generator=gen(2))
    gx, gr = torch.autograd.grad(s, (xs, rs), ds.cuda())
    assert torch.equal(gr.cpu(), ds) and torch.equal(gx.cpu(), ds.to(BF16))
    y, _ = pk.residual_rms_norm(xs, ws, residual=rs)
    got = torch.autograd.grad(y, (rs,), cu(x))[0]
    y2, s2 = pk.residual_rms_norm(xs, ws, residual=rs)
    zero = torch.autograd.grad((y2, s2), (rs,), (cu(x), torch.zeros(6, 96).cuda()))[0]
    assert torch.equal(got, zero)


@pytest.mark.parametrize("dtype,rdt,shape,block", [
    (BF16, BF16, (9, 256), 128), (BF16, None, (3, 5, 4096), 128), (F16, F32, (4, 1056), 32), (F32, None, (130, 64), 64),
    (BF16, BF16, (7, 1000), None), (F32, F32, (3, 257), None), (BF16, None, (2, 16384), 128), (F32, None, (2, 8224), 32),
    (BF16, F32, (5, 192), None), (F16, None, (2, 16384), None), (F32, F32, (3, 96), 32), (BF16, BF16, (2, 5001), None)])
def test_quantized_norm(pk, dtype, rdt, shape, block):
    x, weight, res = norm_inputs(dtype, rdt, "x", shape, 5 + sum(shape))
    x.view(-1, shape[-1])[0] = 0
    if res is not None:
        res.view(-1, shape[-1])[0] = 0          # a row of zeros
    got = pk.residual_rms_norm_quantized(cu(x), cu(weight), residual=cu(res), block=block)
    q, scale = got[:2]
    n = block or shape[-1]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == x.shape[:-1] + (shape[-1] // n,)
    s = x if res is None else got[2].cpu()
    want = oo.norm(s, weight)[0].reshape(-1, shape[-1] // n, n)
    top = want.abs().amax(-1)
    ws = torch.where(top > 0, top / 448, torch.ones_like(top))
    off(scale.reshape(-1, shape[-1] // n), ws, U, 40 * U * ws, "scale")
    assert float(scale.reshape(-1, shape[-1] // n)[0, 0]) == 1.0 and not q.reshape(-1, shape[-1])[0].float().any()
    value = q.cpu().double().reshape(want.shape) * scale.cpu().double().reshape(want.shape[:2])[..., None]
    # half a step of 3 bits of mantissa, 2^-4 of the value, or of the subnormal steps of 2^-9 (scaled); what the scale is off
    assert bool(((value - want).abs() <= 2.0 ** -4 * want.abs() * (1 + 1e-4) + (2.0 ** -10 * ws)[..., None] * (1 + 1e-4) + 80 * U * want.abs()).all())


def test_quantized_norm_of_bad_values(pk):
    """An infinity or a NaN spoils its row, and no other."""
    x = torch.randn(4, 256, generator=gen(1))
    clean = pk.residual_rms_norm_quantized(x.cuda(), block=64)
    x[1, 70] = float("nan")
    x[2, 3] = float("inf")
    q, scale = pk.residual_rms_norm_quantized(x.cuda(), block=64)
    for row in (0, 3):
        assert torch.equal(q[row].float(), clean[0][row].float()) and torch.equal(scale[row], clean[1][row])
    assert torch.isnan(q[1].float()).all() and torch.isnan(scale[1]).all()
    assert torch.isnan(scale[2, 0]) and torch.isnan(q[2, 3].float())


# ---------------------------------------------------------------------------------------------- together
def block(pk, x, stream, p, states=None):
    """One layer around the scan as a user writes it: sum and norm, projection, convolution, scan, projection."""
    y, stream = pk.residual_rms_norm(x, p["norm"], residual=stream)
    u, z = (y @ p["into"]).chunk(2, -1)
    plain = states is None
    if plain:
        u = pk.short_convolution(u, p["conv"], p["conv_bias"], "silu")
    else:
        u, _ = pk.short_convolution(u, p["conv"], p["conv_bias"], "silu", initial=states[0], return_state=True, state_out=states[0])
    dt, B, C = (u @ p["select"]).split([u.shape[-1], 16, 16], -1)
    args = (u, dt, p["A"], B, C, p["D"], z, p["dt_bias"], True)
    if plain:
        y = pk.state_space_scan(*args)
    else:
        y, _ = pk.state_space_scan(*args, initial=states[1], return_state=True, state_out=states[1])
    return y @ p["out"], stream


def block_parameters(D, E, dtype, seed):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    p = dict(norm=1 + 0.1 * r(D), into=r(D, 2 * E) * D ** -0.5, conv=r(E, 4) * 0.5, conv_bias=0.1 * r(E),
             select=r(E, E + 32) * E ** -0.5, out=r(E, D) * E ** -0.5)
    p = {k: v.to(dtype).cuda() for k, v in p.items()}
    return dict(p, A=-torch.exp(r(E, 16)).cuda(), D=r(E).cuda(), dt_bias=(r(E) - 2).cuda())


def test_layer_prompt_then_tokens_equals_the_whole(pk):
    """The layer over a whole sequence against the same sequence as a prompt and tokens, in a captured graph, behind it."""
    D, E, S, P, n = 64, 128, 45, 32, 2
    p = block_parameters(D, E, F32, 1)
    x, stream = (torch.randn(n, S, D, generator=gen(k)).cuda() for k in (2, 3))
    want, _ = block(pk, x, stream, p)
    states = [torch.zeros(n, 3, E).cuda(), torch.zeros(n, E, 16).cuda()]
    got = [block(pk, x[:, :P].contiguous(), stream[:, :P].contiguous(), p, states)[0]]
    xs, ss = torch.zeros(n, 1, D).cuda(), torch.zeros(n, 1, D).cuda()
    keep = [t.clone() for t in states]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block(pk, xs, ss, p, states)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = block(pk, xs, ss, p, states)
    for t, k in zip(states, keep):
        t.copy_(k)
    for t in range(P, S):
        xs.copy_(x[:, t:t + 1])
        ss.copy_(stream[:, t:t + 1])
        graph.replay()
        got.append(out.clone())
    got = torch.cat(got, 1)
    # the projections are library products whose order of summing differs with the number of rows: fp32, a few hundred terms
    torch.testing.assert_close(got, want, rtol=2e-3, atol=2e-3)


def test_layer_gradients_in_a_captured_step(pk):
    """Forward and backward of the layer captured into a graph and replayed on new inputs: the bits of the eager step."""
    D, E = 64, 96
    p = block_parameters(D, E, BF16, 4)
    for t in p.values():
        t.requires_grad_(True)
    x, stream = torch.zeros(2, 70, D, dtype=BF16).cuda(), torch.zeros(2, 70, D, dtype=BF16).cuda()

    def step():
        y, s = block(pk, x, stream, p)
        return torch.autograd.grad((y.float().square().sum() + s.float().square().sum()), list(p.values()))
    fill = lambda k: (x.copy_(torch.randn(2, 70, D, generator=gen(k)).to(BF16)), stream.copy_(torch.randn(2, 70, D, generator=gen(k + 1)).to(BF16)))
    fill(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for k in (5, 9):
        fill(k)
        graph.replay()
        got = [t.clone() for t in kept]
        for a, b in zip(got, step()):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_two_streams_at_once(pk):
    """The same calls on two streams at the same time: each gets its own scratch."""
    a, sp = scan_inputs(BF16, 1, 3000, 64, 16, 1, 20)
    d = {k: v.cuda().requires_grad_(True) for k, v in a.items() if v is not None}
    dy = torch.randn(1, 3000, 64, generator=gen(1)).to(BF16).cuda()
    step = lambda scale: torch.autograd.grad(pk.state_space_scan(**{**d, "x": d["x"] * scale}, dt_softplus=True), list(d.values()), dy)
    want = [step(1.0), step(2.0)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = step(1.0 + i)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for u, v in zip(g, w):
            assert torch.equal(u, v)


def test_same_call_same_bits(pk):
    x, weight, res = norm_inputs(BF16, BF16, "x", (5000, 512), 1)
    xs, ws, rs = (cu(t).requires_grad_(True) for t in (x, weight, res))
    runs = [torch.autograd.grad(pk.residual_rms_norm(xs, ws, residual=rs)[0], (xs, ws, rs), cu(x)) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ---------------------------------------------------------------------------------------------- places and sizes off the beaten track
def shifted(t, by=1):
    """The same values, contiguous, ``by`` elements off the start of their memory."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
    flat[by:] = t.reshape(-1).cuda()
    return flat[by:].view(t.shape)


def test_unaligned_tensors_give_the_same(pk):
    """Contiguous views into flat buffers, off by one element: the slower accesses, the same arithmetic, so the same bits (for
    the norm, whose rows are summed in another order, the same to a few roundings)."""
    x, w, b, init, dy = conv_inputs(BF16, 2, 70, 96, 4, True, True, 1)
    for make in (cu, shifted):
        t = [make(v).requires_grad_(True) for v in (x, w, b)]
        y, s = (v.detach() for v in pk.short_convolution(*(v.detach() for v in t), "silu", initial=make(init), return_state=True))
        g = torch.autograd.grad(pk.short_convolution(*t, "silu"), t, make(dy))
        if make is cu:
            want = (y, s, g[0])
        else:
            assert all(torch.equal(u, v) for u, v in zip((y, s, g[0]), want))
    a, sp = scan_inputs(BF16, 2, 40, 64, 16, 1, 2, initial=True)
    for S in (40, 3):
        cut = {k: (v[:, :S].contiguous() if k in ("x", "dt", "B", "C", "z") else v) for k, v in a.items()}
        one = pk.state_space_scan(**on_gpu(cut), dt_softplus=sp, return_state=True)
        two = pk.state_space_scan(**{k: shifted(v) for k, v in cut.items()}, dt_softplus=sp, return_state=True)
        assert all(torch.equal(u, v) for u, v in zip(one, two))
    x, w, r = norm_inputs(BF16, BF16, "x", (9, 256), 3)
    (y0, s0), (y1, s1) = pk.residual_rms_norm(cu(x), cu(w), residual=cu(r)), pk.residual_rms_norm(shifted(x), shifted(w), residual=shifted(r))
    assert torch.equal(s0, s1)
    off(y1, oo.norm(s0.cpu(), w)[0], oo.HALF_STEP[BF16], 32 * U * y0.cpu().double().abs(), "y")


@pytest.mark.parametrize("S", [6, 90])
def test_scan_padding(pk, S):
    """dt = -inf behind a softplus, in front of, between and behind the tokens: what is left is the sequence without those
    positions, and they get gradients of 0."""
    a, _ = scan_inputs(F32, 1, S, 64, 16, 1, 21, initial=True)
    keep = torch.rand(S, generator=gen(3)) < 0.6
    keep[0] = keep[-1] = False
    a["dt"][:, ~keep] = -float("inf")
    y, state = pk.state_space_scan(**on_gpu(a), dt_softplus=True, return_state=True)
    short = {k: (v[:, keep] if k in ("x", "dt", "B", "C", "z") else v) for k, v in a.items()}
    want, end = oo.scan(**short, softplus=True)
    ym, hm = scan_mag(short, True)
    off(state, end, U, scan_loss(S, 16) * hm, "state")
    off(y[:, keep.cuda()], want, U, scan_loss(S, 16) * ym, "y")
    d = {k: cu(v).requires_grad_(True) for k, v in a.items() if k != "initial"}
    got = dict(zip(d, torch.autograd.grad(pk.state_space_scan(**d, dt_softplus=True).square().sum(), list(d.values()))))
    assert all(bool(torch.isfinite(g).all()) for g in got.values())
    assert not got["dt"][:, ~keep.cuda()].any() and not got["B"][:, ~keep.cuda()].any()


def test_saved_tensors_that_come_back_with_other_strides(pk):
    """Hooks that move what the backward needs to the host and back (contiguous then, where slices were saved)."""
    wide = torch.randn(2, 30, 192, generator=gen(1)).to(BF16).cuda().requires_grad_(True)
    w = (torch.randn(64, 4, generator=gen(2)) * 0.5).to(BF16).cuda().requires_grad_(True)
    a, sp = scan_inputs(BF16, 2, 30, 64, 16, 1, 4, gated=False)
    rest = {k: cu(v) for k, v in a.items() if k not in ("x", "z", "dt") and v is not None}

    def step():
        x, dt, z = wide.split(64, -1)
        x = pk.short_convolution(x, w, None, "silu")
        y = pk.state_space_scan(x, dt, z=z, dt_softplus=sp, **rest)
        y = pk.residual_rms_norm(y, w[:, 0].contiguous())
        return torch.autograd.grad(y.float().square().sum() + x.float().sum(), (wide, w))
    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_scan_gradients_in_groups_of_batch_entries(pk):
    """More partial sums of dB, dC than are held at one time: the last group is what its batch entries give alone."""
    b, S, ch, N = 34, 1024, 2048, 64
    assert pk._lib.lib().mlstm_ssm_bwd_workspace(b, S, ch, 1, N) < b * (ch // 64) * S * N * 8
    g = torch.Generator("cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, dt, z, dy = (r(b, S, ch).to(BF16) for _ in range(4))
    B, C = (r(b, S, N).to(BF16) for _ in range(2))
    A, D, bias = -torch.exp(r(ch, N)), r(ch), r(ch) - 2

    def run(k):
        y, kept = pk.state_space_scan_forward(x[-k:], dt[-k:], A, B[-k:], C[-k:], D, z[-k:], bias, True, keep=True)
        got = pk.state_space_scan_backward(dy[-k:], kept, x[-k:], dt[-k:], A, B[-k:], C[-k:], D, z[-k:], bias, True)
        return [y] + [got[i] for i in (0, 1, 3, 4, 6)]
    for u, v in zip(run(b), run(8)):
        assert torch.equal(u[-8:], v)


def test_offsets_beyond_32_bits(pk):
    """More than 2^31 values in a tensor: the last channels at the last positions are what they are alone."""
    g = torch.Generator("cuda").manual_seed(7)
    B, S, C = 2, 16640, 64640          # 2.15e9 values
    assert B * S * C > 2 ** 31
    x = torch.empty(B, S, C, dtype=BF16, device="cuda").normal_(generator=g)
    w = (torch.randn(C, 4, device="cuda", generator=g) * 0.5).to(BF16)
    y = pk.short_convolution(x, w, None, "silu")
    cut = slice(C - 64, C)
    assert torch.equal(y[:, :, cut], pk.short_convolution(x[:, :, cut], w[cut].contiguous(), None, "silu"))
    dx, _, _ = pk.short_convolution_backward(x, x, w, None, "silu")
    assert torch.equal(dx[:, :, cut], pk.short_convolution_backward(x[:, :, cut].contiguous(), x[:, :, cut], w[cut].contiguous(), None, "silu")[0])
    del dx
    A, bias = -torch.exp(torch.randn(C, 1, device="cuda", generator=g)), torch.full((C,), -2.0, device="cuda")
    Bv, Cv = (torch.randn(B, S, 1, device="cuda", generator=g).to(BF16) for _ in range(2))
    y, kept = pk.state_space_scan_forward(x, x, A, Bv, Cv, None, None, bias, True, keep=True)
    xs = x[:, :, cut].contiguous()
    ys, ks = pk.state_space_scan_forward(xs, xs, A[cut], Bv, Cv, None, None, bias[cut], True, keep=True)
    # (the narrow call is cut into segments, the wide one is not: the same sums in another order)
    torch.testing.assert_close(y[:, :, cut].float(), ys.float(), rtol=2 * 2.0 ** -8, atol=1e-3)
    got = pk.state_space_scan_backward(x, kept, x, x, A, Bv, Cv, None, None, bias, True)
    want = pk.state_space_scan_backward(xs, ks, xs, xs, A[cut], Bv, Cv, None, None, bias[cut], True)
    for k in (0, 1):
        torch.testing.assert_close(got[k][:, :, cut].float(), want[k].float(), rtol=2 * 2.0 ** -8, atol=2e-3)
    torch.testing.assert_close(got[2][cut], want[2], rtol=1e-3, atol=1e-2)
    del got, kept, y
    rows = x.view(-1, 8080)
    n = pk.residual_rms_norm(rows)
    assert torch.equal(n[-3:], pk.residual_rms_norm(rows[-3:].clone()))
    assert torch.equal(pk.residual_rms_norm_backward(rows, rows)[0][-3:], pk.residual_rms_norm_backward(rows[-3:].clone(), rows[-3:].clone())[0])


def test_library_refusals(pk):
    L, one = pk._lib.lib(), torch.zeros(64, device="cuda").data_ptr()
    assert L.mlstm_conv_fwd(one, one, None, None, None, one + 1, None, 1, 1, 8, 4, 2, 2, 1, None) == -3
    assert L.mlstm_ssm_fwd(one, one, one, one, one, None, None, None, None, None, one, None, None, None, 0, 1, 4096, 8, 1, 4, 2, 1, None) == -5
    assert L.mlstm_rms_bwd(one, None, one, one, one, None, one, None, 0, 1, 8, 1, 1, 1e-6, 0, 0, 0, 0, None) == -5


# ---------------------------------------------------------------------------------------------- 8 bits at the edges
def eight_bits(y, block):
    """(values, scales) of fp32 results by the definition; a quotient in fp32 is one in 64 bits, rounded (53 > 2 * 24 + 1)."""
    v = y.cpu().double().reshape(-1, y.shape[-1] // block, block)
    top = v.abs().amax(-1)
    exact = torch.where(top > 0, top / 448, torch.ones_like(top))
    scale = exact.float()
    up = (scale < 2.0 ** -126) & (scale.double() < exact)         # below the normal numbers: rounded up
    return v, torch.where(up, scale + 2.0 ** -149, scale)


def assert_eight_bits(q, scale, y, block):
    v, want = eight_bits(y, block)
    assert torch.equal(scale.cpu().reshape(want.shape), want)
    nearest = (v / want.double()[..., None]).float().to(torch.float8_e4m3fn).float()
    assert torch.equal(q.cpu().float().reshape(v.shape), nearest), int((q.cpu().float().reshape(v.shape) != nearest).sum())


@pytest.mark.parametrize("shape,block", [((300, 4096), 128), ((90, 2048), None), ((999, 256), 32), ((64, 8200), None),
                                         ((40, 777), None), ((3, 16384), 64)])
def test_quantized_norm_to_the_nearest(pk, shape, block):
    """Values of 16 bits, whose quotients by the scale lie on ties now and then: each goes where its quotient goes."""
    x = (torch.randn(*shape, generator=gen(shape[0])) * 2).to(BF16)
    res = torch.zeros(shape)
    y = pk.residual_rms_norm(x.float().cuda())
    for got in (pk.residual_rms_norm_quantized(x.cuda(), block=block), pk.residual_rms_norm_quantized(x.float().cuda(), block=block),
                pk.residual_rms_norm_quantized(x.cuda(), residual=res.cuda(), block=block)):
        assert_eight_bits(got[0], got[1], y, block or shape[-1])


@pytest.mark.parametrize("D,block", [(256, 64), (4096, 128), (96, None), (257, None)])
def test_quantized_norm_of_tiny_and_huge_values(pk, D, block):
    """Blocks whose largest magnitude has no finite reciprocal, or a scale below the normal numbers, beside ordinary ones."""
    x = torch.randn(8, D, generator=gen(D))
    x[0] *= 1e-40                        # (eps holds the root at 1e-3: results of 1e-37)
    x[1] *= 1e-43
    x[1, ::3] = 0
    x[2] = 0
    x[2, 5] = 2.0 ** -149                # the least of all numbers
    x[3, : D // 2] *= 1e-37
    x[4] = (x[4] * 3).round() * 2.0 ** -149
    x[5] *= 1e-30
    w = torch.ones(D)
    for weight in (w, w * 0.1, w * 2e37):
        y = pk.residual_rms_norm(x.cuda(), weight.cuda())
        q, scale = pk.residual_rms_norm_quantized(x.cuda(), weight.cuda(), block=block)
        assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(q.float()).all())
        assert_eight_bits(q, scale, y, block or D)


# ---------------------------------------------------------------------------------------------- segments whose decay leaves the range
def long_call(rate, step, S=3000):
    """A narrow, long call (cut into segments) of 64 channels and 4 states, without a softplus."""
    r = lambda *s: torch.randn(*s, generator=gen(31))
    return dict(x=torch.zeros(1, S, 64), dt=torch.full((1, S, 64), step), A=torch.full((64, 4), rate), B=r(1, S, 4), C=r(1, S, 4), D=None, z=None,
                dt_bias=None)


def test_scan_segments_whose_decay_leaves_the_range(pk):
    """A segment's decay may be more, or less, than a float holds: nothing grows to nothing, next to nothing to something, and
    something is left of what is large, as position by position."""
    S = 3000
    assert pk._lib.lib().mlstm_ssm_fwd_workspace(1, S, 64, 1, 4) > 0
    a = long_call(4.0, 1.0)
    a["x"][:, -10:] = 1.0                              # e^40 behind them; e^192 over 48 positions in front
    y, state = pk.state_space_scan(**on_gpu(a), return_state=True)
    want, end = oo.scan(**a)
    ym, hm = scan_mag(a, False)
    off(state, end, U, scan_loss(S, 4) * hm, "state from nothing")
    off(y, want, U, scan_loss(S, 4) * ym, "y from nothing")
    for rate, before in ((2.0, 1e-36), (-2.0, 1e36)):
        a = long_call(rate, 0.0)
        a["dt"][:, :48] = 1.0                          # e^96, then nothing
        a["initial"] = torch.full((1, 64, 4), before)
        y, state = pk.state_space_scan(**on_gpu(a), return_state=True)
        want, end = oo.scan(**a)
        ym, hm = scan_mag(a, False)
        off(state, end, U, scan_loss(S, 4) * hm, "state")
        off(y, want, U, scan_loss(S, 4) * ym, "y")


def test_scan_gradients_over_segments_whose_decay_leaves_the_range(pk):
    """The same on the way back: where no gradient comes from behind, none grows out of it."""
    S = 3000
    a = long_call(4.0, 1.0)
    a["dt"][:, :100] = 0.02
    dy = torch.zeros(1, S, 64)
    dy[:, :100] = torch.randn(1, 100, 64, generator=gen(1))
    names = [n for n in NAMES if a[n] is not None]
    d = {k: cu(v).requires_grad_(True) for k, v in a.items() if v is not None}
    got = torch.autograd.grad(pk.state_space_scan(**d), [d[n] for n in names], dy.cuda())
    ref = {k: oo.leaf(v) for k, v in a.items()}
    want = torch.autograd.grad(oo.scan(**ref)[0], [ref[n] for n in names], dy.double())
    mag = gradient_mag(a, dy, False)
    assert float(want[0].abs().max()) > 0.1
    for n, gv, wv in zip(names, got, want):
        off(gv, wv, U, (2 * scan_loss(S, 4) + (2 * S + 1 + 64) * U) * mag[n], "d" + n)


# ---------------------------------------------------------------------------------------------- many groups
def test_scan_of_many_groups(pk):
    """More groups than a grid's second dimension has places, one channel each."""
    G, S, N = 65537, 2, 1
    g = gen(33)
    r = lambda *s: torch.randn(*s, generator=g)
    a = dict(x=r(1, S, G), dt=r(1, S, G), A=-torch.exp(r(G, N)), B=r(1, S, G, N), C=r(1, S, G, N), D=None, z=None, dt_bias=None)
    dy = r(1, S, G)
    names = [n for n in NAMES if a[n] is not None]
    d = {k: cu(v).requires_grad_(True) for k, v in a.items() if v is not None}
    y = pk.state_space_scan(**d, dt_softplus=True)
    got = torch.autograd.grad(y, [d[n] for n in names], dy.cuda())
    ref = {k: oo.leaf(v) for k, v in a.items()}
    out = oo.scan(**ref, softplus=True)[0]
    off(y, out, U, scan_loss(S, N) * scan_mag(a, True)[0], "y")
    want = torch.autograd.grad(out, [ref[n] for n in names], dy.double())
    mag = gradient_mag(a, dy, True)
    for n, gv, wv in zip(names, got, want):
        off(gv, wv, U, (2 * scan_loss(S, N) + (2 * S + 1 + 64) * U) * mag[n], "d" + n)


# ---------------------------------------------------------------------------------------------- padding beside decays of -inf
def test_scan_gradients_of_padding_beside_decays_of_minus_infinity(pk):
    a, _ = scan_inputs(F32, 2, 60, 64, 16, 1, 41)
    a["A"][3, 2] = a["A"][10, 0] = -float("inf")
    gap = torch.zeros(60, dtype=torch.bool)
    gap[[0, 1, 17, 18, 33, 58, 59]] = True
    a["dt"][:, gap] = -float("inf")
    dy = 100 * torch.randn(2, 60, 64, generator=gen(42))
    names = [n for n in NAMES if a[n] is not None]
    d = {k: cu(v).requires_grad_(True) for k, v in a.items() if v is not None}
    got = dict(zip(names, torch.autograd.grad(pk.state_space_scan(**d, dt_softplus=True), [d[n] for n in names], dy.cuda())))
    assert all(bool(torch.isfinite(g).all()) for g in got.values())
    assert not got["dt"][:, gap.cuda()].any() and not got["B"][:, gap.cuda()].any()


# ---------------------------------------------------------------------------------------------- values near the largest
@pytest.mark.parametrize("S,C", [(1, 8), (3, 7), (3, 8), (70, 8)])
@pytest.mark.parametrize("silu", [True, False])
def test_convolution_gradient_behind_a_huge_last_input(pk, S, C, silu):
    """What the walk adds up behind the last position may be beyond a float; it belongs to no output."""
    x, dy = torch.randn(1, S, C, generator=gen(S)), torch.randn(1, S, C, generator=gen(2))
    x[:, -1] = 3e38
    w = torch.tensor([1.5, -1.25, 2.0, 0.5]).repeat(C, 1)          # half of it at the last position, twice of it behind
    xc = x.cuda().requires_grad_(True)
    got = torch.autograd.grad(pk.short_convolution(xc, w.cuda(), None, "silu" if silu else None), xc, dy.cuda())[0]
    ref = oo.leaf(x)
    want = torch.autograd.grad(oo.conv(ref, w, None, silu)[0], ref, dy.double())[0]
    # as in test_convolution_gradients; the slope is exactly 1 where the last input counts
    x[:, -1] = 0
    pre, d = oo.conv(x.abs(), w.abs())[0], 1.1 * dy.double().abs()
    fold = lambda t: oo.conv(t.flip(1), w.abs())[0].flip(1)
    off(got, want, U, fold(d * (5 * U * pre * silu + 16 * U)) + 4 * U * fold(d), "dx")


# ---------------------------------------------------------------------------------------------- kernels that only large calls reach
@pytest.mark.parametrize("dtype,b,S,ch,N,G,softplus,skip,gated,bias,initial,wide", [
    (BF16, 38, 33, 256, 16, 1, True, True, True, True, False, 0), (F32, 38, 17, 255, 16, 1, True, True, False, True, False, 0),
    (F16, 75, 40, 192, 11, 2, True, False, True, True, False, 0), (F32, 50, 24, 160, 9, 1, False, True, False, False, False, 0),
    (BF16, 38, 7, 250, 16, 1, True, True, False, True, False, 2), (F16, 150, 50, 21, 13, 1, True, True, True, True, False, 0)])
def test_scan_gradients_of_many_blocks(pk, dtype, b, S, ch, N, G, softplus, skip, gated, bias, initial, wide):
    """9 to 16 states with more than 148 blocks of 64 channels: two blocks of four warps on each SM, in the place of one of eight."""
    assert b * G * -(-ch // G // 64) > 148
    test_scan_gradients(pk, dtype, b, S, ch, N, G, softplus, skip, gated, bias, initial, wide)


@pytest.mark.parametrize("dtype,b,S,ch,N,G", [(BF16, 200, 1, 4096, 16, 1), (F32, 151, 3, 4096, 13, 2), (F16, 301, 2, 2048, 64, 1), (BF16, 700, 1, 1000, 4, 1),
                                              (F32, 233, 1, 1037, 30, 1)])
def test_scan_tokens_of_a_full_batch(pk, dtype, b, S, ch, N, G):
    """More sequences than the blocks along them: each block takes several, an uneven share at the end, its states fetched ahead."""
    g = torch.Generator("cuda").manual_seed(b)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, dt, z = (r(b, S, ch).to(dtype) for _ in range(3))
    B, C = (r(b, S, G, N).to(dtype) for _ in range(2))
    A, D, bias, first = -torch.exp(r(ch, N)), r(ch), r(ch) - 2, r(b, ch, N)
    call = lambda at, **kw: pk.state_space_scan(x[at], dt[at], A, B[at], C[at], D, z[at], bias, True, initial=first[at], return_state=True, **kw)
    y, state = call(slice(None))
    alone = [call(slice(k, k + 1)) for k in range(b)]
    assert torch.equal(y, torch.cat([v[0] for v in alone])) and torch.equal(state, torch.cat([v[1] for v in alone]))
    a = dict(x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=bias, initial=first)
    a = {k: v.cpu() for k, v in a.items()}
    want, end = oo.scan(**a, softplus=True)
    ym, hm = scan_mag(a, True)
    off(state, end, U, scan_loss(S, N) * hm, "state")
    off(y, want, oo.HALF_STEP[dtype], scan_loss(S, N) * ym, "y")
    again, over = call(slice(None), state_out=first)          # over the states that come in
    assert over is first and torch.equal(again, y) and torch.equal(first, state)


ALIGNED = [(dtype, 2, 333, C, W, bias, silu, False, w32, wide)
           for dtype, C, w32 in ((BF16, 136, False), (BF16, 72, True), (F16, 64, False), (F16, 200, True), (F32, 66, False))
           for W in (2, 3, 4) for silu, bias, wide in ((True, False, 0), (False, True, 0), (True, True, 8), (False, False, 16))]


@pytest.mark.parametrize("dtype,B,S,C,W,bias,silu,initial,w32,wide", ALIGNED)
def test_convolution_of_aligned_channels(pk, dtype, B, S, C, W, bias, silu, initial, w32, wide):
    """Several channels per thread with every number of taps, with and without silu and bias, in both directions."""
    test_convolution(pk, dtype, B, S, C, W, bias, silu, initial, w32, wide)
    test_convolution_gradients(pk, dtype, B, S, C, W, bias, silu, initial, w32, wide)


# ---------------------------------------------------------------------------------------------- combinations of the norm's options
@pytest.mark.parametrize("D,block", [(64, 32), (96, None), (128, 64), (33, None)])
def test_quantized_norm_of_every_head(pk, D, block):
    g = gen(D)
    h, w, res = torch.randn(2, 3, 41, D, generator=g) * 4, 1 + 0.3 * torch.randn(3, D, generator=g), torch.randn(2, 3, 41, D, generator=g)
    y = pk.residual_rms_norm(h.cuda(), w.cuda())
    q, scale = pk.residual_rms_norm_quantized(h.cuda(), w.cuda(), block=block)
    assert q.shape == h.shape and scale.shape == (2, 3, 41, D // (block or D))
    assert_eight_bits(q, scale, y, block or D)
    y, s = pk.residual_rms_norm(h.cuda(), w.cuda(), residual=res.cuda())
    q, scale, total = pk.residual_rms_norm_quantized(h.cuda(), w.cuda(), residual=res.cuda(), block=block)
    assert torch.equal(total, s)
    assert_eight_bits(q, scale, y, block or D)


@pytest.mark.parametrize("dtype,wdt,out", [(F16, F16, BF16), (BF16, F32, F16), (BF16, BF16, F32), (F32, F32, F16), (F16, F32, F16)])
@pytest.mark.parametrize("shape,heads", [((37, 520), 0), ((2, 3, 50, 64), 3), ((5, 1001), 0)])
def test_norm_of_a_float32_stream_in_every_type(pk, dtype, wdt, out, shape, heads):
    """A float32 residual stream takes x of any type and gives its norm in any other; gradients of both, through both results."""
    g = gen(sum(shape))
    D = shape[-1]
    x, res = (2 * torch.randn(*shape, generator=g)).to(dtype), 3 * torch.randn(*shape, generator=g)
    weight = (1 + 0.3 * torch.randn(*((heads, D) if heads else (D,)), generator=g)).to(wdt)
    dy, ds = torch.randn(*shape, generator=g).to(out), torch.randn(*shape, generator=g)
    leaves = [cu(t).requires_grad_(True) for t in (x, weight, res)]
    y, s = pk.residual_rms_norm(leaves[0], leaves[1], residual=leaves[2], out_dtype=out)
    assert y.dtype == out and s.dtype == F32
    got = torch.autograd.grad((y, s), leaves, (cu(dy), cu(ds)))
    v, wl = oo.leaf(s.detach().cpu()), oo.leaf(weight)
    want = oo.norm(v, wl)[0]
    off(y, want, oo.HALF_STEP[out], 32 * U * want.abs(), "y")
    ref = torch.autograd.grad(want, (v, wl), dy.double())
    # as in test_norm_gradients
    r = 1 / torch.sqrt(v.detach().square().mean(-1, keepdim=True) + 1e-6)
    u = dy.double().abs() * (weight.double().abs()[:, None] if heads else weight.double().abs())
    mag = r * (u + v.detach().abs() * r * r * (u * v.detach().abs()).mean(-1, keepdim=True)) + ds.double().abs()
    dv = ref[0] + ds.double()
    off(got[0], dv, oo.HALF_STEP[dtype], 64 * U * mag, "dx")
    off(got[2], dv, U, 64 * U * mag, "dresidual")
    lost = (dy.double() * v.detach() * r).abs()
    lost = lost.sum((0, 2)) if heads else lost.reshape(-1, D).sum(0)
    off(got[1], ref[1], oo.HALF_STEP[wdt], (s.numel() / D / 100 + 300) * U * lost, "dweight")
