"""The operators around a recurrent sequence mixer, as measurable cases: the short causal convolution in front of it, the
selective state space scan (prompts, training, single tokens) and the root-mean-square norm with the residual's addition.

    listed()              the named cases
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   what a user has in hand before the call, on the GPU, from the seed alone
    run(state)            one pass through an operator, outputs whole
    work(case)            bytes and flops of one pass that the operator cannot do without
    exact(case, seed)     the outputs of ``run`` from the operator's definition in 64 bits

With ``own`` false ``run`` computes the operators in elementary torch operations in 32 bits, rounded once at the end; with
``own`` true it calls this library's entry points.  A case has a ``kind``, which says who calls what:

    conv        ``short_convolution``: a prompt, forward
    convtrain   the same with its gradients
    convtoken   the same for one or a few new tokens behind a carried state
    scan        ``state_space_scan``: a prompt behind a carried state, the state carried out
    scantrain   the same without states, with the gradients of all inputs
    scantoken   one or a few new tokens behind a carried state
    norm        ``residual_rms_norm``: forward
    normtrain   the same with its gradients
    normheads   ``residual_rms_norm`` on a mixer's float32 output, head by head, with its gradients
    normquant   ``residual_rms_norm_quantized``: forward, the result in 8 bits with scales
"""
import importlib
import math

import torch

own = False

_PKG = "xlstm-triton-cuda-implementation_b200"
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_FP8_MAX = 448.0          # the largest value of the 8-bit type (4 bits of exponent, 3 of mantissa)
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _conv(kind, dtype, B, S, C, W=4, act="silu", bias=True, name=None):
    c = dict(kind=kind, dtype=dtype, B=B, S=S, C=C, W=W, act=act, bias=bias)
    return c if name is None else dict(c, name=name)


def _scan(kind, dtype, B, S, C, N, G=1, gated=True, skip=True, name=None):
    c = dict(kind=kind, dtype=dtype, B=B, S=S, C=C, N=N, G=G, gated=gated, skip=skip)
    return c if name is None else dict(c, name=name)


def _norm(kind, dtype, rows, D, NH=1, residual=True, weight=True, block=0, name=None):
    c = dict(kind=kind, dtype=dtype, rows=rows, D=D, NH=NH, residual=residual, weight=weight, block=block)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one new token of each of a few sequences: nearly all latency
        _conv("convtoken", "bf16", 16, 1, 2048, name="conv_token_bf16"),
        # a few short prompts, with a length that is a multiple of nothing
        _conv("conv", "fp16", 3, 777, 1344, name="conv_prompt_ragged_fp16"),
        # a model-scale training step's convolution, forward and backward
        _conv("convtrain", "bf16", 4, 4096, 4096, name="conv_train_bf16"),
        # one new token of a single sequence
        _scan("scantoken", "bf16", 1, 1, 1024, 16, name="scan_token_one_bf16"),
        # one new token of each sequence of a full serving batch
        _scan("scantoken", "bf16", 256, 1, 4096, 16, name="scan_token_batch_bf16"),
        # a long prompt of a single sequence, its state carried out
        _scan("scan", "bf16", 1, 16384, 1024, 16, name="scan_prompt_long_bf16"),
        # a few prompts in full precision, sizes that are multiples of nothing, two groups of channels
        _scan("scan", "fp32", 3, 1001, 600, 24, G=2, name="scan_prompt_ragged_fp32"),
        # a small model's training step
        _scan("scantrain", "fp16", 2, 1000, 512, 16, name="scan_train_small_fp16"),
        # a model-scale training step
        _scan("scantrain", "bf16", 4, 4096, 4096, 16, name="scan_train_bf16"),
        # the norm of one new token of each of a few sequences
        _norm("norm", "bf16", 16, 2048, name="norm_token_bf16"),
        # a model-scale training step's norm, residual stream in and out, forward and backward
        _norm("normtrain", "bf16", 16384, 4096, name="norm_train_bf16"),
        # a prompt's norm whose result goes to an 8-bit product: one scale for 128 values
        _norm("normquant", "bf16", 8192, 4096, block=128, name="norm_quant_bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One case of the ranges behind the listed ones: lengths, batches and widths over their logarithm, half of the widths
    as they fall and half a multiple of 64; no more values, states or products than the largest listed case has."""
    kind = rng.choice(["conv", "convtrain", "convtoken", "scan", "scan", "scantrain", "scantrain", "scantoken", "norm", "normtrain",
                       "normheads", "normquant"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        width = lambda lo, hi: (lambda c: c // 64 * 64 if c >= 64 and rng.random() < 0.5 else c)(_log_int(rng, lo, hi))
        if kind.startswith("conv"):
            S = rng.choice([1, 1, 1, 2, 5, 8]) if kind == "convtoken" else _log_int(rng, 2, 16384)
            c = _conv(kind, dtype, _log_int(rng, 1, 256 if kind == "convtoken" else 16), S, width(48, 8192), rng.choice([2, 3, 4, 4, 4]),
                      rng.choice(["silu", "silu", "none"]), rng.random() < 0.7)
            if c["B"] * c["S"] * c["C"] <= 4 * 4096 * 4096:
                return c
        elif kind.startswith("scan"):
            S = rng.choice([1, 1, 1, 2, 5, 8]) if kind == "scantoken" else _log_int(rng, 2, 16384)
            G = rng.choice([1, 1, 1, 2, 4])
            c = _scan(kind, dtype, _log_int(rng, 1, 256 if kind == "scantoken" else 16), S, G * width(48 // G, 8192 // G),
                      rng.choice([4, 8, 16, 16, 16, 24, 32, 64]), G, rng.random() < 0.6, rng.random() < 0.8)
            states = c["B"] * c["C"] * c["N"]
            if states * S <= 4 * 4096 * 4096 * 16 and states <= 256 * 4096 * 16:
                return c
        else:
            NH = rng.choice([1, 2, 4, 8]) if kind == "normheads" else 1
            rows, D = NH * _log_int(rng, 1, 65536), width(32, 256) if kind == "normheads" else width(64, 16384)
            block = rng.choice([0, 32, 128]) if kind == "normquant" else 0
            if block:
                D = max(block, D // block * block)
            c = _norm(kind, dtype, rows, D, NH, kind != "normheads" and rng.random() < 0.7, rng.random() < 0.9, block)
            if rows * D <= 16384 * 4096:
                return c


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt, kind = _DTYPES[case["dtype"]], case["kind"]
    normal = lambda *shape: torch.randn(shape, device=dev, generator=g)
    uniform = lambda lo, hi, *shape: lo + (hi - lo) * torch.rand(shape, device=dev, generator=g)
    s = dict(case=case)
    if kind.startswith("conv"):
        B, S, C, W = (case[n] for n in ("B", "S", "C", "W"))
        s["x"] = normal(B, S, C).to(dt)
        s["weight"] = (normal(C, W) * W ** -0.5).to(dt)
        s["bias"] = (0.1 * normal(C)).to(dt) if case["bias"] else None
        if kind == "convtoken":
            s["initial"] = normal(B, W - 1, C).to(dt)
        if kind == "convtrain":
            s["dy"] = normal(B, S, C).to(dt)
    elif kind.startswith("scan"):
        B, S, C, N, G = (case[n] for n in ("B", "S", "C", "N", "G"))
        v = normal(B, S, C)
        s["x"] = (v * torch.sigmoid(v)).to(dt)                     # behind the convolution's activation
        s["dt"] = (0.5 * normal(B, S, C)).to(dt)                   # pre-activation of the time step
        s["B"], s["C"] = (normal(B, S, G, N).to(dt) for _ in range(2))
        s["A"] = -torch.arange(1, N + 1, device=dev, dtype=torch.float32) * torch.exp(0.1 * normal(C, N))
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), C))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))       # softplus of it is the step
        s["D"] = 1.0 + 0.1 * normal(C) if case["skip"] else None
        s["z"] = normal(B, S, C).to(dt) if case["gated"] else None
        if kind == "scantrain":
            s["dy"] = normal(B, S, C).to(dt)
        else:
            s["initial"] = 0.3 * normal(B, C, N)
    else:
        rows, D, NH = (case[n] for n in ("rows", "D", "NH"))
        if kind == "normheads":                                    # a mixer's float32 result, [batch, heads, positions, head dimension]
            s["x"] = normal(1, NH, rows // NH, D) * torch.exp(normal(1, NH, rows // NH, 1))
            s["weight"] = 1.0 + 0.1 * normal(NH, D) if case["weight"] else None
        else:
            s["x"] = normal(rows, D).to(dt)
            s["residual"] = (3.0 * normal(rows, D)).to(dt) if case["residual"] else None
            s["weight"] = (1.0 + 0.1 * normal(D)).to(dt) if case["weight"] else None
        if kind in ("normtrain", "normheads"):
            s["dy"] = normal(*s["x"].shape).to(dt)
            if s.get("residual") is not None:
                s["ds"] = normal(rows, D).to(dt)                   # what the residual stream's later users hand back
    if kind in ("convtrain", "scantrain", "normtrain", "normheads"):
        s["leaves"] = [n for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "weight", "bias", "residual") if s.get(n) is not None]
        for n in s["leaves"]:
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the library's entry points
def _own(s):
    pkg, case, kind = importlib.import_module(_PKG), s["case"], s["case"]["kind"]
    if kind.startswith("conv"):
        act = None if case["act"] == "none" else case["act"]
        if kind == "convtoken":
            return pkg.short_convolution(s["x"], s["weight"], s["bias"], act, initial=s["initial"], return_state=True)
        y = pkg.short_convolution(s["x"], s["weight"], s["bias"], act)
    elif kind.startswith("scan"):
        args = (s["x"], s["dt"], s["A"], s["B"], s["C"])
        more = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
        if kind != "scantrain":
            return pkg.state_space_scan(*args, **more, initial=s["initial"], return_state=True)
        y = pkg.state_space_scan(*args, **more)
    elif kind == "normquant":
        return pkg.residual_rms_norm_quantized(s["x"], s["weight"], residual=s["residual"], eps=_EPS, block=case["block"] or None)
    elif kind == "normheads":
        y = pkg.residual_rms_norm(s["x"], s["weight"], eps=_EPS, out_dtype=_DTYPES[case["dtype"]])
    else:
        y = pkg.residual_rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
    if "leaves" not in s:
        return y
    ys, dys = ((y, s["dy"]) if isinstance(y, torch.Tensor) else (y, (s["dy"], s["ds"])))
    grads = torch.autograd.grad(ys, [s[n] for n in s["leaves"]], dys)
    return {"y": [y.detach()] if isinstance(y, torch.Tensor) else [v.detach() for v in y], "grad": dict(zip(s["leaves"], grads))}


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_conv(s):
    case = s["case"]
    W, silu = case["W"], case["act"] == "silu"
    x, w = s["x"].detach(), s["weight"].detach().float()
    B, S, C = x.shape
    before = s["initial"] if "initial" in s else x.new_zeros(B, W - 1, C)
    rows = torch.cat([before, x], 1)
    # every output row is a product of W neighbouring rows with the weights
    windows = rows.float().unfold(1, W, 1)                         # [B, S, C, W]
    pre = (windows * w).sum(-1)
    if s["bias"] is not None:
        pre = pre + s["bias"].detach().float()
    sig = torch.sigmoid(pre)
    y = (pre * sig if silu else pre).to(x.dtype)
    if case["kind"] == "convtoken":
        return y, rows[:, S:].contiguous()
    if case["kind"] == "conv":
        return y
    d = s["dy"].float()
    if silu:
        d = d * sig * (1 + pre * (1 - sig))
    later = torch.cat([d, d.new_zeros(B, W - 1, C)], 1).unfold(1, W, 1)
    grad = {"x": (later * w.flip(1)).sum(-1).to(x.dtype), "weight": (d[..., None] * windows).sum((0, 1)).to(s["weight"].dtype)}
    if s["bias"] is not None:
        grad["bias"] = d.sum((0, 1)).to(s["bias"].dtype)
    return {"y": [y], "grad": grad}


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dimension 1 by doubling, a and b being used up."""
    d = 1
    while d < a.shape[1]:
        b[:, d:] = b[:, d:] + a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _plain_scan(s):
    case = s["case"]
    N, G = case["N"], case["G"]
    x16, train = s["x"].detach(), case["kind"] == "scantrain"
    B, S, C = x16.shape
    P = C // G
    wide = lambda t: t.detach().float().view(B, S, G, P, 1)        # a value for each channel
    per = lambda t: t.detach().float().view(B, S, G, 1, N)         # a vector for each group
    x, A = wide(x16), s["A"].detach().view(G, P, N)
    raw = s["dt"].detach().float() + s["dt_bias"].detach()
    delta = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    dl, Bv, Cv = delta.view(B, S, G, P, 1), per(s["B"]), per(s["C"])
    a = torch.exp(dl * A)
    b = (dl * x) * Bv
    if "initial" in s:
        b[:, 0] += a[:, 0] * s["initial"].view(B, G, P, N)
    h = _recurrence(a.clone() if train else a, b)
    y = (h * Cv).sum(-1).view(B, S, C)
    if s["D"] is not None:
        y = y + s["D"].detach() * x16.float()
    if s["z"] is not None:
        z = s["z"].detach().float()
        sig = torch.sigmoid(z)
    out = (y * z * sig if s["z"] is not None else y).to(x16.dtype)
    if not train:
        return out, h[:, -1].reshape(B, C, N).clone()
    dy, grad = s["dy"].float(), {}
    if s["z"] is not None:
        grad["z"] = (dy * y * sig * (1 + z * (1 - sig))).to(x16.dtype)
        dy = dy * z * sig
    dyv = dy.view(B, S, G, P, 1)
    grad["C"] = (dyv * h).sum(3).to(x16.dtype)
    back = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    g = _recurrence(back, (dyv * Cv).flip(1)).flip(1)              # the gradient of the state behind every position
    del back
    carried = torch.cat([torch.zeros_like(h[:, :1]), a[:, 1:] * h[:, :-1]], 1)
    del a, h
    grad["B"] = (g * (dl * x)).sum(3).to(x16.dtype)
    into = (g * Bv).sum(-1).view(B, S, C)
    carried *= g
    del g
    ddelta = into * x16.float() + (carried * A).sum(-1).view(B, S, C)
    carried *= dl
    grad["A"] = carried.sum((0, 1)).view(C, N)
    dx = delta * into
    if s["D"] is not None:
        dx = dx + s["D"].detach() * dy
        grad["D"] = (dy * x16.float()).sum((0, 1))
    draw_ = ddelta * torch.sigmoid(raw)
    grad["x"], grad["dt"], grad["dt_bias"] = dx.to(x16.dtype), draw_.to(x16.dtype), draw_.sum((0, 1))
    return {"y": [out], "grad": grad}


def _plain_norm(s):
    case, kind = s["case"], s["case"]["kind"]
    x, r, w = s["x"].detach(), s.get("residual"), s["weight"]
    out = _DTYPES[case["dtype"]]
    total = x if r is None else (x.float() + r.detach().float()).to(r.dtype)     # the residual stream, in its own type
    v = total.float()
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    wf = 1.0 if w is None else w.detach().float().view(-1, 1, case["D"]) if kind == "normheads" else w.detach().float()
    y = v * rstd * wf
    if kind == "normquant":
        block = case["block"] or case["D"]
        blocks = y.view(-1, case["D"] // block, block)
        top = blocks.abs().amax(-1)
        scale = torch.where(top > 0, top / _FP8_MAX, torch.ones_like(top))
        q = (blocks / scale[..., None]).view(y.shape).to(torch.float8_e4m3fn)
        return (q, scale) if r is None else (q, scale, total)
    ys = [y.to(out)] if r is None else [y.to(out), total]
    if kind == "norm":
        return ys[0] if r is None else tuple(ys)
    dy, grad = s["dy"].float(), {}
    if w is not None:
        grad["weight"] = (dy * v * rstd).sum((0, 2) if kind == "normheads" else 0).to(w.dtype)
    dn = dy * wf
    dv = rstd * (dn - v * rstd * rstd * (dn * v).mean(-1, keepdim=True))
    if r is not None:
        dv = dv + s["ds"].float()
        grad["residual"] = dv.to(r.dtype)
    grad["x"] = dv.to(x.dtype)
    return {"y": ys, "grad": grad}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return _plain_conv(state) if kind.startswith("conv") else _plain_scan(state) if kind.startswith("scan") else _plain_norm(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es, kind = (4 if case["dtype"] == "fp32" else 2), case["kind"]
    if kind.startswith("conv"):
        n, W = case["B"] * case["S"] * case["C"], case["W"]
        params = case["C"] * (W + case["bias"]) * es
        act = 5 if case["act"] == "silu" else 0
        if kind == "convtrain":          # x, dy in, y, dx out; product forward, and by x and by the weights backward
            return {"bytes": float(4 * n * es + 2 * params), "flops": float(n * (6 * W + 3 * act))}
        state = 2 * case["B"] * (W - 1) * case["C"] * es if kind == "convtoken" else 0
        return {"bytes": float(2 * n * es + params + state), "flops": float(n * (2 * W + act))}
    if kind.startswith("scan"):
        B, S, C, N, G = (case[n] for n in ("B", "S", "C", "N", "G"))
        wide, vectors, params = B * S * C * es, 2 * B * S * G * N * es, 4 * C * (N + 1 + case["skip"])
        ins = wide * (2 + case["gated"]) + vectors + params
        if kind == "scantrain":          # the inputs and dy in, y and the inputs' gradients out
            return {"bytes": float(2 * ins + 2 * wide), "flops": float(B * S * C * (21 * N + 30))}
        # per state: its decay (product, exponential), the new state (two products, a sum) and its part of the output
        return {"bytes": float(ins + wide + 8 * B * C * N), "flops": float(B * S * C * (7 * N + 15))}
    n, D = case["rows"] * case["D"], case["D"]
    w = case["NH"] * D * es if case["weight"] else 0
    if kind == "normheads":              # float32 in and its gradient out, 16-bit result and its gradient
        return {"bytes": float(n * (8 + 2 * es) + 2 * case["weight"] * case["NH"] * D * 4), "flops": float(14 * n)}
    if kind == "normtrain":              # x, residual, dy, ds in; y, the sum, dx, dresidual out
        return {"bytes": float(n * es * (8 if case["residual"] else 4) + 2 * w), "flops": float(15 * n)}
    out = n + 4 * n // (case["block"] or D) if kind == "normquant" else n * es
    return {"bytes": float(n * es * (3 if case["residual"] else 1) + out + w), "flops": float(6 * n)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_conv(s):
    case, W = s["case"], s["case"]["W"]
    d = {n: s[n].detach().double().requires_grad_(True) for n in ("x", "weight", "bias") if s[n] is not None}
    before = s["initial"].double() if "initial" in s else d["x"].new_zeros(case["B"], W - 1, case["C"])
    rows, S = torch.cat([before, d["x"]], 1), case["S"]
    y = sum(rows[:, k:k + S] * d["weight"][:, k] for k in range(W))
    if "bias" in d:
        y = y + d["bias"]
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    if case["kind"] == "convtoken":
        return y.detach(), rows[:, S:].detach().clone()
    if case["kind"] == "conv":
        return y.detach()
    return {"y": [y.detach()], "grad": dict(zip(d, torch.autograd.grad(y, list(d.values()), s["dy"].double())))}


def _exact_scan(s):
    """Position by position, a slice of a group's channels at a time; gradients by automatic differentiation."""
    case = s["case"]
    train, N, G, B, S, C = case["kind"] == "scantrain", case["N"], case["G"], case["B"], case["S"], case["C"]
    P, most = C // G, max(1, (1 << 28) // (B * S * N))
    outs, ends, grads = [], [], {}
    with torch.set_grad_enabled(train):
        for at in range(0, C, P):
            vec = {n: s[n].detach()[:, :, at // P].double().requires_grad_(train) for n in ("B", "C")}
            for lo in range(at, at + P, most):
                hi = min(lo + most, at + P)
                d = {n: s[n].detach()[..., lo:hi].double() for n in ("x", "dt", "D", "z", "dt_bias") if s[n] is not None}
                d["A"] = s["A"].detach()[lo:hi].double()
                for t in d.values():
                    t.requires_grad_(train)
                step = torch.nn.functional.softplus(d["dt"] + d["dt_bias"], threshold=700.0)
                keep = torch.exp(step[..., None] * d["A"]).unbind(1)
                new = ((step * d["x"])[..., None] * vec["B"][:, :, None]).unbind(1)
                h, hs = s["initial"][:, lo:hi].double() if "initial" in s else new[0].new_zeros(new[0].shape), []
                for t in range(S):
                    h = torch.addcmul(new[t], keep[t], h)
                    hs.append(h)
                del keep, new
                y = torch.einsum("bscn,bsn->bsc", torch.stack(hs, 1), vec["C"])
                if "D" in d:
                    y = y + d["D"] * d["x"]
                if "z" in d:
                    y = y * d["z"] / (1 + torch.exp(-d["z"]))
                outs.append(y.detach())
                ends.append(h.detach())
                if train:
                    names = list(d) + ["B", "C"]
                    got = torch.autograd.grad(y, list(d.values()) + [vec["B"], vec["C"]], s["dy"][..., lo:hi].double())
                    for n, v in zip(names, got):
                        grads.setdefault(n, []).append((at // P, v))
                del hs, h, y
    y = torch.cat(outs, -1)
    if not train:
        return y, torch.cat(ends, 1)
    grad = {n: torch.cat([v for _, v in got], 0 if n == "A" else -1) for n, got in grads.items() if n not in ("B", "C")}
    for n in ("B", "C"):
        grad[n] = torch.stack([sum(v for k, v in grads[n] if k == group) for group in range(G)], 2)
    return {"y": [y], "grad": grad}


def _exact_norm(s):
    case, kind = s["case"], s["case"]["kind"]
    d = {n: s[n].detach().double() for n in ("x", "residual", "weight") if s.get(n) is not None}
    total = d["x"] if "residual" not in d else (d["x"] + d["residual"]).to(s["residual"].dtype).double()
    v = total.clone().requires_grad_(True)
    w = d["weight"].requires_grad_(True) if "weight" in d else torch.ones((), dtype=torch.float64, device=v.device)
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + _EPS) * (w[:, None] if kind == "normheads" and "weight" in d else w)
    if kind == "normquant":
        block = case["block"] or case["D"]
        blocks = y.detach().reshape(-1, case["D"] // block, block)
        top = blocks.abs().amax(-1)
        scale = torch.where(top > 0, top / _FP8_MAX, torch.ones_like(top))
        q = (blocks / scale[..., None]).reshape(y.shape)           # in 64 bits: what the 8-bit values come near to
        return (q, scale) if "residual" not in d else (q, scale, total)
    ys = [y.detach()] if "residual" not in d else [y.detach(), total]
    if kind == "norm":
        return ys[0] if len(ys) == 1 else tuple(ys)
    got = torch.autograd.grad(y, [v] + ([w] if "weight" in d else []), s["dy"].double())
    dv = got[0] + s["ds"].double() if "residual" in d else got[0]
    grad = {"x": dv}
    if "residual" in d:
        grad["residual"] = dv
    if "weight" in d:
        grad["weight"] = got[1]
    return {"y": ys, "grad": grad}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    return _exact_conv(s) if kind.startswith("conv") else _exact_scan(s) if kind.startswith("scan") else _exact_norm(s)
