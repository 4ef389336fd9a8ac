"""CPU tests of the operators around the mixer: what the entry points refuse before they touch a device, the sizes of their scratch,
and that the C entry points check their arguments."""
import ctypes

import pytest
import torch

BF16 = torch.bfloat16


def test_convolution_refusals(pkg):
    f = pkg.short_convolution
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    for bad in (dict(x=torch.zeros(2, 5)), dict(x=torch.zeros(2, 0, 8)), dict(weight=torch.zeros(8, 1)), dict(weight=torch.zeros(8, 5)),
                dict(weight=torch.zeros(7, 4)), dict(bias=torch.zeros(7)), dict(activation="gelu"), dict(state_out=torch.zeros(2, 3, 8))):
        with pytest.raises(ValueError):
            f(**{**dict(x=x, weight=w), **bad})
    for bad in (dict(weight=w.half()), dict(bias=torch.zeros(8, dtype=BF16)), dict(x=x.to(BF16), weight=w.half())):
        with pytest.raises(TypeError):
            f(**{**dict(x=x, weight=w), **bad})
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, w)
    with pytest.raises(ValueError, match="plain call"):
        f(x.requires_grad_(True), w, return_state=True)
    with pytest.raises(ValueError, match="plain call"):
        f(torch.zeros(2, 5, 8), w, initial=torch.zeros(2, 3, 8, requires_grad=True))


def test_scan_refusals(pkg):
    f = pkg.state_space_scan
    ok = dict(x=torch.zeros(2, 5, 8), dt=torch.zeros(2, 5, 8), A=torch.zeros(8, 16), B=torch.zeros(2, 5, 16), C=torch.zeros(2, 5, 16))
    for bad in (dict(x=torch.zeros(2, 8)), dict(x=torch.zeros(0, 5, 8), dt=torch.zeros(0, 5, 8)), dict(dt=torch.zeros(2, 5, 1)),
                dict(z=torch.zeros(2, 4, 8)), dict(A=torch.zeros(8, 15)), dict(A=torch.zeros(16)), dict(B=torch.zeros(2, 5, 15)),
                dict(B=torch.zeros(2, 5, 3, 16), C=torch.zeros(2, 5, 3, 16)), dict(B=torch.zeros(2, 5, 0, 16), C=torch.zeros(2, 5, 0, 16)),
                dict(D=torch.zeros(7)), dict(dt_bias=torch.zeros(8, 1)), dict(state_out=torch.zeros(2, 8, 16)),
                dict(A=torch.zeros(8, 65), B=torch.zeros(2, 5, 65), C=torch.zeros(2, 5, 65)),
                dict(A=torch.zeros(8, 0), B=torch.zeros(2, 5, 0), C=torch.zeros(2, 5, 0))):
        with pytest.raises(ValueError):
            f(**{**ok, **bad})
    for bad in (dict(x=torch.zeros(2, 5, 8, dtype=BF16)), dict(A=torch.zeros(8, 16, dtype=BF16)), dict(D=torch.zeros(8, dtype=BF16)),
                dict(z=torch.zeros(2, 5, 8, dtype=BF16))):
        with pytest.raises(TypeError):
            f(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="CUDA"):
        f(**ok)
    with pytest.raises(RuntimeError, match="contiguous"):
        f(**{**ok, "A": torch.zeros(16, 8).t()})
    with pytest.raises(ValueError, match="plain call"):
        f(**{**ok, "A": torch.zeros(8, 16, requires_grad=True)}, return_state=True)


def test_norm_refusals(pkg):
    f, q = pkg.residual_rms_norm, pkg.residual_rms_norm_quantized
    x = torch.zeros(3, 64)
    for bad in (dict(x=torch.zeros(3, 0)), dict(x=torch.zeros(0, 64)), dict(x=torch.zeros(1, 16385)), dict(weight=torch.zeros(63)),
                dict(weight=torch.zeros(3, 64)), dict(x=torch.zeros(2, 3, 4, 64), weight=torch.zeros(2, 64)), dict(residual=torch.zeros(64))):
        with pytest.raises(ValueError):
            f(**{**dict(x=x), **bad})
    for bad in (dict(weight=torch.zeros(64, dtype=BF16)), dict(residual=torch.zeros(3, 64, dtype=BF16)), dict(out_dtype=torch.int8),
                dict(x=x.to(BF16), out_dtype=torch.float32), dict(x=x.double())):
        with pytest.raises(TypeError):
            f(**{**dict(x=x), **bad})
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x)
    for block in (16, 48, 256, 128):
        with pytest.raises(ValueError):
            q(x, block=block)
    with pytest.raises(ValueError, match="no gradients"):
        q(torch.zeros(3, 64, requires_grad=True))


def test_c_entry_points_check_their_arguments(pkg):
    L, p = pkg._lib.lib(), ctypes.c_void_p(4096)
    conv = lambda *d, dt=2, w=2: L.mlstm_conv_fwd(p, p, None, None, None, p, None, *d, dt, w, 1, None)
    assert conv(0, 1, 8, 4) == -1 and conv(1, 1, 8, 5) == -2 and conv(1, 1, 8, 1) == -2 and conv(70000, 1, 8, 4) == -2
    assert conv(1, 1, 8, 4, dt=3) == -1 and conv(1, 1, 8, 4, dt=2, w=1) == -1
    assert L.mlstm_conv_fwd(None, p, None, None, None, p, None, 1, 1, 8, 4, 2, 2, 1, None) == -1
    ssm = lambda *d, ws=None, n=0: L.mlstm_ssm_fwd(p, p, p, p, p, None, None, None, None, None, p, None, None, ws, n, *d, 2, 1, None)
    assert ssm(1, 5, 8, 3, 16) == -2 and ssm(1, 5, 8, 1, 65) == -2 and ssm(1, 0, 8, 1, 16) == -1
    assert ssm(1, 5000, 8, 1, 16) == -5 and ssm(1, 5000, 8, 1, 16, ws=p, n=64) == -5
    bad = (ctypes.c_longlong * 10)(*[-1] * 10)
    assert L.mlstm_ssm_fwd(p, p, p, p, p, None, None, None, None, bad, p, None, None, None, 0, 1, 5, 8, 1, 16, 2, 1, None) == -1
    # a gradient for an input that is not there, or none for one that is
    assert L.mlstm_ssm_bwd(p, p, p, p, p, p, None, None, None, None, p, p, p, p, p, p, p, None, None, p, 1 << 30, 1, 5, 8, 1, 16, 2, 1, None) == -1
    rms = lambda rows, D, groups=1, inner=1, block=0, s=2: L.mlstm_rms_fwd(p, None, None, p, None, p if block else None, rows, D, groups, inner,
                                                                          block, 1e-6, 2, s, 0, 2, None)
    assert rms(0, 8) == -1 and rms(1, 16385) == -2 and rms(10, 8, 3, 1) == -2 and rms(1, 64, block=48) == -2 and rms(1, 96, block=64) == -2
    assert rms(1, 8, s=0) == -1
    for code in (-1, -2, -3, -5):
        assert L.mlstm_status_string(code)


def test_scratch_sizes(pkg):
    L = pkg._lib.lib()
    # the channels alone fill the chip: one pass, no scratch; a narrow, long call is cut into segments
    assert L.mlstm_ssm_fwd_workspace(8, 4096, 4096, 1, 16) == 0 < L.mlstm_ssm_fwd_workspace(1, 16384, 512, 1, 16)
    assert L.mlstm_ssm_fwd_workspace(1, 16384, 512, 1, 65) == 0 == L.mlstm_ssm_bwd_workspace(1, 16384, 512, 3, 16)
    # a state of every 16 positions, the channels of each group rounded up to 64
    assert L.mlstm_ssm_checkpoint_floats(2, 100, 96, 2, 16) == 2 * 7 * 16 * 128
    # partial dB, dC: at most 512 MB at a time, whatever the batch
    one = 64 * 4096 * 16 * 8
    for B in (1, 4, 64, 1000):
        assert one <= L.mlstm_ssm_bwd_workspace(B, 4096, 4096, 1, 16) <= (512 << 20) + B * 18 * 4096 * 4 * 2 + (1 << 20)
    assert L.mlstm_rms_bwd_workspace(16384, 4096, 1, 1) <= 148 * 8 * 4096 * 4
    assert 0 < L.mlstm_rms_bwd_workspace(7, 100, 1, 1) <= 7 * 100 * 4
    assert L.mlstm_conv_bwd_workspace(4, 4096, 4096, 4, 2) <= 4 * 4096 // 64 * 5 * 4096 * 4


def test_convolution_scratch_covers_every_access_width(pkg):
    """The number of partial sums follows from the channels per thread, which follow from types, sizes and alignment: the query has
    to cover them all.  A call checks its scratch before its first launch (which fails here: no device)."""
    L = pkg._lib.lib()
    # 4 channels per thread: 16 blocks across 2048 channels, runs of 32 positions in blocks of four, one partial row each
    assert L.mlstm_conv_bwd_workspace(4, 4096, 2048, 4, 2) >= 4 * (4096 // (32 * 4)) * 5 * 2048 * 4
    if torch.cuda.is_available():
        pytest.skip("the calls would launch")
    at = lambda a: ctypes.c_void_p(a)
    for dt in (0, 2):
        for B, S, C in ((4, 4096, 2048), (1, 2000, 512), (2, 8192, 1024), (3, 777, 1344), (16, 500, 96), (1, 16384, 4096), (8, 3000, 768)):
            for base in (4096, 4100):                # all channels of a thread at once, or one by one
                need = L.mlstm_conv_bwd_workspace(B, S, C, 4, dt)
                rc = L.mlstm_conv_bwd(at(base), at(base), at(4096), None, None, at(base), at(4096), None, at(4096), need, B, S, C, 4, dt, dt, 1, None)
                assert rc not in (0, -5), (dt, B, S, C, base, rc)


def test_sizes_that_do_not_fit_are_refused_before_they_become_32_bits(pkg):
    at = lambda *s: torch.empty(s, device="meta")
    for shape in ((1, 2 ** 32 + 8, 8), (1, 2 ** 23 + 1, 8), (2 ** 32 + 1, 1, 8), (65536, 1, 8), (1, 1, 2 ** 24 + 1), (1, 1, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="at most"):
            pkg.short_convolution(at(*shape), at(shape[2], 4))
        if shape[1] != 2 ** 23 + 1:
            with pytest.raises(ValueError, match="at most"):
                pkg.state_space_scan(at(*shape), at(*shape), at(shape[2], 16), at(*shape[:2], 16), at(*shape[:2], 16))
    with pytest.raises(ValueError, match="fewer than"):
        pkg.state_space_scan(at(1, 2 ** 31 - 32, 8), at(1, 2 ** 31 - 32, 8), at(8, 16), at(1, 2 ** 31 - 32, 16), at(1, 2 ** 31 - 32, 16))
