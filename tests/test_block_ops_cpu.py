"""The block operators without a GPU: the 64-bit references' gradients against
differences, and every refusal that is made on the host."""

import ctypes

import pytest
import torch

import block_refs as refs
from gated_deltanet_jax_b200 import _build, _lib, ops


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        _build.build()
    return _lib.load()


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _check_differences(fn, args, cots, grads, eps=1e-6):
    """<grad, v> against a central difference of sum(out * cot) along a random v,
    for every argument: the difference's own error is O(eps^2) + 2^-53 / eps, far
    below 1e-7 of the value for these smooth functions of order-one numbers."""
    def value(a):
        return sum((o * c).sum() for o, c in zip(fn(*a), cots))
    for i, g in enumerate(grads):
        if args[i] is None:
            continue
        v = _rand(*args[i].shape, seed=100 + i)
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + eps * v, args[i] - eps * v
        num = (value(up) - value(dn)) / (2 * eps)
        assert abs(num - (g * v).sum()) <= 1e-7 * max(1.0, abs(num).item()), i


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("full", [True, False])
def test_scan_reference_gradients_match_differences(softplus, full):
    b, T, ch, G, N = 2, 7, 6, 2, 3
    x, dt = _rand(b, T, ch, seed=1), _rand(b, T, ch, seed=2)
    A = -_rand(ch, N, seed=3).abs()
    B, C = _rand(b, T, G, N, seed=4), _rand(b, T, G, N, seed=5)
    D, z = (_rand(ch, seed=6), _rand(b, T, ch, seed=7)) if full else (None, None)
    bias, h0 = (_rand(ch, seed=8), _rand(b, ch, N, seed=9)) if full else (None, None)
    dy, dhT = _rand(b, T, ch, seed=10), _rand(b, ch, N, seed=11)
    if not softplus:   # step sizes as given: positive, as a decay needs them
        dt, bias = dt.abs(), None if bias is None else bias.abs()

    def fn(*a):
        o = refs.scan_ref(*a, softplus=softplus)
        return o["y"], o["state"]
    args = [x, dt, A, B, C, D, z, bias, h0]
    g = refs.scan_ref(*args, softplus=softplus, dy=dy, dhT=dhT)
    _check_differences(fn, args, (dy, dhT), [g.get(k) for k in (
        "dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dstate")])


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("T", [1, 2, 9])
def test_conv_reference_gradients_match_differences(act, T):
    b, C, K = 2, 4, 4
    args = [_rand(b, T, C, seed=1), _rand(K, C, seed=2), _rand(C, seed=3),
            _rand(b, K - 1, C, seed=4)]
    dy, ds = _rand(b, T, C, seed=5), _rand(b, K - 1, C, seed=6)

    def fn(*a):
        o = refs.conv_ref(*a, act=act)
        return o["y"], o["state"]
    g = refs.conv_ref(*args, act=act, dy=dy, dstate=ds)
    _check_differences(fn, args, (dy, ds), [g[k] for k in ("dx", "dw", "dbias", "dstate")])


def test_glu_reference_gradients_match_differences():
    x, wg, wu = _rand(5, 6, seed=1), _rand(4, 6, seed=2), _rand(4, 6, seed=3)
    dy = _rand(5, 4, seed=4)
    g = refs.glu_ref(x, wg, wu, dy)
    _check_differences(lambda *a: (refs.glu_ref(*a)["y"],), [x, wg, wu], (dy,),
                       [g[k] for k in ("dx", "dwg", "dwu")])


# ---- refusals of the C entry points (before any CUDA call) ----

P, Q = ctypes.c_void_p(16), ctypes.c_void_p(32)
BAD = ctypes.c_void_p(24)
BF16, FP32 = _lib.GDN_DTYPE_BF16, _lib.GDN_DTYPE_FP32
INVALID, UNSUPPORTED, OK = _lib.GDN_ERR_INVALID, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_OK


def test_glu_rejects_bad_arguments(lib):
    def fwd(x=P, wg=P, wu=P, h=P, g=None, u=None, M=4, D=64, I=32, dtype=BF16):
        return lib.gdn_glu_fwd(x, wg, wu, h, g, u, M, D, I, dtype, None)
    assert fwd(M=-1) == INVALID and fwd(dtype=5) == INVALID
    assert fwd(x=None) == INVALID and fwd(wg=BAD) == INVALID and fwd(h=BAD) == INVALID
    assert fwd(g=P) == INVALID                       # u missing
    assert fwd(M=65535 * 64 + 1, dtype=FP32) == UNSUPPORTED
    assert fwd(M=65535 * 64 + 1, D=60) == UNSUPPORTED      # no multiple of 8: CUDA cores
    assert fwd(M=(1 << 30) + 1) == UNSUPPORTED
    assert fwd(M=0) == OK and fwd(I=0) == OK

    def bwd(ws=P, n=1 << 20, g=P, dh=P, dx=Q, dwg=Q, dwu=Q, M=4, D=64, I=32, dtype=BF16):
        return lib.gdn_glu_bwd(P, P, P, g, P, dh, dx, dwg, dwu, M, D, I, dtype, ws, n, None)
    need = lib.gdn_glu_bwd_workspace_bytes(4, 64, 32, BF16)
    assert need >= 2 * 4 * 32 * 2
    assert bwd(n=need - 1) == INVALID and bwd(ws=None) == INVALID and bwd(ws=BAD) == INVALID
    assert bwd(g=None) == INVALID and bwd(dh=BAD) == INVALID and bwd(dwu=None) == INVALID
    assert bwd(dx=BAD) == INVALID and bwd(D=-1) == INVALID
    assert bwd(dx=P) == INVALID                      # x itself


def test_scan_rejects_bad_arguments(lib):
    def fwd(x=P, dt=P, A=P, B=P, C=P, D=None, z=None, h0=None, y=P, hT=None, ck=None, b=2, T=5,
            ch=8, N=4, G=1, sp=1, dtype=BF16, ws=None, n=0):
        return lib.gdn_selective_scan_fwd(x, dt, A, B, C, D, z, None, h0, y, hT, ck, b, T, ch, N,
                                          G, sp, dtype, ws, n, None)
    for kw in (dict(T=-1), dict(dtype=9), dict(sp=2), dict(G=0), dict(G=3), dict(x=None),
               dict(A=None), dict(y=None), dict(z=BAD), dict(h0=BAD), dict(hT=BAD), dict(ck=BAD),
               dict(T=(1 << 30) + 1)):
        assert fwd(**kw) == INVALID, kw
    for kw in (dict(N=0), dict(N=65), dict(b=65536)):
        assert fwd(**kw) == UNSUPPORTED, kw
    assert fwd(b=0) == OK and fwd(ch=0) == OK and fwd(T=0) == OK
    # a long row of few channels is cut into chunks and needs room for their states
    need = lib.gdn_selective_scan_workspace_bytes(2, 5000, 8, 4, 1)
    assert need > 0 and lib.gdn_selective_scan_workspace_bytes(2, 5, 8, 4, 1) == 0
    assert fwd(T=5000) == INVALID and fwd(T=5000, ws=P, n=need - 1) == INVALID
    assert fwd(T=5000, ws=BAD, n=need) == INVALID
    assert lib.gdn_selective_scan_checkpoint_bytes(2, 33, 8, 16) == 2 * 3 * 8 * 16 * 4
    assert lib.gdn_selective_scan_checkpoint_bytes(2, 33, 8, 65) == 0

    def bwd(ck=P, dy=P, dA=P, D=None, dD=None, z=None, dz=None, dh0=None, ws=P, n=1 << 24, N=4):
        return lib.gdn_selective_scan_bwd(P, P, P, P, P, D, z, None, ck, dy, None, P, P, dA, P, P,
                                          dD, dz, None, dh0, 2, 5, 8, N, 1, 1, BF16, ws, n, None)
    need = lib.gdn_selective_scan_bwd_workspace_bytes(2, 5, 8, 4, 1)
    for kw in (dict(ck=None), dict(dy=None), dict(dA=None), dict(D=P), dict(dD=P), dict(z=P),
               dict(dz=P), dict(dh0=BAD), dict(ws=None), dict(ws=BAD), dict(n=need - 1)):
        assert bwd(**kw) == INVALID, kw
    assert bwd(N=65) == UNSUPPORTED


def test_conv_bias_and_backward_reject_bad_arguments(lib):
    def fwd(bias=P, C=64):
        return lib.gdn_short_conv_fwd_bias(P, P, bias, None, None, P, 2, 10, C, 4, 1, BF16, None)
    assert fwd(bias=BAD) == INVALID and fwd(C=60) == UNSUPPORTED

    def bwd(x=P, w=P, dy=ctypes.c_void_p(32), ds=None, dx=ctypes.c_void_p(48), dw=P, db=None,
            dst=None, K=4, C=64, ws=P, n=1 << 24):
        return lib.gdn_short_conv_bwd(x, w, None, None, dy, ds, dx, dw, db, dst, 2, 10, C, K, 1,
                                      BF16, ws, n, None)
    need = lib.gdn_short_conv_bwd_workspace_bytes(2, 10, 64, 4)
    assert need > 0 and lib.gdn_short_conv_bwd_workspace_bytes(2, 10, 64, 9) == 0
    for kw in (dict(w=None), dict(dy=None), dict(dx=None), dict(dx=P), dict(dw=None),
               dict(dw=BAD), dict(db=BAD), dict(dst=BAD), dict(ds=BAD), dict(ws=None),
               dict(n=need - 1)):
        assert bwd(**kw) == INVALID, kw
    assert bwd(K=9) == UNSUPPORTED and bwd(C=60) == UNSUPPORTED


# ---- refusals of the Python ops ----

def test_ops_refuse_cpu_tensors_and_types():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_linear_unit(x, torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan(x, x, torch.zeros(8, 2), torch.zeros(2, 3, 2), torch.zeros(2, 3, 2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.short_convolution(x, torch.zeros(4, 8), bias=torch.zeros(8))
    with pytest.raises(TypeError, match="Tensor"):
        ops.gated_linear_unit([1.0], torch.zeros(4, 1), torch.zeros(4, 1))
