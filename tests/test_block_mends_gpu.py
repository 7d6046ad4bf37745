"""Faults that the block operators once had, each with the call that showed it, and
the calls around them.  Tolerances: a stored bf16 value is off by at most 2^-8 of it,
an fp32 one by 2^-24; an fp32 sum of n terms by n 2^-24 of the terms' magnitudes."""

import pytest
import torch
import torch.nn.functional as F

from gated_deltanet_jax_b200 import (GatedDeltaNetConfig, GatedDeltaNetMLP, ShortConvolution, _lib,
                                     chunk_gated_delta_rule, fused_recurrent_gated_delta_rule,
                                     gated_linear_unit, gated_rms_norm, selective_scan,
                                     short_convolution)
from test_block_ops_gpu import GRAD, HALF, _f64, _names, _scan_inputs, _scan_ref, _scan_tol

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


# ---------------------------------------------------------------------------
# gated linear unit: long contractions on the tensor cores
# ---------------------------------------------------------------------------

def _silu_grads(g, u, dh):
    s = torch.sigmoid(g)
    return dh * u * (s * (1 + g * (1 - s))), dh * (g * s)


def _sum_error(out, ref, what):
    """Sums of positive terms: each accumulator takes 32768 of them at most (2^-9), its
    operands are rounded one by one to either side (below 1e-4 of a sum of so many), and
    the result once."""
    off = (out.double() - ref) / ref
    assert float(off.mean().abs()) <= 2.0 ** -9 + 2e-4, (what, off.mean())
    assert float(off.abs().max()) <= 2.0 ** -8 + 2.0 ** -9 + 2e-4, (what, off.abs().max())


@pytest.mark.parametrize("M,D,I", [(32768, 64, 96), (32769, 72, 40), (100_000, 64, 96),
                                   ((1 << 20) + 77, 64, 264)])
def test_glu_weight_gradients_of_many_tokens(cuda, M, D, I):
    """The weights' gradients are sums over the tokens, however many."""
    gen = _gen(cuda, M)
    rand = lambda *s: torch.rand(*s, device=cuda, generator=gen).bfloat16()   # noqa: E731
    x, dh = rand(M, D), rand(M, I)
    wg, wu = ((rand(I, D) * 0.02).requires_grad_(True) for _ in range(2))
    dg, du = torch.autograd.grad(gated_linear_unit(x, wg, wu), [wg, wu], dh)
    xd = x.double()
    a, b = _silu_grads(xd @ wg.detach().double().T, xd @ wu.detach().double().T, dh.double())
    _sum_error(dg, a.T @ xd, "dwg")
    _sum_error(du, b.T @ xd, "dwu")
    assert _lib.load().gdn_device_error(0) == 0


@pytest.mark.parametrize("M,D,I", [(3, 64, 70_000), (300, 72, 40_000)])
def test_glu_input_gradient_of_many_columns(cuda, M, D, I):
    """dx is one sum over both projections' columns."""
    gen = _gen(cuda, I)
    rand = lambda *s: torch.rand(*s, device=cuda, generator=gen).bfloat16()   # noqa: E731
    x, dh = rand(M, D).requires_grad_(True), rand(M, I)
    wg, wu = rand(I, D) * 0.02, rand(I, D) * 0.02
    (dx,) = torch.autograd.grad(gated_linear_unit(x, wg, wu), [x], dh)
    xd, gd, ud = x.detach().double(), wg.double(), wu.double()
    a, b = _silu_grads(xd @ gd.T, xd @ ud.T, dh.double())
    _sum_error(dx, a @ gd + b @ ud, "dx")
    assert _lib.load().gdn_device_error(0) == 0


def test_glu_inputs_wider_than_the_tensor_core_form(cuda):
    """D past 131072 runs on the CUDA cores."""
    gen = _gen(cuda, 1)
    D = 131072 + 8
    x = torch.rand(3, D, device=cuda, generator=gen).bfloat16()
    w = (torch.rand(2, 16, D, device=cuda, generator=gen) * 1e-5).bfloat16()
    h = gated_linear_unit(x, w[0], w[1])
    g, u = x.double() @ w[0].double().T, x.double() @ w[1].double().T
    _sum_error(h, g * torch.sigmoid(g) * u, "h")


FORMS = [(5, 256, 328), (64, 512, 136), (300, 256, 328), (1100, 72, 264), (300, 130, 66),
         (7, 250, 66)]   # few tokens, tiles of CTA pairs, CUDA cores


@pytest.mark.parametrize("M,D,I", FORMS)
def test_glu_bf16_gradients_carry_two_roundings(cuda, M, D, I):
    """A gradient is rounded once itself and once through dg or du, the products' bf16
    operands.  Roundings of one spread (relative, between 0.39 and 0.43 of 2^-8 in the
    mean square for values of such distributions) make 1.42 of one at most 1.5."""
    gen = _gen(cuda, M + I)
    rn = lambda *s: torch.randn(*s, device=cuda, generator=gen)   # noqa: E731
    x, dh = rn(M, D).bfloat16(), rn(M, I).bfloat16()
    wg, wu = ((rn(I, D) * D ** -0.5).bfloat16() for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    got = torch.autograd.grad(gated_linear_unit(*leaves), leaves, dh)
    xd, gd, ud = (t.detach().double() for t in leaves)
    a, b = _silu_grads(xd @ gd.T, xd @ ud.T, dh.double())
    for out, ref in zip(got, (a @ gd + b @ ud, a.T @ xd, b.T @ xd)):
        once = (ref.bfloat16().double() - ref).norm()
        assert float((out.double() - ref).norm() / once) <= 1.5


@pytest.mark.parametrize("M,D,I", FORMS)
def test_glu_projections_kept_in_either_type(cuda, M, D, I):
    """The library's two forms: g and u in fp32 are the fp32 sums, in bf16 those rounded
    once; h is the same, and the gradients are the same but for their roundings."""
    lib = _lib.load()
    gen = _gen(cuda, M)
    rn = lambda *s: torch.randn(*s, device=cuda, generator=gen)   # noqa: E731
    x, dh = rn(M, D).bfloat16(), rn(M, I).bfloat16()
    wg, wu = ((rn(I, D) * D ** -0.5).bfloat16() for _ in range(2))
    st = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(lib.gdn_glu_bwd_workspace_bytes(M, D, I, _lib.GDN_DTYPE_BF16),
                     dtype=torch.uint8, device=cuda)
    p = lambda *ts: [t.data_ptr() for t in ts]   # noqa: E731
    out = {}
    for kept, dt in ((_lib.GDN_DTYPE_FP32, torch.float32), (_lib.GDN_DTYPE_BF16, torch.bfloat16)):
        h = torch.empty(M, I, device=cuda, dtype=torch.bfloat16)
        flat = torch.full((2, (M * I + 64) // 64 * 64), 3.0, device=cuda, dtype=dt)
        g, u = flat[0, :M * I].view(M, I), flat[1, :M * I].view(M, I)
        grads = [torch.empty_like(t) for t in (x, wg, wu)]
        assert lib.gdn_glu_fwd_kept(*p(x, wg, wu, h, g, u), M, D, I, 1, kept, st) == 0
        assert lib.gdn_glu_bwd_kept(*p(x, wg, wu, g, u, dh, *grads), M, D, I, 1, kept, *p(ws),
                                    ws.numel(), st) == 0
        assert bool((flat[:, M * I:] == 3.0).all())
        out[dt] = [h, g, u] + grads
    a, b = out[torch.float32], out[torch.bfloat16]
    assert torch.equal(a[0], b[0])
    assert torch.equal(a[1].bfloat16(), b[1]) and torch.equal(a[2].bfloat16(), b[2])
    # (an accumulator's step of 16 terms drops a last place, 2^-23, of it at most)
    assert _rel(a[1], x.double() @ wg.double().T) <= (D / 16 + 8) * 2.0 ** -23
    for s, t in zip(a[3:], b[3:]):
        assert _rel(t, s) <= 5 * 2.0 ** -8
    # the calls without a type keep x's
    h, g, u = (torch.empty_like(t) for t in b[:3])
    assert lib.gdn_glu_fwd(*p(x, wg, wu, h, g, u), M, D, I, 1, st) == 0
    grads = [torch.empty_like(t) for t in (x, wg, wu)]
    assert lib.gdn_glu_bwd(*p(x, wg, wu, g, u, dh, *grads), M, D, I, 1, *p(ws), ws.numel(), st) == 0
    assert all(torch.equal(s, t) for s, t in zip([h, g, u] + grads, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D,I", [(0, 64, 40), (5, 64, 0), (0, 64, 0), (5, 0, 40), (0, 33, 7),
                                   (5, 33, 0), (0, 64, 5_000_000)])
def test_glu_backward_of_empty_sizes(cuda, dtype, M, D, I):
    """Through the C entry point, with every pointer given: what depends on nothing is
    zero, and nothing else is written."""
    lib = _lib.load()
    n = max(M * D, I * D, 1)
    bufs = [torch.full((n + 64,), 3.0, device=cuda, dtype=dtype) for _ in range(9)]
    x, wg, wu, g, u, dh, dx, dwg, dwu = (t.data_ptr() for t in bufs)
    kind = {torch.bfloat16: _lib.GDN_DTYPE_BF16, torch.float32: _lib.GDN_DTYPE_FP32}[dtype]
    if I > 65535 * 64 and dtype == torch.float32:
        I = 4_000_000
    st = torch.cuda.current_stream().cuda_stream
    rc = lib.gdn_glu_bwd(x, wg, wu, g, u, dh, dx, dwg, dwu, M, D, I, kind, None, 0, st)
    assert rc == _lib.GDN_OK, lib.gdn_last_error()
    for t, k in zip(bufs[6:], (M * D, I * D, I * D)):
        assert float(t[:k].abs().sum()) == 0.0 and bool((t[k:] == 3.0).all())
    assert all(bool((t == 3.0).all()) for t in bufs[:6])


# ---------------------------------------------------------------------------
# selective scan: states without memory, growing states
# ---------------------------------------------------------------------------

def _close(out, ref, tol, what):
    """Within the tolerance, and NaN where the reference is."""
    out = _f64(out)
    assert torch.equal(out.isnan(), ref.isnan()), what
    off = torch.where(ref.isnan(), torch.zeros_like(ref), (out - ref).abs() - tol.nan_to_num(0.0))
    assert bool((off <= 0).all()), (what, off.max())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", [(2, 1, 36, 16, 1, True), (2, 1, 20, 24, 2, True),
                                  (1, 2, 33, 16, 1, True), (2, 15, 40, 4, 1, True),
                                  (2, 16, 40, 8, 1, False), (1, 17, 40, 16, 1, True),
                                  (1, 20, 24, 32, 2, True), (1, 22, 24, 64, 1, True),
                                  (2, 32, 40, 16, 1, True), (3, 33, 40, 16, 1, True),
                                  (1, 300, 34, 12, 2, False), (1, 701, 40, 16, 1, True)])
def test_scan_states_without_memory(cuda, dtype, case):
    """A = -inf: a decay of zero at every length, whatever tile it ends in."""
    b, T, ch, N, G, full = case
    s, dy, dhT = _scan_inputs(*case, dtype, cuda, T + N)
    s["A"][1::5, ::3] = -float("inf")
    y, st = selective_scan(**s, output_final_state=True)          # (one token: the step kernels)
    ref, mag = _scan_ref(s, True, dy, dhT), _scan_ref(s, True, dy, dhT, absval=True)
    assert bool(ref["state"].isfinite().all()) and bool(ref["y"].isfinite().all())
    _close(y, ref["y"], _scan_tol(ref, mag, "y", T, 0, 0, HALF[dtype]), "y")
    _close(st, ref["state"], _scan_tol(ref, mag, "state", T, 0, 0, HALF["fp32"]), "state")
    names = _names(s)
    for k in names:
        s[k].requires_grad_(True)
    out = selective_scan(**s, output_final_state=True)
    _close(out[1], ref["state"], _scan_tol(ref, mag, "state", T, 0, 0, HALF["fp32"]), "state")
    for k, g in zip(names, torch.autograd.grad(out, [s[k] for k in names], (dy, dhT))):
        key = GRAD.get(k, "d" + k)
        half = HALF["bf16"] if g.dtype == torch.bfloat16 else HALF["fp32"]
        _close(g, ref[key], _scan_tol(ref, mag, key, 2 * T, ch, b * T, half), key)


@pytest.mark.parametrize("zero_start", [True, False])
def test_scan_growing_states_in_cut_rows(cuda, zero_start):
    """A > 0 with a chunk's factor (e^128) past fp32's range, where no state is: states
    of zero until the last token, and a tiny one that grows and shrinks again."""
    T, ch, N = 1024, 32, 16
    s, dy, dhT = _scan_inputs(1, T, ch, N, 1, True, "fp32", cuda, 3)
    s.update(dt=torch.zeros_like(s["dt"]), dt_bias=None, A=torch.ones_like(s["A"]))
    assert _lib.load().gdn_selective_scan_workspace_bytes(1, T, ch, N, 1) > 0     # it is cut
    s["A"][:, 1::2] = 0.5
    s["x"][:, :-1] = 0.0
    if zero_start:
        s["initial_state"] = None
        s["dt"] += 1.0
        dy, dhT = dy.clone(), torch.zeros_like(dhT)
        dy[:, 1:] = 0.0                                 # (the adjoint states likewise)
    else:
        s["dt"][:, 128:256] = 1.0
        s["A"][ch // 2:] *= -1.0
        s["initial_state"][:, :ch // 2] *= 1e-30
        s["initial_state"][:, ch // 2:] *= 1e30
        dy, dhT = dy * 1e-36, dhT * 1e-30
    names = _names(s)
    for k in names:
        s[k].requires_grad_(True)
    y, st = selective_scan(**s, dt_softplus=False, output_final_state=True)
    grads = torch.autograd.grad((y, st), [s[k] for k in names], (dy, dhT))
    ref, mag = _scan_ref(s, False, dy, dhT), _scan_ref(s, False, dy, dhT, absval=True)
    for k, t, n, rows in ([("y", y, T, 0), ("state", st, T, 0)]
                          + [(GRAD.get(k, "d" + k), g, 2 * T, T) for k, g in zip(names, grads)]):
        assert float(mag[k].max()) < 1e38                # nothing leaves fp32's range
        _close(t, ref[k], _scan_tol(ref, mag, k, n, ch, rows, HALF["fp32"]) + 1e-36, k)


# ---------------------------------------------------------------------------
# second derivatives and batched gradients
# ---------------------------------------------------------------------------

def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


def _penalty(out, x, params, dy):
    """Gradients of |d <out, dy> / dx|^2 by x and the parameters."""
    (g,) = torch.autograd.grad(out, x, dy, create_graph=True)
    return (g,) + torch.autograd.grad(g.double().square().sum(), [x] + params)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
def test_short_convolution_module_second_derivatives(cuda, dtype, bias):
    """Sums of 12 terms of order one: fp32 to 1e-5 of them; bf16 up to four roundings of
    2^-8 on a path (y's and dx's gradients, weights, the result)."""
    torch.manual_seed(0)
    conv = ShortConvolution(64, 4, use_bias=bias).to(cuda, dtype)
    x = torch.randn(2, 75, 64, device=cuda).to(dtype).requires_grad_(True)
    y = conv(x)
    dy = torch.randn_like(y)
    (plain,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    params = list(conv.parameters())
    got = _penalty(y, x, params, dy)
    assert torch.equal(got[0], plain)                  # the kernel's gradient, with a graph
    r = [t.detach().double().requires_grad_(True) for t in [x] + params]
    xp = F.pad(r[0], (0, 0, 3, 0))
    pre = sum(r[1][j] * xp[:, j:j + 75] for j in range(4)) + (r[2] if bias else 0)
    for a, b in zip(got, _penalty(F.silu(pre), r[0], r[1:], dy.double())):
        assert _rel(a, b) <= (1e-5 if dtype == torch.float32 else 4 * 2.0 ** -8)


@pytest.mark.parametrize("shape", [(5, 64), (2, 130, 64)])
def test_mlp_module_second_derivatives(cuda, shape):
    """bf16 throughout: ten rounded tensors on the longest path (g, u, h, dh, dg, du, dx,
    its gradient, two products of it), 2^-8 each at most."""
    torch.manual_seed(0)
    mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64)).to(cuda, torch.bfloat16)
    x = torch.randn(*shape, device=cuda).bfloat16().requires_grad_(True)
    y = mlp(x)
    dy = torch.randn_like(y)
    (plain,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    params = list(mlp.parameters())
    got = _penalty(y, x, params, dy)
    assert torch.equal(got[0], plain)
    r = [t.detach().double().requires_grad_(True) for t in [x] + params]
    z, wg, wu, wd = r
    ref = (F.silu(z @ wg.T) * (z @ wu.T)) @ wd.T
    for a, b in zip(got, _penalty(ref, z, r[1:], dy.double())):
        assert _rel(a, b) <= 10 * 2.0 ** -8


def test_sum_of_outputs_keeps_its_graph(cuda):
    """The incoming gradient is a constant here, and the result still has a graph."""
    torch.manual_seed(0)
    conv = ShortConvolution(64, 4).to(cuda)
    mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64)).to(cuda, torch.bfloat16)
    for m, x in ((conv, torch.randn(2, 9, 64, device=cuda)),
                 (mlp, torch.randn(9, 64, device=cuda).bfloat16())):
        x.requires_grad_(True)
        (g,) = torch.autograd.grad(m(x).sum(), x, create_graph=True)
        assert g.requires_grad
        assert float(torch.autograd.grad(g.float().square().sum(), x)[0].norm()) > 0


def test_batched_gradients(cuda):
    torch.manual_seed(0)
    conv = ShortConvolution(64, 4).to(cuda)
    x = torch.randn(2, 9, 64, device=cuda, requires_grad=True)
    y = conv(x)
    d = torch.randn(3, *y.shape, device=cuda)
    got = torch.autograd.grad(y, (x, conv.weight), d, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(y, (x, conv.weight), d[i], retain_graph=True)):
            assert _rel(a[i], b) <= 1e-5
    w = [torch.randn(96, 64, device=cuda, requires_grad=True) for _ in range(2)]
    v = torch.randn(7, 64, device=cuda, requires_grad=True)
    h = gated_linear_unit(v, *w)
    d = torch.randn(3, *h.shape, device=cuda)
    got = torch.autograd.grad(h, [v] + w, d, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(h, [v] + w, d[i], retain_graph=True)):
            assert _rel(a[i], b) <= 1e-5


def test_scan_second_derivatives_raise(cuda):
    s, dy, dhT = _scan_inputs(2, 20, 40, 16, 1, True, "bf16", cuda, 1)
    names = _names(s)
    for k in names:
        s[k].requires_grad_(True)
    out = selective_scan(**s, output_final_state=True)
    leaves = [s[k] for k in names]
    plain = torch.autograd.grad(out, leaves, (dy, dhT), retain_graph=True)
    kept = torch.autograd.grad(out, leaves, (dy, dhT), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))
    with pytest.raises(NotImplementedError, match="second"):
        torch.autograd.grad(kept[0].float().sum(), leaves)
    with pytest.raises(NotImplementedError, match="batched"):
        torch.autograd.grad(out[0], leaves, dy[None], is_grads_batched=True)


def test_strided_and_unaligned_inputs_keep_their_gradients(cuda):
    """Inputs that are copied for the kernels: gradients of the originals' layout and type."""
    torch.manual_seed(0)
    base = torch.randn(2, 21, 131, device=cuda).bfloat16().requires_grad_(True)
    w = torch.randn(4, 64, device=cuda).bfloat16().requires_grad_(True)
    y, _ = short_convolution(base[..., 3:67], w)
    dy = torch.randn_like(y)
    gx, gw = torch.autograd.grad(y, [base, w], dy)
    x2, w2 = (t.detach().clone().requires_grad_(True) for t in (base[..., 3:67], w.float()))
    hx, hw = torch.autograd.grad(short_convolution(x2, w2)[0], [x2, w2], dy)
    assert torch.equal(gx[..., 3:67], hx) and float(gx[..., 67:].abs().max()) == 0.0
    assert torch.equal(gw, hw.bfloat16())


# ---------------------------------------------------------------------------
# forward mode
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_raises(cuda, grad):
    """No operator gives an output without the tangent that it should have; the modules'
    torch routes keep theirs."""
    fw = torch.autograd.forward_ad
    x = torch.randn(1, 9, 64, device=cuda)
    w, A, B = torch.randn(64, 64, device=cuda), -torch.rand(64, 16, device=cuda), x[..., :16]
    q, b = x.view(1, 9, 1, 64), x[..., :1]
    with fw.dual_level(), torch.set_grad_enabled(grad):
        d = fw.make_dual(x, torch.randn_like(x))
        calls = [lambda: gated_linear_unit(d, w, w),
                 lambda: selective_scan(x, d, A, B, B),
                 lambda: selective_scan(x, x, A, d[..., :16], B),
                 lambda: short_convolution(d, w[:4]), lambda: gated_rms_norm(d),
                 lambda: chunk_gated_delta_rule(d.view(1, 9, 1, 64), q, q, b, b),
                 lambda: fused_recurrent_gated_delta_rule(q, q, d.view(1, 9, 1, 64), b, b)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        gated_linear_unit(x, w, w)                      # no tangent: as always
        conv = ShortConvolution(64, 4).to(cuda)
        if grad:
            assert fw.unpack_dual(conv(d)).tangent is not None
        mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64)).to(cuda)
        assert fw.unpack_dual(mlp(d)).tangent is not None


# ---------------------------------------------------------------------------
# short convolution: decoding over a module's parameters
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 2, 40])
def test_conv_decodes_in_place_over_parameters(cuda, T):
    """Weights that require grad, outside no_grad, with the window updated in place: the
    values of a call without gradients, and the weights' gradients of one out of place."""
    gen = _gen(cuda, T)
    rn = lambda *s: torch.randn(*s, device=cuda, generator=gen)   # noqa: E731
    w, bias = torch.nn.Parameter(rn(4, 64)), torch.nn.Parameter(rn(64))
    x = [rn(2, T, 64).bfloat16() for _ in range(3)]
    dy = rn(2, T, 64).bfloat16()
    start = rn(2, 3, 64).bfloat16()
    S, P, state = start.clone(), start.clone(), start
    ys, zs = [], []
    for v in x:
        y, out = short_convolution(v, w, bias=bias, conv_state=S, final_state_out=S)
        assert out is S and not S.requires_grad
        with torch.no_grad():
            plain, _ = short_convolution(v, w, bias=bias, conv_state=P, final_state_out=P)
        z, state = short_convolution(v, w, bias=bias, conv_state=state, output_final_state=True)
        state = state.detach()
        assert torch.equal(y, plain) and torch.equal(S, P) and torch.equal(S, state)
        ys.append(y)
        zs.append(z)
    for y, z in zip(ys, zs):                           # (the windows have moved on since)
        for a, b in zip(torch.autograd.grad(y, [w, bias], dy), torch.autograd.grad(z, [w, bias], dy)):
            assert torch.equal(a, b)
    for bad in (dict(x=x[0].clone().requires_grad_(True)),
                dict(x=x[0], conv_state=start.clone().requires_grad_(True))):
        with pytest.raises(NotImplementedError, match="final_state_out"):
            short_convolution(bad.pop("x"), w, bias=bias, final_state_out=S, **bad)


# ---------------------------------------------------------------------------
# short convolution: many rows, long rows
# ---------------------------------------------------------------------------

def test_short_convolution_module_trains_on_many_rows(cuda):
    """More rows than the kernels' grid takes keep torch's convolution."""
    torch.manual_seed(0)
    conv = ShortConvolution(8, 4).to(cuda)
    x = torch.randn(65537, 3, 8, device=cuda, requires_grad=True)
    y = conv(x)
    y.sum().backward()
    few = x.detach()[-2:].clone().requires_grad_(True)
    z = conv(few)
    (g,) = torch.autograd.grad(z.sum(), few)
    assert torch.allclose(y[-2:], z, atol=1e-5) and torch.allclose(x.grad[-2:], g, atol=1e-5)


def _room(gb):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB of device memory")


@pytest.mark.parametrize("T,grad,gb", [((1 << 30) + 77, True, 90), ((1 << 31) - 64, False, 90)])
def test_conv_rows_past_2_30_tokens(cuda, T, grad, gb):
    """The last tokens of a row as long as the kernels take, against those on their own."""
    _room(gb)
    tail = 100
    x = torch.randn(1, T, 8, device=cuda, dtype=torch.bfloat16).requires_grad_(grad)
    w = torch.randn(4, 8, device=cuda) * 0.5
    y, s = short_convolution(x, w, output_final_state=True)
    cut = x.detach()[:, -tail:].clone().requires_grad_(grad)
    yt, st = short_convolution(cut, w, conv_state=x.detach()[:, -tail - 3:-tail].clone(),
                               output_final_state=True)
    assert torch.equal(y[:, -tail:], yt) and torch.equal(s, st)
    if grad:
        dy = torch.randn_like(y)
        (dx,) = torch.autograd.grad(y, x, dy)
        (dt,) = torch.autograd.grad(yt, cut, dy[:, -tail:].clone())
        assert torch.equal(dx[:, -tail:], dt)
    del x, y
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# the modules under torch's tracing and dispatch modes
# ---------------------------------------------------------------------------

def test_modules_trace_to_torch_operations(cuda):
    """A traced module is a graph of torch's operations that another input, and another
    program, can run."""
    from torch.utils.flop_counter import FlopCounterMode
    torch.manual_seed(0)
    mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64)).to(cuda, torch.bfloat16)
    conv = ShortConvolution(64, 4).to(cuda)
    for m, x, shape in ((mlp, torch.randn(5, 64, device=cuda).bfloat16(), (9, 64)),
                        (conv, torch.randn(2, 9, 64, device=cuda), (2, 9, 64))):
        traced = torch.jit.trace(m, x)
        assert "PythonOp" not in str(traced.inlined_graph)
        v = torch.randn(*shape, device=cuda).to(x.dtype)
        with torch.no_grad():
            assert torch.allclose(traced(v).float(), m(v).float(), rtol=3e-2, atol=3e-2)
        with FlopCounterMode(display=False) as counted:
            m(x)
        assert counted.get_total_flops() > 0


# ---------------------------------------------------------------------------
# sizes past 32 bits
# ---------------------------------------------------------------------------

def test_sizes_past_32_bits_are_refused(cuda):
    """They once arrived as their low halves, and outputs came back unwritten."""
    _room(80)
    big = (1 << 32) + 5
    w = torch.ones(8, 8, device=cuda, dtype=torch.bfloat16)
    x = torch.empty(big, 8, device=cuda, dtype=torch.bfloat16)
    for call in (lambda: gated_linear_unit(x, w, w),
                 lambda: gated_linear_unit(x.view(1, big, 8), w, w),
                 lambda: gated_linear_unit(x[:2], x, x),
                 lambda: short_convolution(x[None], w[:4]),
                 lambda: short_convolution(x[:, None], w[:4]),
                 lambda: short_convolution(x[:, None, :0], w[:4, :0])):
        with pytest.raises(ValueError, match="too large"):
            call()
    A = torch.ones(1, 1, device=cuda)
    v = x.view(-1)[:big].view(1, big, 1)
    with pytest.raises(ValueError, match="too large"):
        selective_scan(v, v, A, v, v)
    del x, v
    torch.cuda.empty_cache()
