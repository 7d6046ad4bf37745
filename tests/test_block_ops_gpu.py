"""The block operators on the GPU against their 64-bit references (block_refs),
at the sizes where they can go wrong: one token, lengths that end inside a
tile, widths that fill no vector, groups, states that pad, batches of none.

Tolerances: a stored value is off by at most half a step of its type (bf16 2^-8,
fp32 2^-24 of it); fp32 arithmetic by a relative error per operation times the
sum of the absolute terms, which the references give."""

import pytest
import torch

import block_refs as refs
from gated_deltanet_jax_b200 import _lib, gated_linear_unit, selective_scan, short_convolution

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp32": 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen) * std


def _f64(t):
    return None if t is None else t.detach().cpu().double()


def _within(out, ref, tol, what):
    out = _f64(out)
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    over = ((out - ref).abs() - tol)
    assert torch.isfinite(out).all(), what
    assert bool((over <= 0).all()), f"{what}: over its bound by {over.max().item():.3e}"


# ---------------------------------------------------------------------------
# gated linear unit
# ---------------------------------------------------------------------------

GLU = [(1, 64, 64), (1, 2048, 136), (2, 256, 96), (3, 40, 24), (7, 250, 66), (33, 128, 200),
       (64, 64, 128), (127, 72, 56), (128, 128, 128), (129, 192, 320), (257, 520, 264),
       (300, 33, 17), (1000, 256, 768), (5, 1600, 4808), (37, 2048, 136), (2, 136, 9600), (4099, 72, 40)]


def _glu_inputs(M, D, I, dtype, dev, seed):
    g = _gen(seed)
    return [t.to(DT[dtype]).to(dev) for t in (_randn(g, M, D), _randn(g, I, D, std=D ** -0.5),
                                              _randn(g, I, D, std=D ** -0.5), _randn(g, M, I))]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M,D,I", GLU)
def test_glu_forward(cuda, dtype, M, D, I):
    x, wg, wu, _ = _glu_inputs(M, D, I, dtype, cuda, M + D)
    h = gated_linear_unit(x, wg, wu)
    assert h.dtype == x.dtype
    a = [_f64(t) for t in (x, wg, wu)]
    _within(h, refs.glu_ref(*a)["y"], refs.glu_bound(*a, HALF[dtype])["y"], "h")
    assert _lib.load().gdn_device_error(0) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M,D,I", GLU)
def test_glu_gradients(cuda, dtype, M, D, I):
    x, wg, wu, dy = _glu_inputs(M, D, I, dtype, cuda, M + I)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    h = gated_linear_unit(*leaves)
    plain = gated_linear_unit(*(t.detach() for t in leaves))
    assert torch.equal(h, plain)                       # keeping g and u changes nothing
    grads = torch.autograd.grad(h, leaves, dy)
    a = [_f64(t) for t in (x, wg, wu)]
    ref, tol = refs.glu_ref(*a, _f64(dy)), refs.glu_bound(*a, HALF[dtype], _f64(dy))
    for k, t in zip(("dx", "dwg", "dwu"), grads):
        _within(t, ref[k], tol[k], k)
        # roundings of single values average out in a norm: five of at most half a
        # step each, and the arithmetic's share.  A running fp32 sum of n terms of
        # size s and random sign: after k of them it is about s sqrt(k), an addition
        # errs by at most 2^-24 of that (over sqrt(3) in the mean square), together
        # s 2^-24 / sqrt(3) sqrt(1 + 2 + .. + n) = s 2^-24 n / sqrt(6) beside a result of
        # s sqrt(n): 2^-24 sqrt(n / 6) of it.  Twice that is allowed.
        n = 2 * I if k == "dx" else M
        off = (_f64(t) - ref[k]).norm() / ref[k].norm()
        assert off <= 5 * HALF[dtype] + 2e-6 + 2.0 ** -23 * (n / 6) ** 0.5, (k, off)
    assert _lib.load().gdn_device_error(0) == 0


# Few tokens on the CUDA cores (one to sixteen at once, widths off a vector and off a
# warp's 128 elements, a last column on its own), each tile, and contractions in parts.
CUDA_CORES = [(1, 129, 7), (1, 300, 1), (2, 7, 9), (3, 1000, 33), (4, 128, 10), (5, 254, 31),
              (8, 131, 6), (9, 300, 5), (16, 6, 50), (17, 2050, 33), (40, 512, 90), (50, 90, 700),
              (20, 41, 3001), (64, 130, 1100), (130, 250, 1030), (700, 260, 300), (5001, 30, 22),
              (513, 1024, 130), (1100, 130, 2100)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M,D,I", CUDA_CORES)
def test_glu_cuda_core_forms(cuda, dtype, M, D, I):
    test_glu_gradients(cuda, dtype, M, D, I)


def test_glu_cuda_core_padding_is_not_read(cuda):
    """Infinities in the rows and columns after a call's tensors do not reach it."""
    for M, D, I in [(3, 132, 6), (9, 130, 5), (70, 36, 33), (300, 260, 70)]:
        x, wg, wu, dy = _glu_inputs(M, D, I, "fp32", cuda, M)
        leaves = []
        for t in (x, wg, wu):
            flat = torch.full((t.numel() + 4096,), float("inf"), device=cuda)
            flat[:t.numel()] = t.reshape(-1)
            leaves.append(flat[:t.numel()].view(t.shape).requires_grad_(True))
        h = gated_linear_unit(*leaves)
        ref = gated_linear_unit(x, wg, wu)
        assert torch.equal(h, ref)
        for t in torch.autograd.grad(h, leaves, dy):
            assert bool(torch.isfinite(t).all())


@pytest.mark.parametrize("std", [0.05, 1.0, 4.0, 30.0])
def test_conv_bf16_silu_keeps_the_bits_of_the_exact_division(cuda, std):
    """The bf16 convolution forms its SiLU with fast instructions where they cannot
    change the rounded result: every output has the bits of the fp32 call (an exact
    division) on the same values, rounded to bf16."""
    g = _gen(int(std * 100))
    for K, bias in ((4, True), (3, False), (1, True)):
        x = _randn(g, 3, 700, 512, std=std).to(torch.bfloat16).to(cuda)
        w = _randn(g, K, 512).to(torch.float32).to(cuda)
        b = _randn(g, 512).to(torch.float32).to(cuda) if bias else None
        y, _ = short_convolution(x, w, bias=b)
        ref, _ = short_convolution(x.float(), w, bias=b)
        assert torch.equal(y, ref.to(torch.bfloat16))


def test_conv_bf16_silu_special_values(cuda):
    """Zeros, the ends of the range, subnormals, infinities and NaN."""
    v = torch.tensor([0.0, -0.0, 1e-38, -1e-38, 1e-40, -1e-40, 3e38, -3e38, -8.0, -7.97, -8.06,
                      -88.0, -100.0, -200.0, 88.0, 200.0, float("inf"), -float("inf"),
                      float("nan"), 1.0], device=cuda).to(torch.bfloat16)
    for shift in range(4):                        # each value beside every other kind
        x = v.roll(shift).repeat(2).view(1, 1, -1).contiguous()
        w = torch.ones(1, x.shape[2], device=cuda)
        y, _ = short_convolution(x, w)
        ref, _ = short_convolution(x.float(), w)
        assert torch.equal(y.view(torch.int16), ref.to(torch.bfloat16).view(torch.int16))


def test_glu_shapes_strides_and_partial_gradients(cuda):
    x, wg, wu, dy = _glu_inputs(24, 64, 96, "bf16", cuda, 5)
    h = gated_linear_unit(x, wg, wu)
    assert torch.equal(gated_linear_unit(x.view(2, 3, 4, 64), wg, wu).view(24, 96), h)
    assert gated_linear_unit(x[0], wg, wu).shape == (96,)
    # a strided x, transposed weights' views, and an unaligned start
    wide = torch.zeros(24, 131, dtype=x.dtype, device=cuda)
    wide[:, 3:67] = x
    assert torch.equal(gated_linear_unit(wide[:, 3:67], wg.t().contiguous().t(), wu), h)
    flat = torch.zeros(24 * 64 + 1, dtype=x.dtype, device=cuda)
    flat[1:] = x.reshape(-1)
    assert torch.equal(gated_linear_unit(flat[1:].view(24, 64), wg, wu, activation="swish"), h)
    # no tokens, no width
    assert gated_linear_unit(x[:0], wg, wu).shape == (0, 96)
    assert gated_linear_unit(x, wg[:0], wu[:0]).shape == (24, 0)
    x0 = x[:0].clone().requires_grad_(True)
    w0 = wg.clone().requires_grad_(True)
    g0 = torch.autograd.grad(gated_linear_unit(x0, w0, wu).sum(), [x0, w0])
    assert g0[0].shape == (0, 64) and float(g0[1].abs().max()) == 0.0
    # gradients of one input alone equal those of all
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    full = torch.autograd.grad(gated_linear_unit(*leaves), leaves, dy)
    for i in range(3):
        args = [t.detach() for t in leaves]
        args[i] = leaves[i]
        (one,) = torch.autograd.grad(gated_linear_unit(*args), [leaves[i]], dy)
        assert torch.equal(one, full[i])
    # the same graph twice
    y = gated_linear_unit(*leaves)
    a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    b = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a, b, full))


def test_glu_saturated_gate(cuda):
    """Gates far on either side: silu is g or 0, nothing overflows."""
    x = torch.ones(4, 64, device=cuda)
    wg = torch.full((64, 64), 3.0, device=cuda)
    wg[::2] *= -1
    wu = torch.full((64, 64), 0.25, device=cuda)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    h = gated_linear_unit(*leaves)
    grads = torch.autograd.grad(h, leaves, torch.ones_like(h))
    ref = refs.glu_ref(*(_f64(t) for t in leaves), torch.ones(4, 64, dtype=torch.float64))
    assert torch.allclose(_f64(h), ref["y"], rtol=1e-5, atol=1e-30)
    for k, g in zip(("dx", "dwg", "dwu"), grads):
        assert torch.isfinite(g).all()
        assert torch.allclose(_f64(g), ref[k], rtol=1e-5, atol=1e-30), k


def test_glu_refusals(cuda):
    x, wg, wu, _ = _glu_inputs(4, 64, 32, "bf16", cuda, 1)
    with pytest.raises(TypeError):
        gated_linear_unit(x, wg.float(), wu)
    with pytest.raises(TypeError):
        gated_linear_unit(x.half(), wg.half(), wu.half())
    with pytest.raises(ValueError, match="activation"):
        gated_linear_unit(x, wg, wu, activation="relu")
    with pytest.raises(ValueError):
        gated_linear_unit(x, wg[:, :32], wu[:, :32])
    with pytest.raises(ValueError):
        gated_linear_unit(x, wg, wu[:16])
    with pytest.raises(ValueError):
        gated_linear_unit(x, wg.cpu(), wu)


# ---------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------

# batch, length, channels, states, groups, full (D, z, dt_bias, initial state)
SCAN = [(1, 1, 8, 16, 1, True), (3, 1, 40, 16, 1, False), (2, 1, 24, 5, 2, True),
        (2, 1, 36, 4, 1, True), (2, 1, 32, 64, 2, True), (2, 2, 32, 16, 1, True),
        (1, 15, 33, 16, 1, True), (2, 16, 64, 16, 2, False), (1, 17, 66, 16, 3, True),
        (2, 33, 40, 3, 1, True), (1, 64, 96, 8, 1, True), (2, 31, 20, 7, 1, False),
        (1, 40, 48, 24, 2, True), (1, 35, 36, 32, 1, True), (1, 23, 40, 64, 1, True),
        (1, 130, 7, 16, 1, True), (2, 200, 64, 16, 1, True), (1, 300, 34, 12, 2, False),
        (1, 700, 40, 16, 1, True), (3, 129, 8, 6, 1, True)]


def _scan_inputs(b, T, ch, N, G, full, dtype, dev, seed):
    g = _gen(seed)
    dt = DT[dtype]
    s = dict(x=_randn(g, b, T, ch).to(dt), dt=_randn(g, b, T, ch, std=0.5).to(dt),
             A=-torch.exp(_randn(g, ch, N, std=0.7)) * 4, B=_randn(g, b, T, G, N).to(dt),
             C=_randn(g, b, T, G, N).to(dt), D=None, z=None, dt_bias=None, initial_state=None)
    if full:
        s.update(D=_randn(g, ch), z=_randn(g, b, T, ch).to(dt),
                 dt_bias=_randn(g, ch) - 3.0, initial_state=_randn(g, b, ch, N))
    s = {k: None if v is None else v.to(dev) for k, v in s.items()}
    return s, _randn(g, b, T, ch).to(dt).to(dev), _randn(g, b, ch, N).to(dev)


def _scan_ref(s, softplus, dy=None, dhT=None, absval=False):
    a = [_f64(s[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")]
    return refs.scan_ref(*a, softplus=softplus, dy=_f64(dy), dhT=_f64(dhT), absval=absval)


def _scan_tol(ref, mag, k, T, ch, rows, half):
    """Decay factors carry 2^-21 each (the exponential's 2^-22 and its argument's
    rounding, |argument| < 100 adding 2^-24 * 100 < 2^-17 only where the factor is
    below e^-8, beside which the term itself vanishes), step sizes 2^-20; a term passes
    at most T of them, then the sums over states, channels (ch) and tokens (rows)."""
    e = 2.0 ** -21 * (T + 8) + 2.0 ** -24 * (64 + ch + rows)
    return half * ref[k].abs() + e * mag[k] + 1e-30


def _names(s):
    return [k for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")
            if s[k] is not None]


GRAD = {"initial_state": "dstate"}


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", SCAN)
def test_scan_forward(cuda, dtype, case):
    b, T, ch, N, G, full = case
    s, _, _ = _scan_inputs(*case, dtype, cuda, T + ch)
    for softplus in (True, False):
        if not softplus:
            s["dt"] = s["dt"].abs()
            s["dt_bias"] = None if s["dt_bias"] is None else s["dt_bias"].abs()
        y, st = selective_scan(**s, dt_softplus=softplus, output_final_state=True)
        assert y.dtype == s["x"].dtype and st.dtype == torch.float32
        ref, mag = _scan_ref(s, softplus), _scan_ref(s, softplus, absval=True)
        _within(y, ref["y"], _scan_tol(ref, mag, "y", T, 0, 0, HALF[dtype]), "y")
        _within(st, ref["state"], _scan_tol(ref, mag, "state", T, 0, 0, HALF["fp32"]), "state")
    y2, none = selective_scan(**s, dt_softplus=False)
    assert none is None and torch.equal(y2, y)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", SCAN)
def test_scan_gradients(cuda, dtype, case):
    b, T, ch, N, G, full = case
    s, dy, dhT = _scan_inputs(*case, dtype, cuda, T + N)
    names = _names(s)
    for k in names:
        s[k].requires_grad_(True)
    y, st = selective_scan(**s, output_final_state=True)
    grads = torch.autograd.grad((y, st), [s[k] for k in names], (dy, dhT), retain_graph=True)
    again = torch.autograd.grad((y, st), [s[k] for k in names], (dy, dhT))
    ref = _scan_ref(s, True, dy, dhT)
    mag = _scan_ref(s, True, dy, dhT, absval=True)
    for k, g, h in zip(names, grads, again):
        key = GRAD.get(k, "d" + k)
        assert g.dtype == s[k].dtype and torch.equal(g, h), k
        half = HALF["bf16"] if g.dtype == torch.bfloat16 else HALF["fp32"]
        _within(g, ref[key], _scan_tol(ref, mag, key, 2 * T, ch, b * T, half), key)


def test_scan_decode_continues_a_prompt(cuda):
    """The prompt in one call, or in pieces, or token by token with the state in
    place: the same outputs and states (within fp32 rounding of the order)."""
    s, _, _ = _scan_inputs(2, 70, 48, 16, 1, True, "fp32", cuda, 3)
    y, st = selective_scan(**s, output_final_state=True)
    S = s.pop("initial_state").clone()
    ys = []
    for lo, hi in ((0, 33), (33, 34), (34, 66)):
        cut = {k: (v[:, lo:hi] if v is not None and v.dim() > 2 else v) for k, v in s.items()}
        yt, out = selective_scan(**cut, initial_state=S, final_state_out=S)
        assert out is S
        ys.append(yt)
    for t in range(66, 70):
        cut = {k: (v[:, t:t + 1] if v is not None and v.dim() > 2 else v) for k, v in s.items()}
        ys.append(selective_scan(**cut, initial_state=S, final_state_out=S)[0])
    assert torch.allclose(torch.cat(ys, 1), y, rtol=2e-5, atol=2e-5)
    assert torch.allclose(S, st, rtol=2e-5, atol=2e-5)


def test_scan_empty_layouts_and_types(cuda):
    s, dy, dhT = _scan_inputs(2, 9, 32, 16, 1, True, "bf16", cuda, 8)
    y, st = selective_scan(**s, output_final_state=True)
    # [B,T,N] projections, and projections cut out of one wide row
    flat = dict(s, B=s["B"][:, :, 0], C=s["C"][:, :, 0])
    assert torch.equal(selective_scan(**flat)[0], y)
    wide = torch.cat([s["x"], s["z"], s["B"][:, :, 0], s["C"][:, :, 0]], -1)
    x, z, B, C = wide.split([32, 32, 16, 16], -1)
    assert torch.equal(selective_scan(**dict(s, x=x, z=z, B=B, C=C))[0], y)
    # no tokens: the state passes through, and its gradient
    cut = {k: (v[:, :0] if v is not None and k in ("x", "dt", "B", "C", "z") else v)
           for k, v in s.items()}
    h0 = s["initial_state"].clone().requires_grad_(True)
    y0, s0 = selective_scan(**dict(cut, initial_state=h0), output_final_state=True)
    assert y0.shape == (2, 0, 32) and torch.equal(s0, h0)
    (g,) = torch.autograd.grad(s0, [h0], dhT)
    assert torch.equal(g, dhT)
    # no rows
    none = {k: (v[:0] if v is not None and (v.dim() > 2) else v) for k, v in s.items()}
    A = s["A"].clone().requires_grad_(True)
    y1, s1 = selective_scan(**dict(none, A=A), output_final_state=True)
    assert y1.shape == (0, 9, 32) and s1.shape == (0, 32, 16)
    assert float(torch.autograd.grad(y1.sum(), [A])[0].abs().max()) == 0.0
    # no channels: nothing reads B and C
    Bg, Cg = (s[k].clone().requires_grad_(True) for k in ("B", "C"))
    y2, s2 = selective_scan(s["x"][..., :0], s["dt"][..., :0], s["A"][:0], Bg, Cg,
                            output_final_state=True)
    assert y2.shape == (2, 9, 0) and s2.shape == (2, 0, 16)
    gB, gC = torch.autograd.grad(y2.sum() + s2.sum(), [Bg, Cg])
    assert float(gB.abs().max()) == 0.0 and float(gC.abs().max()) == 0.0
    # parameters in bf16 give their gradients in bf16; a state alone has gradients too
    Ab = s["A"].bfloat16().requires_grad_(True)
    h0 = s["initial_state"].clone().requires_grad_(True)
    _, st2 = selective_scan(**dict(s, A=Ab, initial_state=h0), output_final_state=True)
    ga, gh = torch.autograd.grad(st2.sum(), [Ab, h0])
    assert ga.dtype == torch.bfloat16 and gh.shape == h0.shape


def test_scan_extreme_steps(cuda):
    """Step sizes from 0 to where the decay underflows, and infinite gates' tails."""
    b, T, ch, N = 1, 20, 32, 16
    s, _, _ = _scan_inputs(b, T, ch, N, 1, False, "fp32", cuda, 2)
    s["dt"] = torch.linspace(-120.0, 60.0, T, device=cuda)[None, :, None].expand(b, T, ch)
    s["z"] = torch.linspace(-200.0, 200.0, ch, device=cuda).expand(b, T, ch)
    y, st = selective_scan(**s, output_final_state=True)
    ref, mag = _scan_ref(s, True), _scan_ref(s, True, absval=True)
    # the gate's own arithmetic: e^-z to 2^-24 * |z|
    tol = _scan_tol(ref, mag, "y", T, 300, 0, HALF["fp32"]) + 1e-6 * mag["y"]
    _within(y, ref["y"], tol, "y")
    _within(st, ref["state"], _scan_tol(ref, mag, "state", T, 300, 0, HALF["fp32"]), "state")


def test_scan_refusals(cuda):
    s, _, _ = _scan_inputs(2, 9, 32, 16, 1, True, "bf16", cuda, 8)
    bad = [(TypeError, dict(dt=s["dt"].float())), (TypeError, dict(x=s["x"].half())),
           (TypeError, dict(B=None)), (ValueError, dict(z=s["z"][:, :5])),
           (ValueError, dict(A=s["A"][:16])), (ValueError, dict(B=s["B"][:, :4])),
           (ValueError, dict(D=s["D"][:16])), (ValueError, dict(dt_bias=s["dt_bias"][None])),
           (ValueError, dict(initial_state=s["initial_state"][:1])),
           (ValueError, dict(final_state_out=s["initial_state"].bfloat16())),
           (ValueError, dict(B=s["B"].expand(2, 9, 3, 16), C=s["C"].expand(2, 9, 3, 16))),
           (_lib.GDNError, dict(A=torch.ones(32, 65, device=cuda), initial_state=None,
                                B=torch.ones(2, 9, 65, device=cuda, dtype=torch.bfloat16),
                                C=torch.ones(2, 9, 65, device=cuda, dtype=torch.bfloat16)))]
    for err, kw in bad:
        with pytest.raises(err):
            selective_scan(**dict(s, **kw))
    A = s["A"].clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        selective_scan(**dict(s, A=A), final_state_out=s["initial_state"])


# ---------------------------------------------------------------------------
# short convolution: bias and gradients
# ---------------------------------------------------------------------------

CONV = [(1, 1, 8, 4), (2, 1, 64, 1), (3, 2, 96, 4), (2, 3, 64, 8), (1, 31, 40, 2), (2, 32, 64, 3),
        (2, 33, 520, 4), (1, 65, 64, 5), (3, 130, 72, 4), (1, 600, 16, 7), (2, 1030, 136, 4)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,C,K", CONV)
@pytest.mark.parametrize("full", [True, False])
def test_conv_gradients(cuda, dtype, B, T, C, K, full):
    g = _gen(T + C + K)
    dt = DT[dtype]
    x, w = _randn(g, B, T, C).to(dt).to(cuda), _randn(g, K, C, std=0.5).to(cuda)
    bias = _randn(g, C).to(cuda) if full else None
    st = _randn(g, B, K - 1, C).to(dt).to(cuda) if full else None
    dy, ds = _randn(g, B, T, C).to(dt).to(cuda), _randn(g, B, K - 1, C).to(dt).to(cuda)
    for act in ("silu", None):
        leaves = [t.requires_grad_(True) for t in (x, w, bias, st) if t is not None]
        y, s = short_convolution(x, w, bias=bias, activation=act, conv_state=st,
                                 output_final_state=True)
        with torch.no_grad():
            y0, s0 = short_convolution(x, w, bias=bias, activation=act, conv_state=st,
                                       output_final_state=True)
        assert torch.equal(y, y0) and torch.equal(s, s0)
        grads = torch.autograd.grad((y, s), leaves, (dy, ds))
        a = [_f64(t) for t in (x, w, bias, st)]
        ref = refs.conv_ref(*a, act=act is not None, dy=_f64(dy), dstate=_f64(ds))
        mag = refs.conv_ref(*a, act=act is not None, dy=_f64(dy), dstate=_f64(ds), absval=True)
        # K + 1 multiply-adds and the sigmoid's dozen operations
        e = 2.0 ** -24 * (K + 16)
        _within(y, ref["y"], HALF[dtype] * ref["y"].abs() + e * (mag["y"] + ref["y"].abs())
                + 1e-30, "y")
        assert torch.equal(_f64(s), ref["state"])
        keys = ["dx", "dw"] + (["dbias", "dstate"] if full else [])
        for k, t in zip(keys, grads):
            half = HALF["bf16"] if t.dtype == torch.bfloat16 else HALF["fp32"]
            terms = B * T if k in ("dw", "dbias") else 0
            tol = half * ref[k].abs() + (e + 2.0 ** -24 * terms) * 2 * mag[k] + 1e-30
            _within(t, ref[k], tol, k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,C,K", [(64, 70, 4160, 4), (40, 150, 2048, 3), (60, 41, 4104, 8)])
def test_conv_gradients_of_long_tiles(cuda, dtype, B, T, C, K):
    """Rows that are one or two tiles each, walked past the copies in flight."""
    test_conv_gradients(cuda, dtype, B, T, C, K, True)


def test_conv_layouts_empty_and_refusals(cuda):
    g = _gen(4)
    x, w = _randn(g, 2, 20, 64).bfloat16().to(cuda), _randn(g, 4, 64).to(cuda)
    dy = _randn(g, 2, 20, 64).bfloat16().to(cuda)
    x1, w1 = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    a = torch.autograd.grad(short_convolution(x1, w1)[0], [x1, w1], dy)
    # the flax layout, a strided x, bf16 weights, a transposed gradient
    w3 = w.reshape(4, 1, 64).clone().requires_grad_(True)
    xs = x.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    b = torch.autograd.grad(short_convolution(xs, w3)[0], [xs, w3],
                            dy.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1].view(4, 64))
    wb = w.bfloat16().requires_grad_(True)
    assert torch.autograd.grad(short_convolution(x, wb)[0], [wb], dy)[0].dtype == torch.bfloat16
    # no tokens: the window passes through
    st = _randn(g, 2, 3, 64).bfloat16().to(cuda).requires_grad_(True)
    y0, s0 = short_convolution(x[:, :0], w1, conv_state=st, output_final_state=True)
    assert y0.shape == (2, 0, 64) and torch.equal(s0, st)
    gs, gw = torch.autograd.grad(s0, [st, w1], dy[:, :3])
    assert torch.equal(gs, dy[:, :3]) and float(gw.abs().max()) == 0.0
    with pytest.raises(ValueError, match="bias"):
        short_convolution(x, w, bias=torch.zeros(32, device=cuda))
    with pytest.raises(NotImplementedError):
        short_convolution(x1, w, final_state_out=torch.empty(2, 3, 64, device=cuda,
                                                             dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="activation"):
        short_convolution(x, w, activation="relu")
