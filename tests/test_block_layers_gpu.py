"""The block operators together, as a model uses them: the model's own modules on
the kernels (ShortConvolution and GatedDeltaNetMLP with gradients), a
state-space mixer with its feed-forward half trained end to end, decoding that
continues a prompt, and the ways a program runs them (captured graphs, other
streams, retained graphs, two calls at once)."""

import pytest
import torch
import torch.nn.functional as F

from gated_deltanet_jax_b200 import (GatedDeltaNetConfig, GatedDeltaNetMLP, ShortConvolution,
                                     _lib, gated_linear_unit, model, ops, selective_scan,
                                     short_convolution)

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float((a.double().cpu() - b.double().cpu()).norm() / b.double().cpu().norm())


class _Calls:
    """Counts calls of an op made through the module that the model uses."""

    def __init__(self, monkeypatch, name):
        self.n, fn = 0, getattr(ops, name)

        def counted(*a, **kw):
            self.n += 1
            return fn(*a, **kw)
        monkeypatch.setattr(model.ops, name, counted)


@pytest.mark.parametrize("shape", [(3, 37, 64), (1, 256), (2, 130, 128)])
def test_mlp_runs_on_the_kernel_and_matches_float64(cuda, monkeypatch, shape):
    calls = _Calls(monkeypatch, "gated_linear_unit")
    torch.manual_seed(0)
    mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=shape[-1])).to(cuda, torch.bfloat16)
    x = torch.randn(*shape, device=cuda).bfloat16().requires_grad_(True)
    y = mlp(x)
    dy = torch.randn_like(y)
    leaves = [x] + list(mlp.parameters())
    grads = torch.autograd.grad(y, leaves, dy)
    assert calls.n == 1
    r = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    z, wg, wu, wd = r
    ref = (F.silu(z @ wg.T) * (z @ wu.T)) @ wd.T
    want = torch.autograd.grad(ref, r, dy.double().cpu())
    # h, y and every gradient rounded to bf16 (2^-8 each at most, less in the norm),
    # up to six roundings on a path
    assert _rel(y, ref) <= 2 * 2.0 ** -8
    for g, w in zip(grads, want):
        assert _rel(g, w) <= 6 * 2.0 ** -8
    with torch.no_grad():
        plain = mlp(x)                       # inference keeps torch's operations ...
        assert calls.n == 1 and _rel(plain, y) <= 4 * 2.0 ** -8
        mlp.fused_inference = True           # ... unless asked
        assert torch.equal(mlp(x), y) and calls.n == 2


def test_mlp_keeps_torch_where_the_kernel_does_not_stand_in(cuda, monkeypatch):
    calls = _Calls(monkeypatch, "gated_linear_unit")
    mlp = GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64)).to(cuda)
    x = torch.randn(5, 64, device=cuda)
    mlp(x)                                                    # fp32: cuBLAS
    with torch.autocast("cuda", torch.bfloat16):
        assert mlp(x).dtype == torch.bfloat16                 # autocast casts the weights
    mlp = mlp.bfloat16()
    seen = []
    hook = mlp.gate_proj.register_forward_hook(lambda m, a, o: seen.append(1))
    mlp(x.bfloat16())
    hook.remove()
    assert seen == [1]                                        # a hook is not skipped
    g = torch.func.grad(lambda v: mlp(v).float().sum())(x.bfloat16())
    assert g.shape == x.shape
    assert calls.n == 0
    mlp(x.bfloat16())
    assert calls.n == 1
    assert GatedDeltaNetMLP(GatedDeltaNetConfig(hidden_size=64))(torch.randn(2, 64)).shape == (2, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [True, False])
def test_short_convolution_module_trains_on_the_kernel(cuda, monkeypatch, dtype, bias):
    calls = _Calls(monkeypatch, "short_convolution")
    torch.manual_seed(1)
    conv = ShortConvolution(64, 4, use_bias=bias).to(cuda, dtype)
    x = torch.randn(2, 75, 64, device=cuda).to(dtype).requires_grad_(True)
    y = conv(x)
    dy = torch.randn_like(y)
    leaves = [x] + list(conv.parameters())
    grads = torch.autograd.grad(y, leaves, dy)
    assert calls.n == 1
    r = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    xp = F.pad(r[0], (0, 0, 3, 0))
    pre = sum(r[1][j] * xp[:, j:j + 75] for j in range(4)) + (r[2] if bias else 0)
    want = torch.autograd.grad(F.silu(pre), r, dy.double().cpu())
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 2e-6
    assert _rel(y, F.silu(pre)) <= tol
    for g, w in zip(grads, want):
        assert g.dtype == dtype and _rel(g, w) <= tol
    # a width that the kernel does not take keeps torch's convolution
    odd = ShortConvolution(30, 4).to(cuda, dtype)
    odd(torch.randn(1, 5, 30, device=cuda, dtype=dtype).requires_grad_(True)).float().sum().backward()
    assert calls.n == 1 and odd.weight.grad is not None


class Mixer(torch.nn.Module):
    """A selective state-space mixer and a gated feed-forward half, plain torch
    projections around the operators."""

    def __init__(self, D, C, N, R, inter, K=4):
        super().__init__()
        lin = lambda i, o: torch.nn.Linear(i, o, bias=False)   # noqa: E731
        self.in_proj, self.x_proj, self.dt_proj = lin(D, 2 * C), lin(C, R + 2 * N), lin(R, C)
        self.out_proj, self.down = lin(C, D), lin(inter, D)
        self.gate, self.up = lin(D, inter), lin(D, inter)
        self.w, self.wb = (torch.nn.Parameter(torch.randn(K, C) * 0.5),
                           torch.nn.Parameter(torch.randn(C) * 0.1))
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1.0, N + 1)).repeat(C, 1))
        self.D = torch.nn.Parameter(torch.ones(C))
        self.dt_bias = torch.nn.Parameter(torch.rand(C) * 3 - 5)
        self.sizes = (C, N, R)

    def forward(self, v, conv_state=None, state=None):
        C, N, R = self.sizes
        x, z = self.in_proj(v).split(C, -1)
        x, conv_state = short_convolution(x, self.w, bias=self.wb, conv_state=conv_state,
                                          output_final_state=True)
        dt, B, Cm = self.x_proj(x).split([R, N, N], -1)
        y, state = selective_scan(x, self.dt_proj(dt), -torch.exp(self.A_log), B, Cm, D=self.D,
                                  z=z, dt_bias=self.dt_bias, initial_state=state,
                                  output_final_state=True)
        v = v + self.out_proj(y)
        return v + self.down(gated_linear_unit(v, self.gate.weight, self.up.weight)), conv_state, state

    def reference(self, v, p):
        """The same in the parameters' type (float64), token by token."""
        C, N, R = self.sizes
        x, z = (v @ p["in_proj.weight"].T).split(C, -1)
        K, T = p["w"].shape[0], v.shape[1]
        xp = F.pad(x, (0, 0, K - 1, 0))
        x = F.silu(sum(p["w"][j] * xp[:, j:j + T] for j in range(K)) + p["wb"])
        dt, B, Cm = (x @ p["x_proj.weight"].T).split([R, N, N], -1)
        delta = F.softplus(dt @ p["dt_proj.weight"].T + p["dt_bias"], threshold=1e9)
        A = -torch.exp(p["A_log"])
        h, ys = 0, []
        for t in range(T):
            h = (torch.exp(delta[:, t, :, None] * A) * h
                 + (delta[:, t] * x[:, t])[..., None] * B[:, t, None, :])
            ys.append((h * Cm[:, t, None, :]).sum(-1) + p["D"] * x[:, t])
        v = v + (torch.stack(ys, 1) * F.silu(z)) @ p["out_proj.weight"].T
        g = F.silu(v @ p["gate.weight"].T) * (v @ p["up.weight"].T)
        return v + g @ p["down.weight"].T


def _mixer(cuda, dtype, seed=0):
    torch.manual_seed(seed)
    m = Mixer(64, 96, 16, 8, 160).to(cuda)
    for n, q in m.named_parameters():
        if n.endswith("weight"):
            q.data = q.data.to(dtype)
    return m


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 6e-2)])
def test_mixer_trains_like_its_definition(cuda, dtype, tol):
    """Output and every parameter's gradient against float64.  bf16: about 15
    rounded tensors on the longest path, 2^-8 each, adding up in squares to 1.5 %
    of a gradient that passes them all, with factors of up to four between where
    terms cancel."""
    m = _mixer(cuda, dtype)
    v = torch.randn(2, 150, 64, device=cuda).to(dtype).requires_grad_(True)
    y, _, _ = m(v)
    dy = torch.randn_like(y)
    names = [n for n, _ in m.named_parameters()]
    leaves = [v] + [q for _, q in m.named_parameters()]
    grads = torch.autograd.grad(y, leaves, dy)
    r = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    ref = m.reference(r[0], dict(zip(names, r[1:])))
    want = torch.autograd.grad(ref, r, dy.double().cpu())
    assert _rel(y, ref) <= tol
    for n, g, w in zip(["v"] + names, grads, want):
        assert _rel(g, w) <= tol, n
    assert _lib.load().gdn_device_error(0) == 0


def test_mixer_decodes_on_from_its_prompt(cuda):
    m = _mixer(cuda, torch.float32, 3)
    v = torch.randn(3, 41, 64, device=cuda)
    with torch.no_grad():
        whole, cs, st = m(v)
        y, c, s = m(v[:, :30])
        out = [y]
        for t in range(30, 41):
            y, c, s = m(v[:, t:t + 1], c, s)
            out.append(y)
    assert _rel(torch.cat(out, 1), whole) <= 1e-5
    assert torch.equal(c.cpu().isfinite(), torch.ones_like(c.cpu(), dtype=torch.bool))
    assert _rel(c, cs) <= 1e-5 and _rel(s, st) <= 1e-5


def test_training_step_captured_and_replayed(cuda):
    """Forward and backward in one captured graph, replayed on new inputs, give the
    eager step's bits; the workspaces belong to the graph."""
    m = _mixer(cuda, torch.bfloat16, 5)
    params = list(m.parameters())
    v = torch.randn(2, 150, 64, device=cuda).bfloat16()
    dy = torch.randn_like(v)

    def step():
        y, _, _ = m(v)
        return (y,) + torch.autograd.grad(y, params, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (1, 2):
        gen = torch.Generator(device=cuda).manual_seed(seed)
        v.copy_(torch.randn(v.shape, device=cuda, generator=gen))
        dy.copy_(torch.randn(v.shape, device=cuda, generator=gen))
        g.replay()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_two_graphs_and_two_streams_do_not_meet(cuda):
    """Two captured calls replayed side by side on two streams, and eager calls on a
    third, each with its own outputs and scratch."""
    gen = torch.Generator(device=cuda).manual_seed(0)
    rn = lambda *s, d=torch.bfloat16: torch.randn(*s, device=cuda, generator=gen).to(d)  # noqa: E731
    sets = []
    for k in range(2):
        x = rn(1, 700, 64)
        s = dict(x=x, dt=rn(1, 700, 64), A=-torch.rand(64, 16, device=cuda) * 4 - 0.1,
                 B=rn(1, 700, 16), C=rn(1, 700, 16))
        glu = (rn(8, 512), rn(192, 512), rn(192, 512))
        sets.append((s, glu))
    want = [(selective_scan(**s)[0], gated_linear_unit(*glu)) for s, glu in sets]
    graphs = []
    for s, glu in sets:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = (selective_scan(**s)[0], gated_linear_unit(*glu))
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = selective_scan(**sets[0][0])[0]
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    assert torch.equal(third, want[0][0])


def test_retained_graph_and_accumulation(cuda):
    """A second backward through a kept graph equals the first, and gradients
    accumulate without touching what was saved."""
    m = _mixer(cuda, torch.float32, 9)
    v = torch.randn(1, 40, 64, device=cuda)
    y, _, _ = m(v)
    loss = y.square().sum()
    loss.backward(retain_graph=True)
    first = [q.grad.clone() for q in m.parameters()]
    loss.backward()
    for q, f in zip(m.parameters(), first):
        assert torch.equal(q.grad, f + f)


# ---------------------------------------------------------------------------
# Offsets past 32 bits: the last rows of tensors of more than 2^31 elements
# against the same rows computed on their own (the same kernels in the same
# order: bf16 results equal up to one rounding)
# ---------------------------------------------------------------------------

def _same(a, b):
    assert a.shape == b.shape and torch.isfinite(a.float()).all()
    assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-3)


@pytest.fixture
def roomy(cuda):
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    yield cuda
    torch.cuda.empty_cache()


def test_conv_past_32_bit_offsets(roomy):
    T, C, tail = 270_000, 8192, 500                      # 2.2e9 elements
    x = torch.randn(1, T, C, device=roomy, dtype=torch.bfloat16)
    dy = torch.randn(1, T, C, device=roomy, dtype=torch.bfloat16)
    w = torch.randn(4, C, device=roomy) * 0.5
    xg = x.requires_grad_(True)
    y, s = short_convolution(xg, w, output_final_state=True)
    (dx,) = torch.autograd.grad(y, [xg], dy)
    x = x.detach()
    win = x[:, T - tail - 3:T - tail].contiguous()
    xt = x[:, -tail:].contiguous().requires_grad_(True)
    yt, st = short_convolution(xt, w, conv_state=win, output_final_state=True)
    (dxt,) = torch.autograd.grad(yt, [xt], dy[:, -tail:].contiguous())
    _same(y[:, -tail:], yt)
    assert torch.equal(s, st)
    _same(dx[:, -tail:], dxt)
    # in place over the whole axis: one tile of all tokens
    S = torch.zeros(1, 3, C, device=roomy, dtype=torch.bfloat16)
    with torch.no_grad():
        y2, _ = short_convolution(x, w, conv_state=S, final_state_out=S)
    assert torch.equal(y2[:, -tail:], y[:, -tail:]) and torch.equal(S, s)


def test_scan_past_32_bit_offsets(roomy):
    T, C, head = 270_000, 8192, 250_000                  # the head ends below 2^31
    mk = lambda *s: torch.randn(*s, device=roomy, dtype=torch.bfloat16)   # noqa: E731
    s = dict(x=mk(1, T, C), dt=mk(1, T, C), B=mk(1, T, 4), C=mk(1, T, 4))
    A = -torch.rand(C, 4, device=roomy) - 0.05
    y, st = selective_scan(A=A, **s, output_final_state=True)
    cut = {k: v[:, :head].contiguous() for k, v in s.items()}
    _, mid = selective_scan(A=A, **cut, output_final_state=True)
    cut = {k: v[:, head:].contiguous() for k, v in s.items()}
    yt, stt = selective_scan(A=A, **cut, initial_state=mid, output_final_state=True)
    _same(y[:, head:], yt)
    assert torch.allclose(st, stt, rtol=1e-4, atol=1e-4)


def test_glu_past_32_bit_offsets(roomy):
    M, D, I, tail = 400_000, 64, 5632, 512               # h has 2.25e9 elements
    x = torch.randn(M, D, device=roomy, dtype=torch.bfloat16).requires_grad_(True)
    wg, wu = (torch.randn(I, D, device=roomy, dtype=torch.bfloat16) * 0.125 for _ in range(2))
    h = gated_linear_unit(x, wg, wu)
    dh = torch.randn(M, I, device=roomy, dtype=torch.bfloat16)
    (dx,) = torch.autograd.grad(h, [x], dh)
    xt = x.detach()[-tail:].clone().requires_grad_(True)
    ht = gated_linear_unit(xt, wg, wu)
    (dxt,) = torch.autograd.grad(ht, [xt], dh[-tail:].clone())
    _same(h[-tail:], ht)
    _same(dx[-tail:], dxt)
    assert _lib.load().gdn_device_error(0) == 0
