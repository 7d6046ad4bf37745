"""Cases for timing and checking the block operators: the gated linear unit of the
feed-forward half, the selective state-space scan, and the short causal convolution
that feeds it.

``run`` makes one pass, either through this package's operators (``own`` true) or in
a plain form made of elementary torch operations in 32 bits.  ``exact`` gives the
same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    glu = dict(op="glu", hidden=2048, inter=5632)          # the default model's MLP widths
    scan = dict(op="scan", channels=4096, states=16, groups=1, gate=True, start=False)
    conv = dict(op="conv", channels=4096, kernel=4, bias=True, start=False)
    return [
        # one sequence decoding: the two projections' weights are streamed once
        dict(glu, name="glu_token", tokens=1, dtype="bf16", train=False),
        # a decode batch of an odd number of sequences
        dict(glu, name="glu_decode_batch", tokens=37, dtype="bf16", train=False),
        # the model's prompt batch: 8 rows of 2048 tokens
        dict(glu, name="glu_prompt", tokens=16384, dtype="bf16", train=False),
        # a training batch of 4 rows whose length fills no tile
        dict(glu, name="glu_train", tokens=4 * 2050, dtype="bf16", train=True),
        # a small model trained in fp32
        dict(op="glu", name="glu_train_fp32", hidden=256, inter=768, tokens=513, dtype="fp32",
             train=True),
        # one decode step of 64 sequences, their states kept between calls
        dict(scan, name="scan_step", batch=64, length=1, dtype="bf16", train=False, start=True),
        # the prompts of 8 sequences, their last states kept for decoding
        dict(scan, name="scan_prompt", batch=8, length=2048, dtype="bf16", train=False),
        # a training batch, narrower
        dict(scan, name="scan_train", batch=4, length=2048, channels=2048, dtype="bf16",
             train=True),
        # one long ungated sequence in fp32 continued from a state: few rows, a long axis
        dict(scan, name="scan_long_fp32", batch=1, length=16387, channels=1024, dtype="fp32",
             train=False, gate=False, start=True),
        # one decode step of the convolution, its window kept between calls
        dict(conv, name="conv_step", batch=64, length=1, dtype="bf16", train=False, start=True),
        # the convolution in a training batch
        dict(conv, name="conv_train", batch=8, length=2048, dtype="bf16", train=True),
        # fp32, an odd length, continued from a window, another kernel size
        dict(conv, name="conv_train_fp32", batch=3, length=1031, channels=640, kernel=3,
             dtype="fp32", train=True, start=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["glu", "scan", "conv"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.5
    if op == "glu":
        # widths in steps of 8 (what models use); tokens of any number
        while True:
            c = dict(op=op, hidden=8 * _log(rng, 8, 512), inter=8 * _log(rng, 12, 1536),
                     tokens=_log(rng, 1, 16384), dtype=dtype, train=train)
            cost = c["hidden"] * c["inter"] * c["tokens"] * (3 if train else 1)
            if cost <= 16384 * 2048 * 5632 // (20 if dtype == "fp32" else 1):
                return c
    start = rng.random() < 0.5
    if op == "scan":
        while True:
            length = 1 if rng.random() < 0.2 else _log(rng, 2, 16384)
            groups = rng.choice([1, 1, 2])
            c = dict(op=op, batch=_log(rng, 1, 64), length=length,
                     channels=8 * groups * _log(rng, 8, 512 // groups),
                     states=rng.choice([4, 8, 16, 16, 16, 24, 32, 64]), groups=groups,
                     gate=rng.random() < 0.7, start=start, dtype=dtype, train=train)
            cost = c["batch"] * length * c["channels"] * c["states"] * (4 if train else 1)
            if cost <= 8 * 2048 * 4096 * 16:
                return c
    while True:
        c = dict(op=op, batch=_log(rng, 1, 64), length=_log(rng, 1, 16384),
                 channels=8 * _log(rng, 8, 512), kernel=rng.choice([2, 3, 4, 4, 5]),
                 bias=rng.random() < 0.5, start=start, dtype=dtype, train=train)
        cost = c["batch"] * c["length"] * c["channels"] * _BYTES[dtype]
        if cost <= 8 * 2048 * 4096 * 2:
            return c


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "glu":
        n, d, i = case["tokens"], case["hidden"], case["inter"]
        if not case["train"]:
            return {"bytes": e * (n * d + 2 * d * i + n * i), "flops": 4 * n * d * i}
        # + dh read, dx and the weights' gradients written; two products each for them
        return {"bytes": e * (2 * n * d + 4 * d * i + 2 * n * i), "flops": 12 * n * d * i}
    b, t, c = case["batch"], case["length"], case["channels"]
    if case["op"] == "scan":
        n, g = case["states"], case["groups"]
        rows, small = b * t * c, b * t * g * n
        state = 4 * b * c * n
        par = 4 * (c * n + 2 * c)
        inp = e * (rows * (2 + case["gate"]) + 2 * small) + par + state * case["start"]
        out = e * rows + state
        # per state and token: the decay's argument and exponential, the input's product,
        # the update and the read-out (two each)
        flops = 7 * rows * n
        if case["train"]:
            out += e * (rows * (2 + case["gate"]) + 2 * small) + par + state * case["start"]
            inp += e * rows + state
            flops += 14 * rows * n
        return {"bytes": inp + out, "flops": flops}
    k = case["kernel"]
    win = e * b * (k - 1) * c
    w = 4 * c * (k + case["bias"])
    total = 2 * e * b * t * c + w + win * (1 + case["start"])
    flops = (2 * k + 4) * b * t * c
    if case["train"]:
        total += 2 * e * b * t * c + w + win * (1 + case["start"])
        flops += (4 * k + 10) * b * t * c
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _leaf(s, name, t):
    if t is not None and s["train"]:
        t.requires_grad_(True)
    s[name] = t


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, device=dev, generator=gen) * std).to(dtype)

    s = dict(op=case["op"], train=case["train"])
    if case["op"] == "glu":
        n, d, i = case["tokens"], case["hidden"], case["inter"]
        _leaf(s, "x", normal(n, d))
        _leaf(s, "wg", normal(i, d, std=d ** -0.5))
        _leaf(s, "wu", normal(i, d, std=d ** -0.5))
        if case["train"]:
            s["dy"] = normal(n, i)
        return s
    b, t, c = case["batch"], case["length"], case["channels"]
    f32 = torch.float32
    if case["op"] == "conv":
        k = case["kernel"]
        _leaf(s, "x", normal(b, t, c))
        _leaf(s, "w", normal(k, c, std=k ** -0.5, dtype=f32))
        _leaf(s, "bias", normal(c, std=0.2, dtype=f32) if case["bias"] else None)
        _leaf(s, "state", normal(b, k - 1, c) if case["start"] else None)
        if case["train"]:
            s["dy"], s["dstate"] = normal(b, t, c), normal(b, k - 1, c)
        else:
            s["out"] = torch.empty(b, k - 1, c, device=dev, dtype=dt)
        return s
    n, g = case["states"], case["groups"]
    _leaf(s, "x", normal(b, t, c))
    _leaf(s, "dt", normal(b, t, c, std=0.5))
    # decay rates -1 .. -states as such layers start from, moved a little
    A = -torch.arange(1, n + 1, device=dev, dtype=f32).expand(c, n)
    _leaf(s, "A", (A * torch.exp(normal(c, n, std=0.1, dtype=f32))).contiguous())
    _leaf(s, "B", normal(b, t, g, n))
    _leaf(s, "C", normal(b, t, g, n))
    _leaf(s, "D", 1 + normal(c, std=0.1, dtype=f32))
    _leaf(s, "z", normal(b, t, c) if case["gate"] else None)
    # step sizes log-uniform in [1e-3, 0.1] through the inverse softplus
    step = torch.rand(c, device=dev, generator=gen) * math.log(100.0) + math.log(1e-3)
    step = torch.exp(step)
    _leaf(s, "dt_bias", step + torch.log(-torch.expm1(-step)))
    _leaf(s, "state", normal(b, c, n, std=0.2, dtype=f32) if case["start"] else None)
    if case["train"]:
        s["dy"], s["dstate"] = normal(b, t, c), normal(b, c, n, std=0.2, dtype=f32)
    else:
        s["out"] = torch.empty(b, c, n, device=dev, dtype=f32)
    return s


_LEAVES = {"glu": ("x", "wg", "wu"), "conv": ("x", "w", "bias", "state"),
           "scan": ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _own_pass(s) if own else _plain_pass(s)


def _own_pass(s):
    from gated_deltanet_jax_b200 import gated_linear_unit, selective_scan, short_convolution
    names = [k for k in _LEAVES[s["op"]] if s[k] is not None]
    if s["op"] == "glu":
        y = gated_linear_unit(s["x"], s["wg"], s["wu"])
        if not s["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(names, grads)}}
    keep = dict(output_final_state=True) if s["train"] else dict(final_state_out=s["out"])
    if s["op"] == "conv":
        y, state = short_convolution(s["x"], s["w"], bias=s["bias"], conv_state=s["state"], **keep)
    else:
        y, state = selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                  dt_bias=s["dt_bias"], initial_state=s["state"], **keep)
    if not s["train"]:
        return {"y": y, "state": state}
    grads = torch.autograd.grad((y, state), [s[k] for k in names], (s["dy"], s["dstate"]))
    return {"y": y, "state": state, **{"d" + k: v for k, v in zip(names, grads)}}


def _plain_pass(s):
    with torch.no_grad():
        p = {k: None if s[k] is None else s[k].detach().float() for k in _LEAVES[s["op"]]}
        if s["train"]:
            p["dy"] = s["dy"].float()
            p["dstate"] = s["dstate"].float() if "dstate" in s else None
        out = {"glu": _plain_glu, "conv": _plain_conv, "scan": _plain_scan}[s["op"]](p, s["train"])
        dts = {"y": s["x"].dtype}
        if s["op"] != "glu":
            dts["state"] = torch.float32 if s["op"] == "scan" else s["x"].dtype
        dts.update({"d" + k: s[k].dtype for k in _LEAVES[s["op"]] if s[k] is not None})
        out = {k: v.to(dts[k]) for k, v in out.items() if k in dts}
        if not s["train"] and "state" in out:
            out["state"] = s["out"].copy_(out["state"])
        return out


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _plain_glu(p, train):
    x, wg, wu = p["x"], p["wg"], p["wu"]
    g, u = x @ wg.T, x @ wu.T
    sg = _sigmoid(g)
    out = {"y": g * sg * u}
    if train:
        dg = p["dy"] * u * sg * (1 + g * (1 - sg))
        du = p["dy"] * g * sg
        out.update(dx=dg @ wg + du @ wu, dwg=dg.T @ x, dwu=du.T @ x)
    return out


def _plain_conv(p, train):
    x, w, bias, state = p["x"], p["w"], p["bias"], p["state"]
    (b, t, c), k = x.shape, w.shape[0]
    if state is None:
        state = x.new_zeros(b, k - 1, c)
    xp = torch.cat([state, x], 1)
    win = xp.unfold(1, k, 1)                                # [b, t, c, k]
    pre = (win * w.T).sum(-1)
    if bias is not None:
        pre = pre + bias
    sg = _sigmoid(pre)
    out = {"y": pre * sg, "state": xp[:, t:]}
    if train:
        dpre = p["dy"] * sg * (1 + pre * (1 - sg))
        pad = dpre.new_zeros(b, k - 1, c)
        back = torch.cat([pad, dpre, pad], 1).unfold(1, k, 1)   # [b, t + k - 1, c, k]
        dxp = (back * w.flip(0).T).sum(-1)
        dxp[:, t:] += p["dstate"]
        out.update(dx=dxp[:, k - 1:], dstate=dxp[:, :k - 1], dbias=dpre.sum((0, 1)),
                   dw=(dpre[..., None] * win).sum((0, 1)).T)
    return out


def _linear_recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from zero, by doubling strides."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        if 2 * step < a.shape[1]:
            a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(p, train):
    x, A = p["x"], p["A"]
    (b, t, c), n, g = x.shape, A.shape[1], p["B"].shape[2]
    wide = lambda v: v.repeat_interleave(c // g, 2)         # noqa: E731  [b, t, c, n]
    pre = p["dt"] + p["dt_bias"]
    delta = _softplus(pre)
    dA = delta[..., None] * A
    a = torch.exp(dA)
    inp = (delta * x)[..., None] * wide(p["B"])
    if p["state"] is not None:
        inp[:, 0] += a[:, 0] * p["state"]
    h = _linear_recurrence(a, inp)
    del inp
    core = (h * wide(p["C"])).sum(-1) + p["D"] * x
    out = {"y": core, "state": h[:, -1].clone()}
    if p["z"] is not None:
        sz = _sigmoid(p["z"])
        out["y"] = core * p["z"] * sz
    if not train:
        return out
    dy = p["dy"]
    if p["z"] is not None:
        out["dz"] = dy * core * sz * (1 + p["z"] * (1 - sz))
        dy = dy * p["z"] * sz
    # adjoint states: r_t = C_t dy_t + a_{t+1} r_{t+1}, the last with the state's gradient
    src = wide(p["C"]) * dy[..., None]
    src[:, -1] += p["dstate"]
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    r = _linear_recurrence(nxt.flip(1), src.flip(1)).flip(1)
    del src, nxt
    dB = r * (delta * x)[..., None]
    out["dB"] = dB.view(b, t, g, c // g, n).sum(3)
    dC = h * dy[..., None]
    out["dC"] = dC.view(b, t, g, c // g, n).sum(3)
    del dB, dC
    rb = (r * wide(p["B"])).sum(-1)
    start = torch.zeros_like(h[:, :1]) if p["state"] is None else p["state"][:, None]
    flow = r * a * torch.cat([start, h[:, :-1]], 1)         # r_t a_t h_{t-1}
    out["dA"] = (flow * delta[..., None]).sum((0, 1))
    ddelta = (flow * A).sum(-1) + rb * x
    out["dx"] = rb * delta + p["D"] * dy
    out["dD"] = (dy * x).sum((0, 1))
    out["ddt"] = ddelta * _sigmoid(pre)
    out["ddt_bias"] = out["ddt"].sum((0, 1))
    out["dstate"] = r[:, 0] * a[:, 0]
    return out


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    names = [k for k in _LEAVES[s["op"]] if s[k] is not None]
    v = {k: s[k].detach().double().requires_grad_(s["train"]) for k in names}
    get = v.get
    with torch.set_grad_enabled(s["train"]):
        if s["op"] == "glu":
            outs = [torch.nn.functional.silu(v["x"] @ v["wg"].T) * (v["x"] @ v["wu"].T)]
        elif s["op"] == "conv":
            outs = _exact_conv(v["x"], v["w"], get("bias"), get("state"))
        else:
            outs = _exact_scan(v, get)
    res = dict(zip(("y", "state"), outs))
    if s["train"]:
        cot = [s[k].double() for k in ("dy", "dstate") if k in s]
        grads = torch.autograd.grad(outs, [v[k] for k in names], cot)
        res.update({"d" + k: g for k, g in zip(names, grads)})
    return {k: r.detach() for k, r in res.items()}


def _exact_conv(x, w, bias, state):
    k, c = w.shape
    if state is None:
        state = torch.zeros(x.shape[0], k - 1, c, dtype=x.dtype, device=x.device)
    xp = torch.cat([state, x], 1)
    pre = sum(w[j] * xp[:, j:j + x.shape[1]] for j in range(k))
    if bias is not None:
        pre = pre + bias
    return [torch.nn.functional.silu(pre), xp[:, x.shape[1]:]]


def _exact_scan(v, get):
    x, A = v["x"], v["A"]
    (b, t, c), g = x.shape, v["B"].shape[2]
    delta = torch.nn.functional.softplus(v["dt"] + v["dt_bias"], threshold=1e9)
    h = get("state")
    if h is None:
        h = torch.zeros(b, c, A.shape[1], dtype=x.dtype, device=x.device)
    ys = []
    # unbind: one backward node for all steps
    for d_t, x_t, B_t, C_t in zip(delta.unbind(1), x.unbind(1), v["B"].unbind(1),
                                  v["C"].unbind(1)):
        B_t = B_t.repeat_interleave(c // g, 1)
        C_t = C_t.repeat_interleave(c // g, 1)
        h = torch.exp(d_t[..., None] * A) * h + (d_t * x_t)[..., None] * B_t
        ys.append((h * C_t).sum(-1) + v["D"] * x_t)
    y = torch.stack(ys, 1)
    if get("z") is not None:
        y = y * torch.nn.functional.silu(v["z"])
    return [y, h]
