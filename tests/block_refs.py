"""64-bit references of the block operators (gated linear unit, selective scan,
short convolution) with their gradients written out, and the sums of absolute
terms that bound how far fp32 arithmetic may be off.

Every function takes float64 CPU tensors.  With ``absval`` every term enters by
its absolute value, so that the result bounds the sum of the terms' magnitudes:
an fp32 evaluation whose terms each carry a relative error of at most ``e`` is
within ``e`` times it."""

import torch


def sig(v):
    return torch.sigmoid(v)


def silu(v):
    return v * sig(v)


def dsilu(v):
    return sig(v) * (1 + v * (1 - sig(v)))


def _mag(absval):
    return (lambda t: t.abs()) if absval else (lambda t: t)


def scan_ref(x, dt, A, B, C, D=None, z=None, bias=None, h0=None, softplus=True, dy=None, dhT=None,
             absval=False):
    """y, hT and, with dy, the gradients of every input (dict)."""
    m = _mag(absval)
    b, T, ch = x.shape
    G, N = B.shape[2], A.shape[1]
    pre = dt if bias is None else dt + bias
    delta = torch.nn.functional.softplus(pre, threshold=1e9) if softplus else pre
    a = torch.exp(delta[..., None] * A)                       # [b, T, ch, N], positive
    rep = lambda v: m(v).repeat_interleave(ch // G, 2)        # noqa: E731
    Bw, Cw, xm, dm = rep(B), rep(C), m(x), m(delta)
    h = torch.zeros(b, ch, N, dtype=x.dtype) if h0 is None else m(h0)
    prev, hs = [], []
    for t in range(T):
        prev.append(h)
        h = a[:, t] * h + (dm[:, t] * xm[:, t])[..., None] * Bw[:, t]
        hs.append(h)
    out = {"state": h}
    if T:
        hs, prev = torch.stack(hs, 1), torch.stack(prev, 1)
    else:
        hs = prev = torch.zeros(b, 0, ch, N, dtype=x.dtype)
    Dm = 0.0 if D is None else m(D)
    core = (hs * Cw).sum(-1) + Dm * xm
    gz = 1.0 if z is None else m(silu(z))
    out["y"] = core * gz
    if dy is None:
        return out
    dyp = m(dy) * gz
    r = torch.zeros(b, ch, N, dtype=x.dtype) if dhT is None else m(dhT)   # a_{t+1} r_{t+1}
    rs = []
    for t in range(T - 1, -1, -1):
        rt = Cw[:, t] * dyp[:, t][..., None] + r
        r = a[:, t] * rt
        rs.append(rt)
    rs = torch.stack(rs[::-1], 1) if T else torch.zeros_like(hs)
    rb = (rs * Bw).sum(-1)
    flow = rs * a * prev
    ddelta = (flow * m(A)).sum(-1) + rb * xm
    dpre = ddelta * (sig(pre) if softplus else 1.0)
    grp = lambda v: v.reshape(b, T, G, ch // G, N).sum(3)     # noqa: E731
    out.update(dx=rb * dm + Dm * dyp, ddt=dpre, dA=(flow * dm[..., None]).sum((0, 1)),
               dB=grp(rs * (dm * xm)[..., None]), dC=grp(hs * dyp[..., None]),
               dD=(dyp * xm).sum((0, 1)), ddt_bias=dpre.sum((0, 1)), dstate=r)
    if z is not None:
        out["dz"] = m(dy) * core * m(dsilu(z))
    return out


def conv_ref(x, w, bias=None, state=None, act=True, dy=None, dstate=None, absval=False):
    """y, the final window and, with dy, the gradients (dict).  The activation
    and its derivative are taken at the signed sum in both forms."""
    m = _mag(absval)
    (b, T, C), K = x.shape, w.shape[0]
    if state is None:
        state = torch.zeros(b, K - 1, C, dtype=x.dtype)
    xp = torch.cat([state, x], 1)
    pre = sum(w[j] * xp[:, j:j + T] for j in range(K))
    pre = pre if bias is None else pre + bias
    mag = sum(m(w[j]) * m(xp[:, j:j + T]) for j in range(K))
    mag = mag if bias is None else mag + m(bias)
    # |silu'| <= 1.1: an error of e in pre is at most 1.1 e in y
    out = {"y": (1.1 * mag if absval else (silu(pre) if act else pre)), "state": xp[:, T:]}
    if dy is None:
        return out
    # |silu''| <= 0.5, so an error of e * mag in pre moves dpre by 0.5 |dy| e mag
    dpre = dy * (dsilu(pre) if act else 1.0)
    if absval:
        dpre = dpre.abs() + 0.5 * dy.abs() * mag + dy.abs()
    dxp = torch.zeros_like(xp)
    dw = torch.zeros_like(w)
    for j in range(K):
        dxp[:, j:j + T] += m(w[j]) * dpre
        dw[j] = (dpre * m(xp[:, j:j + T])).sum((0, 1))
    if dstate is not None:
        dxp[:, T:] += m(dstate)
    out.update(dx=dxp[:, K - 1:], dstate=dxp[:, :K - 1], dw=dw, dbias=dpre.sum((0, 1)))
    return out


def glu_ref(x, wg, wu, dy=None):
    g, u = x @ wg.T, x @ wu.T
    out = {"y": silu(g) * u}
    if dy is not None:
        dg, du = dy * u * dsilu(g), dy * silu(g)
        out.update(dx=dg @ wg + du @ wu, dwg=dg.T @ x, dwu=du.T @ x)
    return out


def glu_bound(x, wg, wu, half, dy=None):
    """How far the outputs may be off: fp32 sums (each product and addition off by
    2^-24 of its value, so k * 2^-24 of the absolute sum over k terms) and roundings
    of g, u, dg, du and the results by ``half`` of their value."""
    e = 2.0 ** -24
    D, I = x.shape[1], wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    mg, mu = x.abs() @ wg.abs().T, x.abs() @ wu.abs().T
    eg, eu = (D + 2) * e * mg, (D + 2) * e * mu
    ref = glu_ref(x, wg, wu, dy)
    # silu' <= 1.1, silu'' <= 0.5; 16 e for the sigmoid's own arithmetic
    ey = 1.1 * eg * u.abs() + silu(g).abs() * eu + eg * eu
    out = {"y": half * ref["y"].abs() + (1 + half) * (ey + 16 * e * ref["y"].abs()) + 1e-30}
    if dy is not None:
        hg, hu = eg + half * g.abs(), eu + half * u.abs()      # g and u as kept
        a = dy.abs()
        dg, du = a * u.abs() * dsilu(g).abs(), a * silu(g).abs()
        edg = a * (0.5 * hg * (u.abs() + hu) + hu * dsilu(g).abs())
        edu = a * 1.1 * hg
        # the sigmoid and the factors around it: 16 e of the largest term, 1.1 |dy u|
        edg = edg + (half + e) * (dg + edg) + 18 * e * a * u.abs()
        edu = edu + (half + e) * (du + edu) + 18 * e * a * g.abs()
        tg, tu = dg + edg, du + edu
        M = x.shape[0]
        out["dx"] = (edg @ wg.abs() + edu @ wu.abs()
                     + (2 * I + 2) * e * (tg @ wg.abs() + tu @ wu.abs())
                     + half * ref["dx"].abs() * 1.01 + 1e-30)
        for k, ed, t in (("dwg", edg, tg), ("dwu", edu, tu)):
            out[k] = (ed.T @ x.abs() + (M + 2) * e * (t.T @ x.abs())
                      + half * ref[k].abs() * 1.01 + 1e-30)
    return out
