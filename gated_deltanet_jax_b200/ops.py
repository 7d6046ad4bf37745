"""Gated delta-rule ops with the reference package's names and signatures.

Mirrors ``gated_deltanet_jax.ops`` (reference ``src/gated_deltanet_jax/ops.py``):

* :func:`chunk_gated_delta_rule_fwd` / :func:`chunk_gated_delta_rule`
  -- ops.py:299 and its alias at ops.py:352;
* :func:`fused_recurrent_gated_delta_rule` / :func:`fused_recurrent_gated_delta_rule_fwd`
  -- the Pallas wrapper ops.py:187 and its aliases at ops.py:350-351.

Arrays are CUDA ``torch.Tensor`` s in the reference layout (q, k ``[B,T,H,dk]``,
v ``[B,T,H,dv]``, g, beta ``[B,T,H]``, states ``[B,H,dk,dv]``).  Every call
goes through the C ABI of ``libgdn_b200.so`` on the tensor's current CUDA
stream; there is no CPU path.  Both ops compute the delta-rule recurrence
(the reference's recurrent kernel, ops.py:170-184) with an fp32 state and
return ``o`` in v's dtype.

Differences from the reference, all additive:

* ``fused_recurrent_gated_delta_rule`` also accepts ``initial_state`` and
  ``output_final_state`` (the reference always starts from zeros and returns
  ``(o, None)``, ops.py:168/219); without them it behaves the same.
* ``final_state_out=`` writes the final state into a given fp32 tensor, which
  may be ``initial_state`` itself (in-place decode).
* ``semantics="reference"`` on the chunk op reproduces ops.py:238-346 as
  written, including its deviations from the recurrence.
* Grouped value heads: q and k may carry fewer heads (Hk) than v, g and beta
  (H, a multiple of Hk).  Value head h then uses q/k head ``h * Hk // H``,
  which is what the reference layer obtains by ``jnp.repeat`` of q and k
  before calling its ops (model.py:132-135), without the repeated copies.
* ``cu_seqlens=`` on the chunk op: several sequences packed back to back in
  one row (q ``[1,T,Hk,dk]`` ...), sequence s being tokens
  ``cu_seqlens[s]:cu_seqlens[s+1]``, with one state per sequence.  Each
  sequence gets what a call on it alone gives.  (The reference takes one
  dense batch only.)
* Both ops are differentiable (exact semantics; the chunk op also with
  ``cu_seqlens``): when an input requires grad, the backward runs the
  gdn_chunk_bwd kernels (gdn_chunk_bwd_varlen for packed sequences).  The
  reference has no backward of its own; it differentiates its chunk path with
  JAX.
"""

from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.GDN_DTYPE_FP32, torch.bfloat16: _lib.GDN_DTYPE_BF16}
_SEMANTICS = {"exact": _lib.GDN_SEMANTICS_EXACT, "reference": _lib.GDN_SEMANTICS_REFERENCE}


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _prepare(q, k, v, g, beta, initial_state, final_state_out, output_final_state,
             n_states=None):
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if q.dim() != 4 or k.shape != q.shape:
        raise ValueError(f"q and k must both be [B,T,Hk,dk]; got {tuple(q.shape)}, {tuple(k.shape)}")
    B, T, Hk, dk = q.shape
    if v.dim() != 4 or tuple(v.shape[:2]) != (B, T):
        raise ValueError(f"v must be [B,T,H,dv] with B,T={B},{T}; got {tuple(v.shape)}")
    H, dv = v.shape[2], v.shape[3]
    if (Hk == 0) != (H == 0) or (H and H % Hk):
        raise ValueError(f"v's {H} heads must be a multiple of q/k's {Hk} heads")
    for name, t in (("g", g), ("beta", beta)):
        if tuple(t.shape) != (B, T, H):
            raise ValueError(f"{name} must be [B,T,H]=({B},{T},{H}); got {tuple(t.shape)}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError(f"q, k, v must share one dtype; got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"dtype {q.dtype} not supported (bfloat16 or float32)")
    dev = q.device
    NS = B if n_states is None else n_states   # states: one per batch row or per sequence
    for name, t in (("k", k), ("v", v), ("g", g), ("beta", beta)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, q on {dev}")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g = g.to(torch.float32).contiguous()
    beta = beta.to(torch.float32).contiguous()
    # The kernels read 16-byte aligned rows; a view that starts mid-row (e.g. a
    # token slice of g) is copied into fresh, aligned storage.
    q, k, v, g, beta = (t if t.data_ptr() % 16 == 0 else t.clone()
                        for t in (q, k, v, g, beta))
    h0 = None
    if initial_state is not None:
        if tuple(initial_state.shape) != (NS, H, dk, dv):
            raise ValueError(f"initial_state must be [{'B' if n_states is None else 'N'},H,dk,dv]"
                             f"=({NS},{H},{dk},{dv}); got {tuple(initial_state.shape)}")
        if initial_state.device != dev:
            raise ValueError(f"initial_state is on {initial_state.device}, q on {dev}")
        h0 = initial_state
        if h0.dtype != torch.float32 or not h0.is_contiguous():
            h0 = h0.to(torch.float32).contiguous()
    hT = None
    if final_state_out is not None:
        if (tuple(final_state_out.shape) != (NS, H, dk, dv) or final_state_out.dtype != torch.float32
                or not final_state_out.is_contiguous() or final_state_out.device != dev):
            raise ValueError("final_state_out must be a contiguous float32 [B,H,dk,dv] tensor "
                             "on the inputs' device")
        hT = final_state_out
    elif output_final_state:
        hT = torch.empty((NS, H, dk, dv), dtype=torch.float32, device=dev)
    o = torch.empty((B, T, H, dv), dtype=v.dtype, device=dev)
    return q, k, v, g, beta, h0, hT, o, (B, T, H, Hk, dk, dv)


def _wants_grad(*ts) -> bool:
    """Whether an input asks for a gradient; raises for tangents (forward mode), which no
    kernel carries on: the output would come without one."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the kernels have no forward-mode derivatives")
    if not torch.is_grad_enabled():
        return False
    for t in ts:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            return True
    return False


class _DeltaRuleFn(torch.autograd.Function):
    """Autograd node of both ops (same function: the recurrence, exact semantics)."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, chunk_size, recurrent, cu_seqlens=None):
        if recurrent:
            o, hT = _recurrent_impl(q, k, v, g, beta, h0, True, None)
        else:
            o, hT = _chunk_impl(q, k, v, g, beta, h0, True, chunk_size, "exact", None,
                                cu_seqlens)
        ctx.set_materialize_grads(False)
        ctx.has_h0 = h0 is not None
        ctx.in_dtypes = (g.dtype, beta.dtype, None if h0 is None else h0.dtype)
        ctx.save_for_backward(q, k, v, g, beta, h0, cu_seqlens)
        return o, hT

    @staticmethod
    def backward(ctx, do, dhT):
        q, k, v, g, beta, h0, cu_seqlens = ctx.saved_tensors
        dq, dk, dv, dg, db, dh0 = _chunk_backward(q, k, v, g, beta, h0, do, dhT, cu_seqlens)
        gd, bd, hd = ctx.in_dtypes
        return (dq, dk, dv, dg.to(gd), db.to(bd), dh0.to(hd) if ctx.has_h0 else None, None,
                None, None)


def _check_cu_seqlens(q, cu_seqlens):
    """Validate packed-sequence offsets (as the forward does); returns N."""
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or \
            cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must be a 1-D int32/int64 tensor of N+1 offsets")
    if q.dim() != 4 or q.shape[0] != 1:
        raise ValueError("with cu_seqlens, q, k, v, g, beta hold one packed row (B == 1)")
    if not cu_seqlens.is_cuda:
        c = cu_seqlens.tolist()
        if c[0] != 0 or c[-1] != q.shape[1] or any(b < a for a, b in zip(c, c[1:])):
            raise ValueError(f"cu_seqlens must rise from 0 to T={q.shape[1]}; got {c}")
    return cu_seqlens.numel() - 1


def _chunk_backward(q, k, v, g, beta, h0, do, dhT, cu_seqlens=None):
    """Gradients of the recurrence through the C ABI: gdn_chunk_bwd, or
    gdn_chunk_bwd_varlen for packed sequences (``cu_seqlens``)."""
    n_seqs = None if cu_seqlens is None else _check_cu_seqlens(q, cu_seqlens)
    q, k, v, g, beta, h0c, _, _, (B, T, H, Hk, dk, dv) = _prepare(
        q, k, v, g, beta, h0, None, False, n_seqs)
    NS = B if n_seqs is None else n_seqs
    dev = q.device
    if do is None:
        do = torch.zeros((B, T, H, dv), dtype=v.dtype, device=dev)
    do = do.to(v.dtype).contiguous()
    if do.data_ptr() % 16:
        do = do.clone()
    dhT_c = None if dhT is None else dhT.to(torch.float32).contiguous()
    dq = torch.empty_like(q)
    dk_ = torch.empty_like(k)
    dv_ = torch.empty_like(v)
    dg = torch.empty((B, T, H), dtype=torch.float32, device=dev)
    db = torch.empty((B, T, H), dtype=torch.float32, device=dev)
    dh0 = torch.empty((NS, H, dk, dv), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        args = (_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(h0c), _ptr(do),
                _ptr(dhT_c), _ptr(dq), _ptr(dk_), _ptr(dv_), _ptr(dg), _ptr(db), _ptr(dh0))
        if n_seqs is None:
            ws_bytes = lib.gdn_chunk_bwd_workspace_bytes_for(B, T, H, Hk, dk, dv,
                                                             _DTYPES[q.dtype])
            ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
            rc = lib.gdn_chunk_bwd(*args, B, T, H, Hk, dk, dv, _DTYPES[q.dtype], _ptr(ws),
                                   ws_bytes, stream)
            what = "gdn_chunk_bwd"
        else:
            cu = cu_seqlens.to(device=dev, dtype=torch.int32).contiguous()
            ws_bytes = lib.gdn_chunk_bwd_varlen_workspace_bytes(n_seqs, T, H, dk, dv)
            ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
            rc = lib.gdn_chunk_bwd_varlen(*args, _ptr(cu), n_seqs, T, H, Hk, dk, dv,
                                          _DTYPES[q.dtype], _ptr(ws), ws_bytes, stream)
            what = "gdn_chunk_bwd_varlen"
    _lib.check(rc, what)
    return dq, dk_, dv_, dg, db, dh0


def chunk_gated_delta_rule_fwd(q, k, v, g, beta, initial_state=None, output_final_state=False,
                               chunk_size=64, *, semantics: str = "exact",
                               final_state_out: Optional[torch.Tensor] = None,
                               cu_seqlens: Optional[torch.Tensor] = None
                               ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Chunked gated delta rule (reference ``chunk_gated_delta_rule_fwd``, ops.py:299).

    Returns ``(o, final_state)`` when ``output_final_state`` (or
    ``final_state_out``) is given, else ``(o, None)`` (ops.py:344-346).
    ``chunk_size`` is 16, 32 or 64.  ``semantics="exact"`` (default) equals the
    recurrence; ``"reference"`` reproduces the reference chunk code as written.
    ``cu_seqlens`` (integer ``[N+1]``, non-decreasing from 0 to T) packs N
    sequences into one row: q ``[1,T,Hk,dk]``, states ``[N,H,dk,dv]``.
    Differentiable (exact semantics, dense or packed) when an input requires grad.
    """
    if _wants_grad(q, k, v, g, beta, initial_state):
        if semantics != "exact" or final_state_out is not None:
            raise NotImplementedError("the backward covers exact semantics without "
                                      "final_state_out")
        cu = None
        if cu_seqlens is not None:
            _check_cu_seqlens(q, cu_seqlens)
            cu = cu_seqlens.to(device=q.device, dtype=torch.int32).contiguous()
        o, hT = _DeltaRuleFn.apply(q, k, v, g, beta, initial_state, int(chunk_size), False, cu)
        return (o, hT) if output_final_state else (o, None)
    return _chunk_impl(q, k, v, g, beta, initial_state, output_final_state, chunk_size,
                       semantics, final_state_out, cu_seqlens)


def _chunk_impl(q, k, v, g, beta, initial_state, output_final_state, chunk_size, semantics,
                final_state_out, cu_seqlens):
    if semantics not in _SEMANTICS:
        raise ValueError(f"semantics must be one of {sorted(_SEMANTICS)}; got {semantics!r}")
    n_seqs = None
    if cu_seqlens is not None:
        n_seqs = _check_cu_seqlens(q, cu_seqlens)
        if semantics != "exact":
            raise ValueError("packed sequences take semantics='exact' only")
    q, k, v, g, beta, h0, hT, o, (B, T, H, Hk, dk, dv) = _prepare(
        q, k, v, g, beta, initial_state, final_state_out, output_final_state, n_seqs)
    lib = _lib.load()
    dtype = _DTYPES[q.dtype]
    sem = _SEMANTICS[semantics]
    with torch.cuda.device(q.device):
        if n_seqs is not None:
            ws_bytes = lib.gdn_chunk_varlen_workspace_bytes(n_seqs, T, H, dk, dv,
                                                            int(chunk_size), dtype, sem)
        else:
            ws_bytes = lib.gdn_chunk_workspace_bytes(B, T, H, dk, dv, int(chunk_size), dtype,
                                                     sem)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        stream = torch.cuda.current_stream(q.device).cuda_stream
        if n_seqs is not None:
            cu = cu_seqlens.to(device=q.device, dtype=torch.int32).contiguous()
            rc = lib.gdn_chunk_fwd_varlen(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta),
                                          _ptr(h0), _ptr(o), _ptr(hT), _ptr(cu), n_seqs, T, H, Hk,
                                          dk, dv, int(chunk_size), dtype, sem, _ptr(ws), ws_bytes,
                                          stream)
        elif Hk == H:
            rc = lib.gdn_chunk_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(h0),
                                   _ptr(o), _ptr(hT), B, T, H, dk, dv, int(chunk_size), dtype,
                                   sem, _ptr(ws), ws_bytes, stream)
        else:
            rc = lib.gdn_chunk_fwd_gva(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(h0),
                                       _ptr(o), _ptr(hT), B, T, H, Hk, dk, dv, int(chunk_size),
                                       dtype, sem, _ptr(ws), ws_bytes, stream)
    _lib.check(rc, "gdn_chunk_fwd")
    return o, hT


def _two_phase_ok(q, k, v) -> bool:
    """Whether gdn_chunk_prepare / gdn_chunk_scan take these tensors (bf16, dk =
    128, dv a multiple of 64 up to 512, dense rows on a CUDA device)."""
    return (isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 4
            and q.dtype == torch.bfloat16 and k.dtype == q.dtype and v.dtype == q.dtype
            and q.shape[-1] == 128 and v.shape[-1] % 64 == 0 and 0 < v.shape[-1] <= 512
            and q.shape[0] * v.shape[2] <= 65535 and q.shape[1] > 0 and q.shape[0] > 0)


def _chunk_prepare(q, k, g, beta):
    """gdn_chunk_prepare: the per-chunk operands of (q, k, g, beta) in a new
    workspace (uint8 CUDA tensor) for _chunk_scan."""
    B, T, Hk, dk = q.shape
    H = g.shape[2]
    lib = _lib.load()
    ws_bytes = lib.gdn_chunk_workspace_bytes(B, T, H, dk, 64, 64, _lib.GDN_DTYPE_BF16,
                                             _lib.GDN_SEMANTICS_EXACT)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        rc = lib.gdn_chunk_prepare(_ptr(q), _ptr(k), _ptr(g), _ptr(beta), B, T, H, Hk, dk,
                                   _lib.GDN_DTYPE_BF16, _ptr(ws), ws_bytes,
                                   torch.cuda.current_stream(q.device).cuda_stream)
    _lib.check(rc, "gdn_chunk_prepare")
    return ws


def _chunk_scan(q, k, v, g, beta, ws, initial_state=None, transition=False, output=True):
    """gdn_chunk_scan over a workspace from _chunk_prepare of the same q, k, g,
    beta.  Returns (o or None, final state); with ``transition`` the final
    state is [B,H,dk,dv+dk]: the end state from a zero start, then the
    transition matrix (initial_state must be None)."""
    B, T, Hk, dk = q.shape
    H, dv = v.shape[2], v.shape[3]
    hT = torch.empty((B, H, dk, dv + (dk if transition else 0)), dtype=torch.float32,
                     device=q.device)
    o = torch.empty((B, T, H, dv), dtype=v.dtype, device=q.device) if output else None
    h0 = None if initial_state is None else initial_state.to(torch.float32).contiguous()
    lib = _lib.load()
    with torch.cuda.device(q.device):
        rc = lib.gdn_chunk_scan(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(h0),
                                _ptr(o), _ptr(hT), B, T, H, Hk, dk, dv, _lib.GDN_DTYPE_BF16,
                                int(bool(transition)), _ptr(ws), ws.numel(),
                                torch.cuda.current_stream(q.device).cuda_stream)
    _lib.check(rc, "gdn_chunk_scan")
    return o, hT


def _fold_states(packed, h0, dv):
    """gdn_fold_states over the gathered summaries ``packed`` [P, B, H, dk,
    dv + dk] fp32 (end state from zero, then transition, per segment) from h0
    [B, H, dk, dv] (None: zero).  Returns [P + 1, B, H, dk, dv]: the state
    entering each segment and, last, the state after the final one."""
    packed = packed.contiguous()
    P, B, H, dk, ld = packed.shape
    out = torch.empty((P + 1, B, H, dk, dv), dtype=torch.float32, device=packed.device)
    h0 = None if h0 is None else h0.to(torch.float32).contiguous()
    lib = _lib.load()
    with torch.cuda.device(packed.device):
        rc = lib.gdn_fold_states(_ptr(packed), packed.data_ptr() + 4 * dv, _ptr(h0), _ptr(out),
                                 P, B * H, dk, dv, ld,
                                 torch.cuda.current_stream(packed.device).cuda_stream)
    _lib.check(rc, "gdn_fold_states")
    return out


def fused_recurrent_gated_delta_rule(q, k, v, g, beta, initial_state=None,
                                     output_final_state=False, *,
                                     final_state_out: Optional[torch.Tensor] = None
                                     ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Fused recurrent gated delta rule (reference Pallas wrapper, ops.py:187-219).

    With neither ``initial_state`` nor ``output_final_state`` this is the
    reference call: zero initial state, returns ``(o, None)``.  For decode pass
    ``initial_state=S, final_state_out=S`` to update the state in place.
    Differentiable (without ``final_state_out``) when an input requires grad.
    """
    if _wants_grad(q, k, v, g, beta, initial_state):
        if final_state_out is not None:
            raise NotImplementedError("the backward does not cover final_state_out")
        o, hT = _DeltaRuleFn.apply(q, k, v, g, beta, initial_state, 64, True)
        return (o, hT) if output_final_state else (o, None)
    return _recurrent_impl(q, k, v, g, beta, initial_state, output_final_state, final_state_out)


def _recurrent_impl(q, k, v, g, beta, initial_state, output_final_state, final_state_out):
    q, k, v, g, beta, h0, hT, o, (B, T, H, Hk, dk, dv) = _prepare(
        q, k, v, g, beta, initial_state, final_state_out, output_final_state)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream(q.device).cuda_stream
        if Hk == H:
            rc = lib.gdn_recurrent_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(h0),
                                       _ptr(o), _ptr(hT), B, T, H, dk, dv, _DTYPES[q.dtype],
                                       stream)
        else:
            rc = lib.gdn_recurrent_fwd_gva(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta),
                                           _ptr(h0), _ptr(o), _ptr(hT), B, T, H, Hk, dk, dv,
                                           _DTYPES[q.dtype], stream)
    _lib.check(rc, "gdn_recurrent_fwd")
    return o, hT


def gated_delta_rule_decode_layer(q, k, v, a, b, A_log, dt_bias, *, gate=None,
                                  norm_weight=None, eps: float = 1e-5, initial_state=None,
                                  output_final_state=False,
                                  final_state_out: Optional[torch.Tensor] = None
                                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The GatedDeltaNet layer's core around the recurrent op
    (gdn_recurrent_fwd_layer): the gates from the raw projections, the
    recurrent step, and the gated RMSNorm of its output.  Single-token decode
    at dk = dv = 128 is one kernel; other shapes run the recurrent kernel with
    the gates formed in it, then the norm kernel (whole sequences on the
    tensor-core shapes take the chunked layer form).

    The reference layer (model.py:136-153) runs these as separate operations:
    ``beta = sigmoid(b)``, ``g = -exp(A_log) * softplus(a + dt_bias)``, the op,
    then ``FusedRMSNormGated`` (model.py:41-53; with ``gate=None`` the plain
    RMSNorm of the ungated layer, whose epsilon is 1e-6).

    q, k ``[B,T,Hk,dk]``; v ``[B,T,H,dv]``; a, b ``[B,T,H]`` (a_proj, b_proj
    outputs); A_log, dt_bias ``[H]``; gate ``[B,T,H,dv]`` in v's dtype or None;
    norm_weight ``[dv]`` (None: ones).  Returns ``(y, final_state)`` like the
    recurrent op (``final_state_out=S`` with ``initial_state=S`` updates S in
    place).  Inference only: there is no backward for this form.
    """
    return _layer_impl("gdn_recurrent_fwd_layer", q, k, v, a, b, A_log, dt_bias, gate,
                       norm_weight, eps, initial_state, output_final_state, final_state_out)


def gated_delta_rule_chunk_layer(q, k, v, a, b, A_log, dt_bias, *, gate=None,
                                 norm_weight=None, eps: float = 1e-5, initial_state=None,
                                 output_final_state=False,
                                 final_state_out: Optional[torch.Tensor] = None,
                                 cu_seqlens: Optional[torch.Tensor] = None
                                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The GatedDeltaNet layer's core over a whole sequence (prefill)
    (gdn_chunk_fwd_layer): the gates from the raw projections, the chunked
    forward (exact semantics), and the gated RMSNorm of every output row --
    what model.py:136-153 computes around chunk_gated_delta_rule_fwd as
    separate operations.  One kernel at dk = dv = 128; at the other
    tensor-core shapes (dk = 256, dv a multiple of 64 -- the reference's
    default dk = 256, dv = 512) the chunk kernel forms the gates and a second
    kernel normalises its output in place.

    q, k ``[B,T,Hk,dk]`` and v ``[B,T,H,dv]`` in bfloat16; a, b ``[B,T,H]``;
    A_log, dt_bias ``[H]``; gate ``[B,T,H,dv]`` in v's dtype or None;
    norm_weight ``[dv]`` (None: ones).  Returns ``(y, final_state)`` like
    chunk_gated_delta_rule, packed sequences included (``cu_seqlens``: one row
    of T tokens holding N sequences, states ``[N,H,dk,dv]``).  Inference
    only: there is no backward for this form.
    """
    return _layer_impl("gdn_chunk_fwd_layer", q, k, v, a, b, A_log, dt_bias, gate,
                       norm_weight, eps, initial_state, output_final_state, final_state_out,
                       cu_seqlens)


def _layer_impl(entry, q, k, v, a, b, A_log, dt_bias, gate, norm_weight, eps, initial_state,
                output_final_state, final_state_out, cu_seqlens=None):
    if _wants_grad(q, k, v, a, b, initial_state):
        raise NotImplementedError("the layer forms have no backward")
    n_seqs = None if cu_seqlens is None else _check_cu_seqlens(q, cu_seqlens)
    q, k, v, a, b, h0, hT, y, (B, T, H, Hk, dk, dv) = _prepare(
        q, k, v, a, b, initial_state, final_state_out, output_final_state, n_seqs)
    dev = q.device

    def vec(t, n, name):
        if t is None:
            return None
        t = torch.as_tensor(t, device=dev).to(torch.float32).contiguous()
        if t.shape != (n,):
            raise ValueError(f"{name} must be [{n}]; got {tuple(t.shape)}")
        return t

    A_log, dt_bias = vec(A_log, H, "A_log"), vec(dt_bias, H, "dt_bias")
    w = vec(norm_weight, dv, "norm_weight")
    if w is None:
        w = torch.ones(dv, dtype=torch.float32, device=dev)
    if gate is not None:
        if tuple(gate.shape) != (B, T, H, dv):
            raise ValueError(f"gate must be [B,T,H,dv]=({B},{T},{H},{dv}); got {tuple(gate.shape)}")
        gate = gate.to(device=dev, dtype=v.dtype).contiguous()
        if gate.data_ptr() % 16:
            gate = gate.clone()
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        head = (_ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b), _ptr(A_log), _ptr(dt_bias),
                _ptr(h0), _ptr(hT), _ptr(gate), _ptr(w), float(eps), _ptr(y))
        if n_seqs is not None:
            entry += "_varlen"
            cu = cu_seqlens.to(device=dev, dtype=torch.int32).contiguous()
            rc = getattr(lib, entry)(*head, _ptr(cu), n_seqs, T, H, Hk, dk, dv,
                                     _DTYPES[q.dtype], stream)
        else:
            rc = getattr(lib, entry)(*head, B, T, H, Hk, dk, dv, _DTYPES[q.dtype], stream)
    _lib.check(rc, entry)
    return y, hT


_ACTIVATIONS = {"silu": 1, "swish": 1, None: 0}


_NO_SWITCH = contextlib.nullcontext()


def _on_device(index: int):
    """``torch.cuda.device`` where it is not the current one already (single-token
    calls are bound by their host work)."""
    # (the raw query: its caller holds a CUDA tensor, so CUDA is initialised)
    return _NO_SWITCH if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def _stream(index: int) -> int:
    # the raw handle: torch.cuda.current_stream() builds a Stream object around it
    return torch._C._cuda_getCurrentRawStream(index)


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and 16-byte aligned, as the kernels read and write."""
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _aligned32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The same in fp32."""
    if t is not None and t.dtype is not torch.float32:
        t = t.to(torch.float32)
    return _aligned(t)


def _on(t, dev):
    """A parameter on ``dev``: CUDA tensors stay, host values are copied."""
    if isinstance(t, torch.Tensor) and t.device == dev:
        return t
    return torch.as_tensor(t, device=dev)


def _check_input(name, t, dev, dtype):
    """A CUDA tensor on the same device and of the same dtype as the first input."""
    if isinstance(t, torch.Tensor):
        if t.dtype is dtype and t.device == dev:
            return
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not on {dev}")
        raise TypeError(f"{name} must be {dtype} like the other inputs; got {t.dtype}")
    raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")


def _cuda_input(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be bfloat16 or float32; got {t.dtype}")


def _check_sizes(name, sizes):
    """The library's sizes are 32-bit; a larger one would arrive as its low half."""
    if sizes and max(sizes) > 0x7fffffff:
        raise ValueError(f"{name} is too large: {tuple(sizes)} has a size past 2^31 - 1")


def _conv_state(t, name, shape, dtype, dev):
    if t is None:
        return None
    if t.shape != shape or t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must be {shape} {dtype} on {dev}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and 16-byte aligned")
    return t


def _alias(t, connect):
    """``t`` as a point to differentiate at: with ``connect`` still a function of what t
    came from, else on its own."""
    if t is None:
        return None
    return t.view_as(t) if connect and t.requires_grad else t.detach().requires_grad_(True)


def _formula_grads(formula, ts, cots):
    """Gradients of ``formula(*ts)`` (a tuple) for the cotangents ``cots`` through torch's
    own operations: where the kernels cannot run (batched cotangents)."""
    connect = torch.is_grad_enabled()
    with torch.enable_grad():
        a = [_alias(t, connect) for t in ts]
        live = [(o, c) for o, c in zip(formula(*a), cots) if c is not None]
        wrt = [t for t in a if t is not None]
        got = iter(torch.autograd.grad([o for o, _ in live], wrt, [c for _, c in live],
                                       create_graph=connect, allow_unused=True))
    return tuple(None if t is None else next(got) for t in a)


def _formula_second(formula, ts, cots, dds):
    """The gradients of that: for cotangents ``dds`` of the gradients by ``ts``, the
    gradients by ``cots`` and by ``ts``, themselves differentiable when grad mode is on."""
    connect = torch.is_grad_enabled()
    by = [i for i, d in enumerate(dds) if d is not None and ts[i] is not None]
    if not by or all(d is None for d in cots):
        return (None,) * (len(cots) + len(ts))
    with torch.enable_grad():
        a, c = [_alias(t, connect) for t in ts], [_alias(t, connect) for t in cots]
        live = [(o, d) for o, d in zip(formula(*a), c) if d is not None]
        first = torch.autograd.grad([o for o, _ in live], [a[i] for i in by],
                                    [d for _, d in live], create_graph=True, allow_unused=True)
        pairs = [(f, dds[i]) for f, i in zip(first, by) if f is not None and f.requires_grad]
        both = c + a
        wrt = [t for t in both if t is not None]
        got = iter(torch.autograd.grad([f for f, _ in pairs], wrt, [d for _, d in pairs],
                                       create_graph=connect, allow_unused=True) if pairs
                   else [None] * len(wrt))
    return tuple(None if t is None else next(got) for t in both)


def _batched(*ts) -> bool:
    """Tensors that stand for a batch of them and have no data pointer
    (``torch.autograd.grad(is_grads_batched=True)``)."""
    ft = torch._C._functorch
    return any(t is not None and (ft.is_legacy_batchedtensor(t) or ft.is_batchedtensor(t))
               for t in ts)


def _conv_formula(act):
    """The short convolution in torch's operations, fp32 inside."""
    def formula(x, w, bias, st):
        (B, T, C), K = x.shape, w.shape[0]
        xe = torch.cat([x.new_zeros(B, K - 1, C) if st is None else st, x], 1)
        pre = sum(w[j] * xe[:, j:j + T].to(w.dtype) for j in range(K))
        pre = pre if bias is None else pre + bias
        y = torch.nn.functional.silu(pre) if act else pre
        return y.to(x.dtype), xe[:, T:]
    return formula


def _short_conv_bwd(dy, ds, x, w, bias, st, act):
    """gdn_short_conv_bwd: (dx, dw, dbias, dstate), the last two None without theirs."""
    B, T, C = x.shape
    K = w.shape[0]
    dy = torch.zeros_like(x) if dy is None else _aligned(dy)
    ds = _aligned(ds)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    db = None if bias is None else torch.empty_like(bias)
    dst = None if st is None else torch.empty_like(st)
    lib = _lib.load()
    dev = x.get_device()
    with _on_device(dev):
        n = lib.gdn_short_conv_bwd_workspace_bytes(B, T, C, K)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)
        rc = lib.gdn_short_conv_bwd(
            _ptr(x), _ptr(w), _ptr(bias), _ptr(st), _ptr(dy), _ptr(ds), _ptr(dx), _ptr(dw),
            _ptr(db), _ptr(dst), B, T, C, K, act, _DTYPES[x.dtype], _ptr(ws), n,
            _stream(dev))
    _lib.check(rc, "gdn_short_conv_bwd")
    return dx, dw, db, dst


# The autograd functions take aligned inputs (weights in fp32 where the kernels want them
# so): what is saved for the backward is then the inputs themselves, and with
# create_graph=True the gradients' own graph reaches them.

class _ShortConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, conv_state, act):
        s_out = x.new_empty((x.shape[0], w.shape[0] - 1, x.shape[2]))
        y = _short_conv_fwd(x, w, bias, conv_state, s_out, act)
        ctx.act = act
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w, bias, conv_state)
        return y, s_out

    @staticmethod
    def backward(ctx, dy, ds):
        ts = ctx.saved_tensors
        if _batched(dy, ds):
            return _formula_grads(_conv_formula(ctx.act), ts, (dy, ds)) + (None,)
        run = _ShortConvBwdFn.apply if torch.is_grad_enabled() else _short_conv_bwd
        return tuple(run(dy, ds, *ts, ctx.act)) + (None,)


class _ShortConvBwdFn(torch.autograd.Function):
    """The backward as a function of its own (create_graph=True): the kernel's gradients,
    whose derivatives are formed by torch's operations."""

    @staticmethod
    def forward(ctx, dy, ds, x, w, bias, conv_state, act):
        ctx.act = act
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(dy, ds, x, w, bias, conv_state)
        return _short_conv_bwd(dy, ds, x, w, bias, conv_state, act)

    @staticmethod
    def backward(ctx, *dds):
        dy, ds, *ts = ctx.saved_tensors
        return _formula_second(_conv_formula(ctx.act), ts, (dy, ds), dds) + (None,)


def _short_conv_fwd(x, w, bias, s_in, s_out, act):
    """gdn_short_conv_fwd_bias on checked, contiguous inputs; returns y."""
    B, T, C = x.shape
    y = torch.empty_like(x)
    lib = _lib.load()
    dev = x.get_device()
    with _on_device(dev):
        rc = lib.gdn_short_conv_fwd_bias(_ptr(x), _ptr(w), _ptr(bias), _ptr(s_in), _ptr(s_out),
                                         _ptr(y), B, T, C, w.shape[0], act, _DTYPES[x.dtype],
                                         _stream(dev))
    _lib.check(rc, "gdn_short_conv_fwd")
    return y


def short_convolution(x, weight, *, bias=None, activation: Optional[str] = "silu",
                      conv_state=None, output_final_state: bool = False,
                      final_state_out: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """ShortConvolution (model.py:15-40) on the GPU (gdn_short_conv_fwd): a
    causal depthwise convolution over time, kernel K, then SiLU for
    ``activation`` ``'silu'`` / ``'swish'`` (None: none).

    x ``[B,T,C]`` bfloat16 or float32 on a CUDA device; weight ``[K,C]`` or the
    flax kernel ``[K,1,C]``, bias ``[C]`` or None (taken to float32).  ``conv_state``
    ``[B,K-1,C]`` in x's dtype replaces the zero padding before token 0 (the
    inputs a previous call ended with).  Returns ``(y, state)``: state
    ``[B,K-1,C]`` holds the last K - 1 inputs when ``output_final_state`` or
    ``final_state_out`` (which may be ``conv_state``, updated in place) is
    given, else None.  The reference's call is ``short_convolution(x, w)`` (no
    state).  Differentiable in x, weight, bias and conv_state, through y and
    the returned state (gdn_short_conv_bwd; with ``final_state_out`` in weight and bias
    alone, of which the state is no function), twice too (second derivatives run on
    torch's operations).
    """
    _cuda_input("x", x)
    if x.dim() != 3:
        raise ValueError(f"x must be [B,T,C]; got {tuple(x.shape)}")
    _check_sizes("x", x.shape)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be 'silu', 'swish' or None; got {activation!r}")
    B, T, C = x.shape
    dev = x.device
    w = _on(weight, dev)
    if w.dim() == 3:
        w = w.reshape(w.shape[0], w.shape[-1])
    if w.dim() != 2 or w.shape[1] != C:
        raise ValueError(f"weight must be [K,{C}] or [K,1,{C}]; got {tuple(weight.shape)}")
    shape = (B, w.shape[0] - 1, C)
    s_in = _conv_state(conv_state, "conv_state", shape, x.dtype, dev)
    s_out = _conv_state(final_state_out, "final_state_out", shape, x.dtype, dev)
    if bias is not None:
        bias = _on(bias, dev)
        if bias.shape != (C,):
            raise ValueError(f"bias must be [{C}]; got {tuple(bias.shape)}")
    if _wants_grad(x, w, bias, conv_state):
        if final_state_out is not None:
            if _wants_grad(x, conv_state):
                raise NotImplementedError("the backward does not cover final_state_out of an x or "
                                          "conv_state that requires grad")
            # the backward reads the window as it entered, which the call may overwrite
            s_in = None if s_in is None else s_in.clone()
        y, state = _ShortConvFn.apply(_aligned(x), _aligned32(w), _aligned32(bias), s_in, act)
        if final_state_out is not None:
            with torch.no_grad():
                return y, s_out.copy_(state)
        return y, state if output_final_state else None
    if s_out is None and output_final_state:
        s_out = torch.empty(shape, dtype=x.dtype, device=dev)
    y = _short_conv_fwd(_aligned(x), _aligned32(w), _aligned32(bias), s_in, s_out, act)
    return y, s_out


def _glu_fwd(x, wg, wu, keep):
    """gdn_glu_fwd on x [M,D], wg, wu [I,D]; returns h [M,I] and, with ``keep``,
    the two projections."""
    (M, D), I = x.shape, wg.shape[0]
    h = x.new_empty((M, I))
    # (in fp32 whatever x's type: rounded to bf16, they would be most of the gradients' error)
    g = u = None
    if keep:
        g, u = h.new_empty((M, I), dtype=torch.float32), h.new_empty((M, I), dtype=torch.float32)
    lib = _lib.load()
    dev = x.get_device()
    with _on_device(dev):
        rc = lib.gdn_glu_fwd_kept(_ptr(x), _ptr(wg), _ptr(wu), _ptr(h), _ptr(g), _ptr(u), M, D, I,
                                  _DTYPES[x.dtype], _lib.GDN_DTYPE_FP32, _stream(dev))
    _lib.check(rc, "gdn_glu_fwd")
    return h, g, u


def _glu_formula(x, wg, wu):
    """The gated linear unit in torch's operations: products in the inputs' type, the
    activation in fp32."""
    lin = torch.nn.functional.linear
    g, u = lin(x, wg), lin(x, wu)
    if x.dtype == torch.bfloat16:
        g, u = g.float(), u.float()
    return ((torch.nn.functional.silu(g) * u).to(x.dtype),)


def _glu_bwd(dh, x, wg, wu, g, u, need_x, need_w):
    """gdn_glu_bwd: (dx, dwg, dwu), None where not needed."""
    (M, D), I = x.shape, wg.shape[0]
    dh = _aligned(dh)
    dx = torch.empty_like(x) if need_x else None
    dwg, dwu = (torch.empty_like(wg), torch.empty_like(wu)) if need_w else (None, None)
    lib = _lib.load()
    dev = x.get_device()
    with _on_device(dev):
        n = lib.gdn_glu_bwd_workspace_bytes(M, D, I, _DTYPES[x.dtype])
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)
        rc = lib.gdn_glu_bwd_kept(_ptr(x), _ptr(wg), _ptr(wu), _ptr(g), _ptr(u), _ptr(dh),
                                  _ptr(dx), _ptr(dwg), _ptr(dwu), M, D, I, _DTYPES[x.dtype],
                                  _lib.GDN_DTYPE_FP32, _ptr(ws), n, _stream(dev))
    _lib.check(rc, "gdn_glu_bwd")
    return dx, dwg, dwu


class _GluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu):
        h, g, u = _glu_fwd(x, wg, wu, True)
        ctx.save_for_backward(x, wg, wu, g, u)
        return h

    @staticmethod
    def backward(ctx, dh):
        x, wg, wu, g, u = ctx.saved_tensors
        if _batched(dh):
            return _formula_grads(_glu_formula, (x, wg, wu), (dh,))
        run = _GluBwdFn.apply if torch.is_grad_enabled() else _glu_bwd
        return tuple(run(dh, x, wg, wu, g, u, ctx.needs_input_grad[0],
                         any(ctx.needs_input_grad[1:])))


class _GluBwdFn(torch.autograd.Function):
    """The backward as a function of its own, as _ShortConvBwdFn."""

    @staticmethod
    def forward(ctx, dh, x, wg, wu, g, u, need_x, need_w):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(dh, x, wg, wu)
        return _glu_bwd(dh, x, wg, wu, g, u, need_x, need_w)

    @staticmethod
    def backward(ctx, *dds):
        dh, *ts = ctx.saved_tensors
        return _formula_second(_glu_formula, ts, (dh,), dds) + (None,) * 4


def gated_linear_unit(x, gate_weight, up_weight, *, activation: str = "silu") -> torch.Tensor:
    """The gated linear unit of the feed-forward block (GatedDeltaNetMLP,
    model.py:162-180, before its down projection) as one kernel (gdn_glu_fwd):
    ``silu(x @ gate_weight.T) * (x @ up_weight.T)``.

    x ``[...,D]``, gate_weight and up_weight ``[I,D]`` (torch's Linear layout)
    in one dtype, bfloat16 or float32, on a CUDA device; returns ``[...,I]``.
    ``activation``: ``'silu'`` / ``'swish'``.  Differentiable in all three
    (gdn_glu_bwd, from the two projections kept in float32), twice too (second
    derivatives run on torch's operations).  bfloat16 widths D and I that are multiples of
    8 (D up to 131072) run on the tensor cores, others on CUDA cores.
    """
    _cuda_input("x", x)
    if activation not in ("silu", "swish"):
        raise ValueError(f"activation must be 'silu' or 'swish'; got {activation!r}")
    if x.dim() < 1:
        raise ValueError("x must be [...,D]")
    D = x.shape[-1]
    dev, dtype = x.device, x.dtype
    _check_input("gate_weight", gate_weight, dev, dtype)
    _check_input("up_weight", up_weight, dev, dtype)
    if gate_weight.dim() != 2 or gate_weight.shape[1] != D or up_weight.shape != gate_weight.shape:
        raise ValueError(f"gate_weight and up_weight must both be [I,{D}]; got "
                         f"{tuple(gate_weight.shape)}, {tuple(up_weight.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), D)
    _check_sizes("x", x2.shape)
    _check_sizes("gate_weight", gate_weight.shape)
    if _wants_grad(x, gate_weight, up_weight):
        h = _GluFn.apply(_aligned(x2), _aligned(gate_weight), _aligned(up_weight))
    else:
        h, _, _ = _glu_fwd(_aligned(x2), _aligned(gate_weight), _aligned(up_weight), False)
    return h if x2 is x else h.reshape(*x.shape[:-1], gate_weight.shape[0])


def _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, h0, hT, keep):
    """gdn_selective_scan_fwd on checked, contiguous inputs; returns y and, with
    ``keep``, the checkpoints of the backward."""
    b, T, ch = x.shape
    G, N = B.shape[2], A.shape[1]
    y = torch.empty_like(x)
    lib = _lib.load()
    dev = x.get_device()
    with _on_device(dev):
        ck = None
        if keep:
            n = lib.gdn_selective_scan_checkpoint_bytes(b, T, ch, N)
            ck = torch.empty(max(n // 4, 4), dtype=torch.float32, device=x.device)
        n = lib.gdn_selective_scan_workspace_bytes(b, T, ch, N, G) if T > 1 else 0
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = lib.gdn_selective_scan_fwd(
            _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(dt_bias),
            _ptr(h0), _ptr(y), _ptr(hT), _ptr(ck), b, T, ch, N, G, softplus, _DTYPES[x.dtype],
            _ptr(ws), n, _stream(dev))
    _lib.check(rc, "gdn_selective_scan_fwd")
    return y, ck


def _scan_bwd(dy, dhT, x, dt, A, B, C, D, z, dt_bias, ck, has_h0, softplus):
    """gdn_selective_scan_bwd: the gradients of x, dt, A, B, C, D, z, dt_bias and the
    initial state, None without theirs."""
    b, T, ch = x.shape
    G, N = B.shape[2], A.shape[1]
    dev = x.get_device()
    dy = torch.zeros_like(x) if dy is None else _aligned(dy)
    dhT = _aligned32(dhT)
    like = lambda t: None if t is None else torch.empty_like(t)  # noqa: E731
    dx, ddt, dA, dB, dC = like(x), like(dt), like(A), like(B), like(C)
    dD, dz, dbias = like(D), like(z), like(dt_bias)
    dh0 = torch.empty((b, ch, N), dtype=torch.float32, device=dev) if has_h0 else None
    lib = _lib.load()
    with _on_device(dev):
        n = lib.gdn_selective_scan_bwd_workspace_bytes(b, T, ch, N, G)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
        rc = lib.gdn_selective_scan_bwd(
            _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(dt_bias),
            _ptr(ck), _ptr(dy), _ptr(dhT), _ptr(dx), _ptr(ddt), _ptr(dA), _ptr(dB), _ptr(dC),
            _ptr(dD), _ptr(dz), _ptr(dbias), _ptr(dh0), b, T, ch, N, G, softplus,
            _DTYPES[x.dtype], _ptr(ws), n, _stream(dev))
    _lib.check(rc, "gdn_selective_scan_bwd")
    return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0


class _SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, softplus):
        hT = torch.empty((x.shape[0], x.shape[2], A.shape[1]), dtype=torch.float32,
                         device=x.device)
        y, ck = _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, h0, hT, True)
        ctx.softplus, ctx.has_h0 = softplus, h0 is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, ck)
        return y, hT

    @staticmethod
    def backward(ctx, dy, dhT):
        if _batched(dy, dhT):
            raise NotImplementedError("selective_scan's backward takes no batched gradients")
        run = _SelectiveScanBwdFn.apply if torch.is_grad_enabled() else _scan_bwd
        return tuple(run(dy, dhT, *ctx.saved_tensors, ctx.has_h0, ctx.softplus)) + (None,)


class _SelectiveScanBwdFn(torch.autograd.Function):
    """The backward with create_graph=True: gradients that say so when they are
    differentiated, instead of being taken as constants."""

    @staticmethod
    def forward(ctx, *args):
        return _scan_bwd(*args)

    @staticmethod
    def backward(ctx, *dds):
        raise NotImplementedError("selective_scan has no second derivatives")


def selective_scan(x, dt, A, B, C, *, D=None, z=None, dt_bias=None, dt_softplus: bool = True,
                   initial_state=None, output_final_state: bool = False,
                   final_state_out: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Selective state-space scan (gdn_selective_scan_fwd), for prompts, training
    and single tokens.  Per row, channel c and token t, with an fp32 state h of
    N values::

        delta = softplus(dt + dt_bias[c])          # dt + dt_bias[c] without dt_softplus
        h     = exp(delta * A[c]) * h + delta * x * B[t]
        y     = (sum(C[t] * h) + D[c] * x) * silu(z)

    x, dt, z ``[B,T,Ch]`` and B, C ``[B,T,N]`` or ``[B,T,G,N]`` (channel c uses
    group ``c // (Ch // G)``) in one dtype, bfloat16 or float32, on a CUDA
    device; A ``[Ch,N]`` (negative in practice), D and dt_bias ``[Ch]`` (taken
    to float32; None: zero; z None: no gate); N up to 64.  Returns ``(y,
    state)`` like the recurrent op: state float32 ``[B,Ch,N]`` when
    ``output_final_state`` or ``final_state_out`` is given (decode:
    ``initial_state=S, final_state_out=S`` updates S in place; else they do not
    overlap), else None.
    Differentiable in every tensor, through y and the returned state (without
    ``final_state_out``; gdn_selective_scan_bwd), once: second derivatives raise
    NotImplementedError.  Its layer feeds x through
    :func:`short_convolution` first.
    """
    _cuda_input("x", x)
    if x.dim() != 3:
        raise ValueError(f"x must be [B,T,Ch]; got {tuple(x.shape)}")
    dev, dtype, shape_x = x.device, x.dtype, x.shape
    _check_input("dt", dt, dev, dtype)
    _check_input("B", B, dev, dtype)
    _check_input("C", C, dev, dtype)
    if z is not None:
        _check_input("z", z, dev, dtype)
    _check_sizes("x", shape_x)
    b, T, ch = shape_x
    if dt.shape != shape_x or (z is not None and z.shape != shape_x):
        raise ValueError(f"dt and z must have x's shape {tuple(shape_x)}")
    A = _on(A, dev)
    if A.dim() != 2 or A.shape[0] != ch:
        raise ValueError(f"A must be [{ch},N]; got {tuple(A.shape)}")
    N = A.shape[1]
    if B.dim() == 3:
        B = B.unsqueeze(2)
    if C.dim() == 3:
        C = C.unsqueeze(2)
    G = B.shape[2] if B.dim() == 4 else 0
    if B.shape != (b, T, G, N) or C.shape != B.shape:
        raise ValueError(f"B and C must be [{b},{T},{N}] or [{b},{T},G,{N}]; got "
                         f"{tuple(B.shape)}, {tuple(C.shape)}")
    _check_sizes("B", B.shape)
    if G < 1 or ch % G:
        raise ValueError(f"x's {ch} channels must be a multiple of the {G} groups of B and C")
    if D is not None:
        D = _on(D, dev)
        if D.shape != (ch,):
            raise ValueError(f"D must be [{ch}]; got {tuple(D.shape)}")
    if dt_bias is not None:
        dt_bias = _on(dt_bias, dev)
        if dt_bias.shape != (ch,):
            raise ValueError(f"dt_bias must be [{ch}]; got {tuple(dt_bias.shape)}")
    shape = (b, ch, N)
    if initial_state is not None and (initial_state.shape != shape
                                      or initial_state.device != dev):
        raise ValueError(f"initial_state must be {shape} on {dev}")
    softplus = int(bool(dt_softplus))
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, initial_state):
        if final_state_out is not None:
            raise NotImplementedError("the backward does not cover final_state_out")
        y, hT = _SelectiveScanFn.apply(
            _aligned(x), _aligned(dt), _aligned32(A), _aligned(B), _aligned(C), _aligned32(D),
            _aligned(z), _aligned32(dt_bias), _aligned32(initial_state), softplus)
        return y, hT if output_final_state else None
    hT = final_state_out
    if hT is not None:
        if (hT.shape != shape or hT.dtype != torch.float32 or not hT.is_contiguous()
                or hT.device != dev or hT.data_ptr() % 16):
            raise ValueError(f"final_state_out must be a contiguous, 16-byte aligned float32 "
                             f"{shape} tensor on {dev}")
    elif output_final_state:
        hT = torch.empty(shape, dtype=torch.float32, device=dev)
    y, _ = _scan_fwd(_aligned(x), _aligned(dt), _aligned32(A), _aligned(B), _aligned(C),
                     _aligned32(D), _aligned(z), _aligned32(dt_bias), softplus,
                     _aligned32(initial_state), hT, False)
    return y, hT


def gated_rms_norm(o, gate=None, weight=None, eps: float = 1e-5, *,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """FusedRMSNormGated (model.py:41-53) on the GPU (gdn_gated_rmsnorm_fwd):
    ``o * rsqrt(mean(o^2, -1) + eps) * weight``, times ``silu(gate)`` when a
    gate is given.  o ``[..., dv]`` bfloat16 or float32; gate like o or None;
    weight ``[dv]`` (None: ones).  ``out`` may be o (in place)."""
    _wants_grad(o, gate, weight)   # (inference only; tangents raise)
    if not (isinstance(o, torch.Tensor) and o.is_cuda and o.dtype in _DTYPES):
        raise ValueError("o must be a bfloat16 or float32 CUDA tensor")
    dv = o.shape[-1]
    o = o.contiguous()
    if gate is not None:
        if gate.shape != o.shape:
            raise ValueError(f"gate must have o's shape {tuple(o.shape)}")
        gate = gate.to(dtype=o.dtype).contiguous()
        if gate.data_ptr() % 16:
            gate = gate.clone()
    w = torch.ones(dv, dtype=torch.float32, device=o.device) if weight is None else \
        torch.as_tensor(weight, device=o.device).to(torch.float32).contiguous()
    if w.shape != (dv,):
        raise ValueError(f"weight must be [{dv}]")
    y = torch.empty_like(o) if out is None else out
    if y.shape != o.shape or y.dtype != o.dtype or not y.is_contiguous():
        raise ValueError("out must be a contiguous tensor of o's shape and dtype")
    lib = _lib.load()
    with torch.cuda.device(o.device):
        rc = lib.gdn_gated_rmsnorm_fwd(_ptr(o), _ptr(gate), _ptr(w), float(eps), _ptr(y),
                                       o.numel() // max(dv, 1), dv, _DTYPES[o.dtype],
                                       torch.cuda.current_stream(o.device).cuda_stream)
    _lib.check(rc, "gdn_gated_rmsnorm_fwd")
    return y


# Aliases with the reference's public names (ops.py:350-352).
fused_recurrent_gated_delta_rule_fwd = fused_recurrent_gated_delta_rule
fused_recurrent_gated_delta_rule_pallas = fused_recurrent_gated_delta_rule
chunk_gated_delta_rule = chunk_gated_delta_rule_fwd

__all__ = [
    "chunk_gated_delta_rule", "chunk_gated_delta_rule_fwd", "fused_recurrent_gated_delta_rule",
    "fused_recurrent_gated_delta_rule_fwd", "fused_recurrent_gated_delta_rule_pallas",
    "gated_delta_rule_decode_layer",
    "gated_delta_rule_chunk_layer",
    "short_convolution",
    "gated_rms_norm",
    "gated_linear_unit",
    "selective_scan",
]
