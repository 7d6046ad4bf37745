"""Refusals and host-side logic of the block operators that were once missing
(without a GPU)."""

import ctypes

import pytest
import torch

import block_refs as refs
from gated_deltanet_jax_b200 import _build, _lib, ops

BF16, FP32 = _lib.GDN_DTYPE_BF16, _lib.GDN_DTYPE_FP32
INVALID = _lib.GDN_ERR_INVALID


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        _build.build()
    return _lib.load()


def _at(n):
    return ctypes.c_void_p(n << 20)


@pytest.mark.parametrize("out,other", [("dx", "x"), ("dx", "dy"), ("dx", "st"), ("dx", "ds"),
                                       ("dst", "x"), ("dst", "dy"), ("dst", "st"), ("dst", "ds"),
                                       ("dst", "dx")])
def test_conv_backward_refuses_its_inputs_as_outputs(lib, out, other):
    """The final window's gradient is read after the entering one's was written."""
    a = dict(x=_at(1), w=_at(2), st=_at(3), dy=_at(4), ds=_at(5), dx=_at(6), dw=_at(7),
             dst=_at(8))
    a[out] = a[other]
    need = lib.gdn_short_conv_bwd_workspace_bytes(2, 1000, 64, 4)
    assert lib.gdn_short_conv_bwd(a["x"], a["w"], None, a["st"], a["dy"], a["ds"], a["dx"],
                                  a["dw"], None, a["dst"], 2, 1000, 64, 4, 1, BF16, _at(9), need,
                                  None) == INVALID
    assert b"may not be" in lib.gdn_last_error()


# ---------------------------------------------------------------------------
# second derivatives: the autograd functions with the library's calls replaced by
# the 64-bit references
# ---------------------------------------------------------------------------

def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.fixture
def reference_calls(monkeypatch):
    def conv_fwd(x, w, bias, s_in, s_out, act):
        o = refs.conv_ref(x, w, bias, s_in, act=bool(act))
        s_out.copy_(o["state"])
        return o["y"]

    def conv_bwd(dy, ds, x, w, bias, st, act):
        o = refs.conv_ref(x, w, bias, st, act=bool(act),
                          dy=torch.zeros_like(x) if dy is None else dy, dstate=ds)
        return (o["dx"], o["dw"], None if bias is None else o["dbias"],
                None if st is None else o["dstate"])

    def glu_fwd(x, wg, wu, keep):
        g, u = x @ wg.T, x @ wu.T
        return refs.silu(g) * u, g, u

    def glu_bwd(dh, x, wg, wu, g, u, need_x, need_w):
        o = refs.glu_ref(x, wg, wu, dh)
        return (o["dx"] if need_x else None,) + ((o["dwg"], o["dwu"]) if need_w else (None, None))
    for name, fn in (("_short_conv_fwd", conv_fwd), ("_short_conv_bwd", conv_bwd),
                     ("_glu_fwd", glu_fwd), ("_glu_bwd", glu_bwd)):
        monkeypatch.setattr(ops, name, fn)


@pytest.mark.parametrize("act", [1, 0])
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("T,K", [(5, 4), (2, 4), (3, 1), (0, 3)])
def test_conv_second_derivatives(reference_calls, act, full, T, K):
    x, w = _rand(2, T, 3, seed=1), _rand(K, 3, seed=2)
    bias, st = (_rand(3, seed=3), _rand(2, K - 1, 3, seed=4)) if full else (None, None)
    leaves = [t.requires_grad_(True) for t in (x, w, bias, st) if t is not None]

    def fn(*a):
        a = iter(a)
        return ops._ShortConvFn.apply(*(None if t is None else next(a) for t in (x, w, bias, st)),
                                      act)
    assert torch.autograd.gradgradcheck(fn, leaves)


@pytest.mark.parametrize("needs", [(True, True, True), (True, False, False), (False, True, False)])
def test_glu_second_derivatives(reference_calls, needs):
    ts = [_rand(*s, seed=i).requires_grad_(n) for i, (s, n) in enumerate(
        zip([(4, 3), (2, 3), (2, 3)], needs))]
    assert torch.autograd.gradgradcheck(ops._GluFn.apply, ts)


def test_second_derivatives_are_taken_once(reference_calls):
    """Where one input is a function of another, its share flows through it alone."""
    x = _rand(1, 6, 3, seed=1).requires_grad_(True)

    def penalty(conv):
        (g,) = torch.autograd.grad(conv(x, torch.tanh(x[0, :4])).square().sum(), x,
                                   create_graph=True)
        return torch.autograd.grad(g.square().sum(), x)[0]
    a = penalty(lambda v, w: ops._ShortConvFn.apply(v, w, None, None, 1)[0])
    b = penalty(lambda v, w: refs.conv_ref(v, w)["y"])
    assert torch.allclose(a, b, rtol=1e-9, atol=1e-12)
    # a third derivative, and a sum whose incoming gradient is a constant
    (g,) = torch.autograd.grad(ops._ShortConvFn.apply(x, x[0, :4], None, None, 1)[0].sum(), x,
                               create_graph=True)
    assert g.requires_grad
    (h,) = torch.autograd.grad(g.square().sum(), x, create_graph=True)
    assert torch.autograd.grad(h.sum(), x)[0].shape == x.shape


def test_batched_gradients(reference_calls):
    x, w = _rand(2, 5, 3, seed=1).requires_grad_(True), _rand(4, 3, seed=2).requires_grad_(True)
    y, s = ops._ShortConvFn.apply(x, w, None, None, 1)
    d = _rand(3, *y.shape, seed=5)
    got = torch.autograd.grad(y, (x, w), d, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(y, (x, w), d[i], retain_graph=True)):
            assert torch.allclose(a[i], b, rtol=1e-10, atol=1e-12)
    ts = [_rand(*q, seed=i).requires_grad_(True) for i, q in enumerate([(4, 3), (2, 3), (2, 3)])]
    h = ops._GluFn.apply(*ts)
    d = _rand(3, *h.shape, seed=6)
    got = torch.autograd.grad(h, ts, d, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(h, ts, d[i], retain_graph=True)):
            assert torch.allclose(a[i], b, rtol=1e-10, atol=1e-12)


def test_scan_says_that_it_has_no_second_derivatives(monkeypatch):
    """Gradients with create_graph=True are as before; differentiating them raises."""
    names = ["x", "dt", "A", "B", "C", "D", "z", "dt_bias"]

    def fwd(x, dt, A, B, C, D, z, dt_bias, softplus, h0, hT, keep):
        o = refs.scan_ref(x, dt, A, B, C, D, z, dt_bias, h0, softplus=bool(softplus))
        hT.copy_(o["state"])
        return o["y"], torch.zeros(1)

    def bwd(dy, dhT, *a):
        *ts, ck, has_h0, softplus = a
        o = refs.scan_ref(*ts, softplus=bool(softplus), dy=dy, dhT=dhT)
        return tuple(None if t is None else o["d" + ("dt_bias" if n == "dt_bias" else n)]
                     for n, t in zip(names, ts)) + (None,)
    monkeypatch.setattr(ops, "_scan_fwd", fwd)
    monkeypatch.setattr(ops, "_scan_bwd", bwd)
    ts = [_rand(1, 5, 4, seed=1), _rand(1, 5, 4, seed=2), -_rand(4, 2, seed=3).abs(),
          _rand(1, 5, 1, 2, seed=4), _rand(1, 5, 1, 2, seed=5), _rand(4, seed=6),
          _rand(1, 5, 4, seed=7), _rand(4, seed=8)]
    ts = [t.requires_grad_(True) for t in ts]
    y, _ = ops._SelectiveScanFn.apply(*ts, None, 1)
    dy = torch.ones_like(y)
    plain = torch.autograd.grad(y, ts, dy, retain_graph=True)
    kept = torch.autograd.grad(y, ts, dy, create_graph=True)
    assert all(torch.equal(a, b) and b.requires_grad for a, b in zip(plain, kept))
    with pytest.raises(NotImplementedError, match="second"):
        torch.autograd.grad(kept[0].square().sum(), ts)
    with pytest.raises(NotImplementedError, match="batched"):
        torch.autograd.grad(y, ts, dy[None].expand(2, *y.shape), is_grads_batched=True)


def test_tangents_are_refused():
    """Forward mode: a dual tensor asks for no gradient, and its tangent would be lost."""
    fw = torch.autograd.forward_ad
    x = torch.randn(3)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones(3))
        assert not ops._wants_grad(x, None, 1.0)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward"):
                ops._wants_grad(x, None, dual)
        assert ops._wants_grad(x, x.clone().requires_grad_(True))
    assert not ops._wants_grad(x)

    def fn(v):
        ops._wants_grad(v)
        return v
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(fn, (x,), (torch.ones(3),))


def test_conv_lengths(lib):
    """T up to 2^31 - 64, and 2^30 where the state is updated in place."""
    def fwd(T, si=None, so=None, dtype=BF16):
        return lib.gdn_short_conv_fwd_bias(_at(1), _at(2), None, si, so, None, 1, T, 8, 4, 1, dtype,
                                           None)
    assert fwd((1 << 31) - 63) == INVALID and b"too large" in lib.gdn_last_error()
    assert fwd((1 << 31) - 64) == INVALID and b"non-NULL" in lib.gdn_last_error()    # y is
    assert lib.gdn_short_conv_fwd_bias(_at(1), _at(2), None, _at(3), _at(3), _at(4), 1,
                                       (1 << 30) + 1, 8, 4, 1, BF16, None) == INVALID
    assert b"in place" in lib.gdn_last_error()
    # the backward's partial rows: a tile for each of 65535 blocks at most
    rows = lib.gdn_short_conv_bwd_workspace_bytes(1, (1 << 31) - 64, 8, 4) // (5 * 8 * 4)
    assert 1000 < rows <= 65535


def test_sizes_past_32_bits_are_refused():
    ops._check_sizes("x", (3, (1 << 31) - 1))
    ops._check_sizes("x", ())
    with pytest.raises(ValueError, match="x is too large"):
        ops._check_sizes("x", (0, 1 << 31))


def test_scan_states_overlap_wholly_or_not_at_all(lib):
    b, T, ch, N = 2, 5000, 8, 16
    n = b * ch * N * 4

    def fwd(h0, hT):
        return lib.gdn_selective_scan_fwd(_at(1), _at(2), _at(3), _at(4), _at(5), None, None, None,
                                          ctypes.c_void_p(h0), _at(6), ctypes.c_void_p(hT), None,
                                          b, T, ch, N, 1, 1, BF16, None, 0, None)
    at = 64 << 20
    for off in (16, n - 16, -16, 16 - n):
        assert fwd(at, at + off) == INVALID and b"apart" in lib.gdn_last_error(), off
    for off in (0, n, -n):                # refused for the workspace that is missing
        assert fwd(at, at + off) == INVALID and b"workspace" in lib.gdn_last_error(), off


PLAN_CHECK = r"""
#include <cstdio>
#include "glu_few_plan.h"
int main() {
  long long bad = 0, seen = 0;
  const int sms[] = {148, 132, 1};
  const int widths[] = {8, 64, 72, 256, 264, 1000, 2048, 4096, 5632, 11008, 28672, 131072, 1 << 20,
                        1 << 30};
  for (int s : sms)
    for (int M = 1; M <= gdn::kFewTokens; ++M)
      for (int D : widths)
        for (int I : widths) {
          if (D > 131072) continue;
          const gdn::FewPlan p = gdn::few_plan(M, D, I, s);
          bool ok = p.fits() && p.stages <= gdn::kFewMaxStages;
          ok = ok && p.n >= M && p.n <= 128 && p.cols >= p.n && p.split * p.share >= M;
          ok = ok && p.split <= gdn::kFewMaxSplit && p.kblocks >= p.split && p.share % 4 == 0;
          // static shared memory below 1 KB, 1 KB kept by the system, 228 KB an SM
          ok = ok && (p.smem + 2048) * (p.smem > 113 * 1024 ? 1 : 2) <= 228 * 1024;
          ok = ok && p.stage_bytes() % 1024 == 0 && (long long)p.tiles * 64 >= I;
          ++seen;
          if (!ok && ++bad < 5) std::printf("M=%d D=%d I=%d sms=%d\n", M, D, I, s);
        }
  std::printf("%lld of %lld\n", bad, seen);
  return bad != 0;
}
"""


def test_glu_few_token_layout_stays_in_its_memory(tmp_path):
    """Stages, exchange and TMEM columns of the kernel for few tokens, over its sizes."""
    import subprocess
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PLAN_CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", _build.CSRC, str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("0 of 64512"), r.stdout


def test_glu_kept_types(lib):
    """g and u in the inputs' type or fp32."""
    def fwd(dtype, kept):
        return lib.gdn_glu_fwd_kept(_at(1), _at(2), _at(3), None, _at(5), _at(6), 4, 64, 32, dtype,
                                    kept, None)
    for dtype, kept in ((FP32, BF16), (BF16, 7)):
        assert fwd(dtype, kept) == INVALID and b"kept" in lib.gdn_last_error()
    for dtype, kept in ((FP32, FP32), (BF16, FP32), (BF16, BF16)):
        assert fwd(dtype, kept) == INVALID and b"h must be" in lib.gdn_last_error()
    assert lib.gdn_glu_bwd_kept(_at(1), _at(2), _at(3), _at(4), _at(5), _at(6), _at(7), _at(8),
                                _at(9), 4, 64, 32, FP32, BF16, _at(10), 1 << 20, None) == INVALID
