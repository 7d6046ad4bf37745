"""Refusals and host-side logic of the block operators that were once missing
(without a GPU)."""

import ctypes

import pytest

from gated_deltanet_jax_b200 import _build, _lib

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
