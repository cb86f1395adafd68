"""Calls of pa_masked_attention and pa_shared_prefix_attention that are refused on the host, before any device work
(the pointers are not memory): outputs that meet the queries, windows of no key."""
from __future__ import annotations

import ctypes as C

import pytest

from onnxruntime_ep_mlx_amd import _capi as capi
from test_masked_host import BF16, FAKE, attn, batch, cache, error

N = 4 * 8 * 128 * 2  # bytes of the queries of four tokens


def call(share, out, c, act):
    lib, b, a = capi.load(), batch(), attn()
    if share:
        s = capi.PaSharedPrefix(FAKE, FAKE, 1, 0)
        return lib.pa_shared_prefix_attention(C.byref(c), C.byref(b), C.byref(a), C.byref(s), None, act, FAKE, out, 4 * FAKE,
                                              1 << 40, None)
    return lib.pa_masked_attention(C.byref(c), C.byref(b), C.byref(a), None, act, FAKE, out, 4 * FAKE, 1 << 40, None)


@pytest.mark.parametrize("share", [False, True], ids=["masked", "shared"])
@pytest.mark.parametrize("off", [0, 16, 1024, N - 16, -16, -(N - 16)])
def test_out_over_the_queries_is_refused(share, off):
    assert call(share, FAKE + off, cache(), BF16) == capi.PA_ERR_INVALID_ARGUMENT
    assert "overlap" in error()


@pytest.mark.parametrize("share", [False, True], ids=["masked", "shared"])
@pytest.mark.parametrize("off", [0, 16, 2 * N - 16, -16])
def test_out_over_the_queries_is_refused_by_the_other_kernel_too(share, off):
    """32-bit rows, twice as long, run without matrix cores."""
    f32 = capi.PA_DTYPE_FLOAT32
    assert call(share, FAKE + off, cache(dt=f32), f32) == capi.PA_ERR_INVALID_ARGUMENT
    assert "overlap" in error()


@pytest.mark.parametrize("share", [False, True], ids=["masked", "shared"])
@pytest.mark.parametrize("act", [BF16, capi.PA_DTYPE_FLOAT32])
@pytest.mark.parametrize("window", [0, -2, -(1 << 31)])
def test_windows_of_no_key_are_refused(monkeypatch, share, act, window):
    monkeypatch.setitem(globals(), "attn", lambda: capi.PaAttn(8, 0.0, 0.0, window, 1, None, 0))
    assert call(share, 8 * FAKE, cache(dt=act), act) == capi.PA_ERR_INVALID_ARGUMENT
    assert "local_window_size" in error()
