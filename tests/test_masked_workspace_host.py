"""Sizes of the workspaces of pa_shared_prefix_attention: one partial row per row, item and worker that can leave
one, no more."""
from __future__ import annotations

import ctypes as C

import pytest

from onnxruntime_ep_mlx_amd import _capi as capi
from test_masked_host import BF16, FAKE, attn, batch, cache


def size(tokens, seqs, groups, heads=32, kv=8, d=128, prefix=0, mq=0, mb=1024):
    c, b = cache(kv=kv, d=d, nb=1 << 20), batch(tokens=tokens, batch=seqs, mq=mq, mb=mb)
    s = capi.PaSharedPrefix(FAKE, FAKE, groups, prefix)
    return capi.load().pa_shared_prefix_attention_workspace_bytes(C.byref(c), C.byref(b), C.byref(attn(heads)), C.byref(s), None,
                                                                  BF16)


@pytest.mark.parametrize("tokens,seqs,groups", [(6 * 8192, 6, 3), (64, 64, 1), (4096, 16, 4), (20000, 500, 30)])
@pytest.mark.parametrize("heads,kv,d", [(32, 8, 128), (64, 8, 64), (16, 2, 256)])
def test_shared_prefixes_ask_for_what_their_items_can_leave(tokens, seqs, groups, heads, kv, d):
    g, mq = heads // kv, -(-tokens // seqs)
    workers = 256 * {64: 3, 128: 2, 256: 1}[d]
    # blocks of up to 128 rows of sequences and groups, one more for each that does not fill its last
    own = kv * (tokens * g // 128 + seqs) if mq * g > 32 else 0
    shared = kv * (tokens * g // 128 + groups)
    rows = 128 * (own + shared + workers) + 32 * (4 * workers + kv * (seqs + groups))
    assert size(tokens, seqs, groups, heads, kv, d, mq=mq) <= rows * (d + 2) * 4 + (1 << 16)


def test_a_bound_on_the_prefixes_is_used():
    assert size(8, 8, 1, kv=1, heads=4, prefix=64, mq=1) <= size(8, 8, 1, kv=1, heads=4, prefix=0, mq=1)
    assert size(100, 2, 1, kv=1, heads=4, prefix=64, mq=50, mb=8) < size(100, 2, 1, kv=1, heads=4, prefix=0, mq=50, mb=8)
