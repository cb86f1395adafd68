"""Workspaces of trees and accounts over pages of other types under a bound on the contexts, on the host."""
from __future__ import annotations

import pytest

from onnxruntime_ep_mlx_amd import _capi as capi
from test_masked_host import BF16, attn, batch, cache
from test_upkeep_host import F32, sizes

FP8 = capi.PA_DTYPE_FP8_E4M3
# (types of pages and rows, head, tokens of each sequence, sequences, bound)
STEPS = [(F32, F32, 128, 32, 48, 1000), (F32, F32, 128, 1, 48, 600), (F32, F32, 64, 4000, 1, 4000),
         (FP8, BF16, 128, 32, 48, 1000), (FP8, BF16, 128, 512, 64, 512), (capi.PA_DTYPE_INT8, BF16, 256, 1, 3, 30),
         (BF16, BF16, 80, 20, 7, 8000), (BF16, BF16, 320, 1, 48, 600), (F32, F32, 512, 2, 30, 2000), (FP8, BF16, 640, 40, 8, 300)]


@pytest.mark.parametrize("pages,act,head,new,seqs,bound", STEPS)
def test_a_bound_is_worth_as_much_over_a_long_table(pages, act, head, new, seqs, bound):
    """What a call needs goes by the contexts that its bound allows, not by the table's capacity."""
    def need(positions, ctx):
        c = cache(nb=1 << 20, dt=pages, d=head, ks=4096, vs=4096, kq=capi.PA_QUANT_PER_TENSOR, vq=capi.PA_QUANT_PER_TENSOR)
        b = batch(tokens=new * seqs, batch=seqs, mb=positions // 16, mq=new, ctx=ctx)
        return sizes(c, b, attn(heads=32), act)[:2]

    short = need(8192, bound)
    for positions in (16384, 131072, 1 << 22):
        assert need(positions, bound) == short
    # (a tree's words and lags; an account's constants and its scores or sums, in fp32)
    tokens, keys = new * seqs, (bound + 63) // 64 * 64
    rows = tokens * 32
    assert short[0] <= tokens * 4 * ((new + 31) // 32 + 1) + max(rows, 1 << 14) * 8 * (head + 2) * 4 + 4096
    assert short[1] <= rows * 4 + max(rows, 32 * 2 * seqs) * keys * 4 + max(rows, 1 << 14) * 8 * (head + 2) * 4 + 4096
