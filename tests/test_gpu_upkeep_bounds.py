"""Trees and accounts over pages of other types behind long tables: contexts at a small bound, and beyond it."""
from __future__ import annotations

import pytest
import torch

import test_gpu_accumulating_attention as weigh
import test_gpu_tree_attention as tree
from masked_cases import check, make_batch
from upkeep_cases import attention64, causal_seen, trees

pytestmark = pytest.mark.gpu

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
KINDS = [(F32, 64, None), (BF16, 80, None), (BF16, 128, FP8), (BF16, 256, torch.int8), (BF16, 320, None), (F32, 264, FP8)]
BATCHES = [([1, 2, 1], [300, 998, 0]), ([32, 7, 0, 30], [70, 993, 64, 400])]


@pytest.mark.parametrize("new,past", BATCHES, ids=["step", "rows"])
@pytest.mark.parametrize("dt,D,kind", KINDS)
def test_small_bounds_over_long_tables(dt, D, kind, new, past):
    st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=1, cache_dtype=kind, spare=60000)
    for bound in (1000, 1024, 100000):
        tree.compare(st, trees(st), call=dict(max_context_len=bound))
        weigh.compare(st, call=dict(max_context_len=bound))
        weigh.compare(st, observed=1, window=150, call=dict(max_context_len=bound))


@pytest.mark.parametrize("new,past", BATCHES, ids=["step", "rows"])
@pytest.mark.parametrize("dt,D,kind", KINDS)
def test_contexts_beyond_the_bound(dt, D, kind, new, past):
    """Outputs do not go by the bound: the last chunk goes to the sequence's end."""
    st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=2, cache_dtype=kind, spare=9000)
    want, tol, _ = attention64(st, [causal_seen(n, p) for n, p in zip(new, past)])
    for bound in (1, 128, 129, 500, 999):
        tree.compare(st, trees(st), call=dict(max_context_len=bound))
        check(weigh.run(st, weigh.account(st), max_context_len=bound), want, tol)
