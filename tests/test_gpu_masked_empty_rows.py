"""Rows that see no key are zeros to the bit beside rows that see infinite and NaN values, and with queries of
their own that are not finite."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, make_batch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("odd", ["values", "query", "finite"])
@pytest.mark.parametrize("new,past", [([40], [100]), ([3], [200]), ([1, 150, 2], [70, 64, 1500])],
                         ids=["wide", "narrow", "mixed"])
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 256), (F32, 64)])
def test_rows_that_see_nothing_are_zero(dt, D, new, past, odd):
    st = make_batch(new, past, H=4, KV=1, D=D, block=16, dtype=dt, seed=50)
    starts, empty = [], []
    for n, p in zip(new, past):
        for r in range(n):
            none = r % 3 == (1 if n > 1 else 0)
            starts.append(p + n + 5 if none else 0)
            empty.append(none)
    empty = torch.tensor(empty, device="cuda")
    if odd == "values":
        for b in range(len(new)):
            for j, x in ((10, float("inf")), (20, float("nan")), (33, -float("inf"))):
                page, row = st["bt"][b, j // 16].long(), j % 16
                for s in ("vc", "vd"):
                    st[s][page, row, 0, 5 + j % 7] = x
    elif odd == "query":
        st["q"][empty, 7] = float("nan")
        st["q"][empty, D + 3] = float("inf")
    got = ep.masked_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=4,
                              document_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                              max_query_len=max(new), max_context_len=max(st["total"]))
    assert not got[empty].contiguous().view(torch.uint8).any()
    if odd == "query":
        st["q"] = st["q"].nan_to_num(0.0, 0.0, 0.0)
    check(got, *attention64(st, starts=starts))
