"""Values and keys that are not finite in places that rows see: the definition's own infinities and NaN, and calls
that stay of the order of finite ones."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, make_batch
from masked_rounding import BF16, F16, run, slopes_of

pytestmark = pytest.mark.gpu


def put(st, b, j, side, d, x):
    page, row = st["bt"][b, j // st["block"]].long(), j % st["block"]
    for s in (side + "c", side + "d"):
        st[s][page, row, 0, d] = x


BATCHES = {"wide": ([90, 40], [20, 300]), "narrow": ([1, 3, 1], [200, 64, 900])}


@pytest.mark.parametrize("form", [{}, dict(slopes=True), dict(softcap=9.0), dict(softcap=500.0), dict(window=60)],
                         ids=["plain", "slopes", "cap", "far_cap", "window"])
@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F16, 96), (BF16, 256)])
def test_rows_show_what_they_see(dt, D, batch, form):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=4, KV=1, D=D, block=16, dtype=dt, seed=60)
    for b, p in enumerate(past):
        put(st, b, 7, "v", 5, float("inf"))
        put(st, b, p - 3, "v", D - 1, -float("inf"))
        put(st, b, p - 10, "v", 33, float("nan"))
    f = dict(form)
    if "slopes" in f:
        f["slopes"] = slopes_of(4)
    check(run(st, **f), *attention64(st, **f))


@pytest.mark.parametrize("dt", [BF16, F16])
def test_keys_that_are_nan_make_their_rows_nan(dt):
    for new, past in BATCHES.values():
        st = make_batch(new, past, H=4, KV=1, D=128, block=16, dtype=dt, seed=61)
        put(st, 0, past[0] - 1, "k", 3, float("nan"))
        starts = [(past[0] if r % 2 else 0) for r in range(new[0])] + [0] * sum(new[1:])
        got = run(st, starts=starts).view(sum(new), 4, 128)
        nan = torch.zeros(sum(new), dtype=torch.bool)
        nan[:new[0]:2] = True
        assert torch.isnan(got[nan]).all() and torch.isfinite(got[~nan]).all()


@pytest.mark.parametrize("dt", [BF16, F16])
def test_shared_prefixes_with_infinite_values(dt):
    for new in ([1, 1, 2, 1], [30, 1, 20, 50]):
        st = make_batch(new, [640, 700, 655, 320], H=4, KV=1, D=128, block=16, dtype=dt, seed=62, group_cum=[0, 3], shared=[640])
        put(st, 0, 100, "v", 9, float("inf"))
        put(st, 1, 690, "v", 10, float("nan"))
        put(st, 3, 3, "v", 11, -float("inf"))
        check(run(st, group_cum=[0, 3], shared=[640]), *attention64(st))


@pytest.mark.parametrize("side,x", [("k", float("nan")), ("v", float("inf")), ("v", float("nan"))])
def test_a_prompt_with_such_a_key_takes_no_thousand_times_as_long(side, x):
    """One key of 4096 that every row sees: rows one by one and key by key took 700 times a finite call."""
    st = make_batch([4096], [0], H=32, KV=8, D=128, block=16, dtype=BF16, seed=63)
    slopes = torch.tensor(slopes_of(32), device="cuda")

    def time():
        best = 1e9
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ep.masked_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=32,
                                distance_slopes=slopes, max_query_len=4096, max_context_len=4096)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    finite = time()
    st[side + "c"][st["bt"][0, 0].long(), 3, :, 7] = x
    assert time() < 100 * finite
