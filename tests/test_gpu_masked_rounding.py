"""Probabilities of pa_masked_attention and pa_shared_prefix_attention enter the second product in two parts: the
outputs err as 32-bit arithmetic with one rounding does (bounds: masked_rounding.py)."""
from __future__ import annotations

import pytest

from masked_cases import check, make_batch
from masked_rounding import BATCHES, BF16, F16, narrow64, run, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_probabilities_keep_two_parts(dt, D, batch):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=40)
    forms = [{}, dict(slopes=slopes_of(8)), dict(window=37, prefix=[3, 0, 150, 70, 5, 9][:len(new)])]
    for form in forms:
        check(run(st, **form), *narrow64(st, **form))
    check(run(st, softcap=20.0), *narrow64(st, softcap=20.0))


@pytest.mark.parametrize("dt", [BF16, F16])
def test_shared_prefixes_keep_two_parts(dt):
    group_cum, shared = [0, 3, 5], [640, 320]
    for new in ([1, 1, 2, 1, 1, 1], [30, 1, 20, 1, 70, 40]):
        st = make_batch(new, [640, 700, 655, 320, 900, 17], H=8, KV=2, D=128, block=16, dtype=dt, seed=41,
                        group_cum=group_cum, shared=shared)
        check(run(st, group_cum=group_cum, shared=shared), *narrow64(st))
