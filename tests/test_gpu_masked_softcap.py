"""Softcaps of any size in pa_masked_attention: large ones act as none, to the scores' own bits (bounds:
masked_rounding.py, none of whose terms grows with the softcap)."""
from __future__ import annotations

import pytest

from masked_cases import check, make_batch
from masked_rounding import BATCHES, BF16, F16, narrow64, run, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [5.0, 50.0, 64.0, 65.0, 1e3, 3e4, 1e6, 1e30, 3e38])
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F16, 256)])
def test_softcaps_of_any_size(dt, D, softcap):
    for name, (new, past) in BATCHES.items():
        st = make_batch(new, past, H=4, KV=2, D=D, block=16, dtype=dt, seed=42, std=1.5)
        check(run(st, softcap=softcap), *narrow64(st, softcap=softcap))
        slopes = slopes_of(4)
        check(run(st, softcap=softcap, slopes=slopes), *narrow64(st, softcap=softcap, slopes=slopes))
