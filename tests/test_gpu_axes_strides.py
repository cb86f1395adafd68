"""pa_multi_axis_rotary_append with one row of positions expanded over the axes, against its definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_multi_axis import BF16, F16, F32, compare, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("distinct", [False, True], ids=["any_slots", "distinct"])
@pytest.mark.parametrize("new,past", [([1], [5]), ([1] * 9, [17 * i for i in range(9)]), ([40, 0, 3], [0, 9, 700])],
                         ids=["one", "step", "prompts"])
@pytest.mark.parametrize("dt,sections,turns", [(BF16, (16, 24, 24), False), (F16, (8, 12, 12), True), (F32, (8, 12, 12), True),
                                               (BF16, (32, 32), False)])
def test_positions_expanded_over_the_axes(dt, sections, turns, new, past, distinct):
    st = make(new, past, H=6, KV=2, D=2 * sum(sections), block=16, dtype=dt, sections=sections, turns=turns, norm=True)
    st["positions"] = st["positions"][1].clone().expand(len(sections), sum(new))
    assert st["positions"].stride(0) == 0
    compare(st, slots_distinct=distinct)
