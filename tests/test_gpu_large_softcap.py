"""Softcaps far above the scores act as none: matrix-core decode, prefill, coded pages and LATENT rows against the
oracle, whose tanh keeps the bits of small arguments.

Bars: rel-L2 <= 2e-3 against the oracle rounded to T and <= 4e-3 against its float64 result, as without a softcap
(a score off by d moves the output by about d; steps of a cap of 1e5 are 2^-7)."""
from __future__ import annotations

import numpy as np
import pytest

import _oracle as orc
from _oracle import BF16, F16, I8
from pa_cases import make_case, make_latent_case, run_gpu_op
from test_gpu_fp8_prefill import fp8_case
from test_gpu_heads import decode_case

pytestmark = pytest.mark.gpu

CAPS = [65.0, 1e5, 1e6, 1e30, 3e38]


def check(case):
    ref, ref_t, _, _ = orc.paged_attention_op(case)
    out, _, _ = run_gpu_op(case)
    dt = case["dtype"]
    got = orc.decode(out, dt).astype(np.float64)
    assert np.isfinite(got).all()
    assert orc.rel_l2(got, orc.decode(ref_t, dt)) <= 2e-3
    assert orc.rel_l2(got, ref) <= 4e-3


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256), (F16, 96)])
def test_decode(dtype, d, cap):
    check(decode_case(d, dtype, seed=d, softcap=cap))
    check(decode_case(d, dtype, seed=d + 1, nq=3, softcap=cap))


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (F16, 64), (BF16, 256), (BF16, 96)])
def test_prompts(dtype, d, cap):
    check(make_case(8, 2, d, 4 * 48, 16, 4, dtype=dtype, seed=d, new_lens=[150, 0, 37, 200], past=np.array([300, 50, 0, 500]),
                    max_blocks=48, std=1.0, softcap=cap))


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("new", [[150, 0, 37, 200], [1, 1, 1, 1]], ids=["prompts", "step"])
def test_coded_pages(new, cap):
    check(fp8_case(128, BF16, new_lens=new, std=1.0, softcap=cap))
    check(make_case(8, 2, 128, 4 * 48, 16, 4, dtype=F16, cache_dtype=I8, seed=3, new_lens=new, past=np.array([300, 50, 0, 500]),
                    max_blocks=48, softcap=cap))


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("H", [16, 64])
def test_latent_rows(H, cap):
    check(make_latent_case(H, 576, 512, 3 * 50, 16, 3, dtype=BF16, seed=H, new_lens=[1, 9, 2], past=np.array([600, 250, 0]),
                           max_blocks=50, do_rotary=1, rot_dim=64, rotary_offset=512, scale=192.0 ** -0.5, std=1.0,
                           softcap=cap))
