"""What multi_axis_rotary_append's wrapper hands to the library, on the host: whatever the strides of its tensors,
no row or position that the descriptors name lies outside their memory (the library call itself is recorded, not
made)."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from onnxruntime_ep_mlx_amd import _capi as capi
from onnxruntime_ep_mlx_amd import ops

H, KV, D, HALF = 4, 2, 64, 32
BF16 = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_need_cuda", lambda name, t: None)
    monkeypatch.setattr(ops, "_on_device", lambda index, call, *args: made.append(args) or capi.PA_OK)
    return made


def inputs(T, **kw):
    rows = lambda n: torch.zeros(T, n * D, dtype=BF16)  # noqa: E731
    cache = lambda: torch.zeros(5, 16, KV, D, dtype=BF16)  # noqa: E731
    x = dict(query=rows(H), key=rows(KV), value=rows(KV), key_cache=cache(), value_cache=cache(),
             cum=torch.tensor([0, T], dtype=torch.int32), past=torch.zeros(1, dtype=torch.int32),
             block_table=torch.zeros(1, 4, dtype=torch.int32),
             positions=torch.arange(3 * T).view(3, T), cos_cache=torch.zeros(9, HALF, dtype=BF16),
             sin_cache=torch.zeros(9, HALF, dtype=BF16), num_heads=H, axis_sections=(8, 12, 12))
    x.update(kw)
    return x


def behind(t):
    """Elements of t's memory from its first on."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


@pytest.mark.parametrize("T", [1, 2, 7])
@pytest.mark.parametrize("form", ["dense", "expanded", "wide", "column", "one_axis"])
def test_positions_stay_in_their_tensor(calls, T, form):
    sections = (8, 12, 12)
    pos = torch.arange(3 * T).view(3, T)
    if form == "expanded":
        pos = torch.arange(T).expand(3, T)
    elif form == "wide":
        pos = torch.arange(3 * 40).view(3, 40)[:, 5:5 + T]
    elif form == "column":
        pos = torch.arange(T)[:, None].T.expand(3, T)
    elif form == "one_axis":
        pos, sections = torch.arange(T).expand(1, T), (HALF,)
    ep.multi_axis_rotary_append(**inputs(T, positions=pos, axis_sections=sections))
    rot = calls[0][10]._obj
    assert isinstance(rot, capi.PaAxisRotary) and rot.positions == pos.data_ptr()
    stride = rot.position_stride or T
    assert (rot.axes - 1) * stride + T <= behind(pos)
    # every frequency turns by its own axis' positions
    assert sum(rot.sections[:rot.axes]) == HALF
    axis = [a for a in range(rot.axes) for _ in range(rot.sections[a])]
    want = [a for a in range(len(sections)) for _ in range(sections[a])]
    flat = pos.as_strided((behind(pos),), (1,))
    for i in range(HALF):
        assert torch.equal(flat[axis[i] * stride:axis[i] * stride + T], pos[want[i]])


@pytest.mark.parametrize("T", [1, 2, 7])
@pytest.mark.parametrize("name,n", [("query", H), ("key", KV), ("value", KV)])
def test_broadcast_rows_are_refused(calls, name, n, T):
    row = torch.zeros(1, n * D, dtype=BF16).expand(T, n * D)
    if T > 1:
        with pytest.raises(ValueError, match=f"{name} .*overlap"):
            ep.multi_axis_rotary_append(**inputs(T, **{name: row}))
        # ... and rows that begin inside the one before
        with pytest.raises(ValueError, match=f"{name} .*overlap"):
            ep.multi_axis_rotary_append(**inputs(T, **{name: torch.zeros(T * n * D, dtype=BF16).as_strided((T, n * D), (8, 1))}))
        assert not calls
    else:  # a single row is dense whatever its stride
        ep.multi_axis_rotary_append(**inputs(T, **{name: row}))


@pytest.mark.parametrize("T", [1, 7])
def test_rows_stay_in_their_tensors(calls, T):
    wide = torch.zeros(T, (H + 2 * KV) * D + 24, dtype=BF16)
    q, k, v, _ = wide.split([H * D, KV * D, KV * D, 24], 1)
    ep.multi_axis_rotary_append(**inputs(T, query=q, key=k, value=v))
    args = calls[0]
    for t, ptr, ld in ((q, *args[4:6]), (k, *args[6:8]), (v, *args[8:10])):
        assert ptr == t.data_ptr() and ld >= t.shape[1] and (T - 1) * ld + t.shape[1] <= behind(t)
