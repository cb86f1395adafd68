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


@pytest.mark.parametrize("kw,text", [
    (dict(past=torch.zeros(0, dtype=torch.int32)), "inconsistent"),
    (dict(cum=torch.zeros(3, dtype=torch.int32)), "inconsistent"),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), "inconsistent"),
    (dict(block_table=torch.zeros(1, 2, 2, dtype=torch.int32)), "inconsistent"),
    (dict(past=torch.zeros(2, dtype=torch.int32), cum=torch.tensor([0, 3, 5], dtype=torch.int32)), "inconsistent"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), "slot_mapping"),
    (dict(key_cache=torch.zeros(5, 16, KV * D, dtype=BF16)), "key_cache"),
    (dict(value_cache=None), "value_cache"),
    (dict(key_cache=torch.zeros(5, 16, KV, D).to(torch.float8_e4m3fn), value_cache=torch.zeros(5, 16, KV, D).to(torch.float8_e4m3fn),
          k_scale=torch.ones(5, KV), v_scale=torch.ones(4, KV)), "v_scale"),
    (dict(key_cache=torch.zeros(5, 16, KV, D, dtype=torch.int8), value_cache=torch.zeros(5, 16, KV, D, dtype=torch.int8),
          k_quant_type="PER_CHANNEL", v_quant_type="PER_TENSOR", k_scale=torch.ones(1), v_scale=torch.ones(1)), "k_scale"),
    (dict(key_cache=torch.zeros(5, 16, KV, D, dtype=torch.int8), value_cache=torch.zeros(5, 16, KV, D, dtype=torch.int8),
          k_quant_type="PER_TENSOR", v_quant_type="PER_TENSOR", k_scale=torch.ones(1), v_scale=torch.ones(0)), "v_scale"),
], ids=lambda x: x if isinstance(x, str) else None)
def test_short_tensors_are_refused(calls, kw, text):
    """Every tensor that the library reads by the batch's and the cache's sizes holds as much."""
    with pytest.raises(ValueError, match=text):
        ep.multi_axis_rotary_append(**inputs(5, **kw))
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(k_scale=torch.ones(5, KV), v_scale=torch.ones(4, KV)),
    dict(k_scale=torch.ones(KV), v_scale=torch.ones(5, KV))])
def test_masked_attention_refuses_short_scales(calls, kw):
    x = inputs(5)
    cache = torch.zeros(5, 16, KV, D).to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="_scale"):
        ep.masked_attention(x["query"], cache, cache, x["cum"], x["past"], x["block_table"], num_heads=H, **kw)
    assert not calls


def test_every_tensor_is_looked_for_on_the_device(calls, monkeypatch):
    seen = set()
    monkeypatch.setattr(ops, "_same_device", lambda index, tensors, contiguous=True: seen.update(n for n, _ in tensors))
    cache = torch.zeros(5, 16, KV, D).to(torch.float8_e4m3fn)
    ep.multi_axis_rotary_append(**inputs(5, key_cache=cache, value_cache=cache, v_scale=torch.ones(5, KV), k_scale=torch.ones(5, KV)))
    assert seen == {"query", "value", "positions", "key_cache", "value_cache", "cum", "past", "block_table", "cos_cache",
                    "sin_cache", "q_norm_weight", "k_norm_weight", "slot_mapping", "q_out", "k_scale", "v_scale"}
