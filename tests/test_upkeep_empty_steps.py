"""A step in which no sequence has new tokens, as the wrappers hand it to the library, on the host."""
from __future__ import annotations

import torch

import onnxruntime_ep_mlx_amd as ep
from onnxruntime_ep_mlx_amd import _capi as capi
from onnxruntime_ep_mlx_amd import ops
from test_upkeep_host import tensors  # noqa: F401  (a fixture)


def test_accepting_without_tokens_gives_no_path(tensors, monkeypatch):  # noqa: F811
    """Empty trees are trees, not a given path, which the library knows by the parents' address."""
    t, made = tensors, []
    monkeypatch.setattr(ops, "_on_device", lambda index, call, *args: made.append(args[-1]._obj) or capi.PA_OK)
    none = torch.zeros(0, dtype=torch.int64)
    at = (t["kc"], t["vc"], t["i32"](0, 0, 0), t["past"], t["bt"])
    for kw in (dict(), dict(max_path=4), dict(max_query_len=3)):
        path, lens, after = ep.accept_drafts(*at, none.int(), none, none, **kw)
        assert path.shape == (2, kw.get("max_path") or kw.get("max_query_len") or 1) and lens.shape == after.shape == (2,)
        assert all((made[-1].parents, made[-1].tokens, made[-1].targets, made[-1].next_tokens))
    ep.accept_drafts(*at, path=t["bt"], path_lens=t["past"])
    assert not any((made[-1].parents, made[-1].tokens, made[-1].targets, made[-1].next_tokens))
