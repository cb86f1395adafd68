"""A step in which no sequence has new tokens."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from test_gpu_accept_drafts import cum_of, drafts, verify
from test_gpu_evict_keys import setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_accepting_without_tokens(kind):
    """Empty paths; caches and accounts as they were."""
    nodes, past = [0, 0, 0], [100, 0, 33]
    for kw in (dict(), dict(max_path=4), dict(max_query_len=7)):
        st = setup(past, D=64, kind=kind)
        w = st["w"].clone()
        verify(st, past, nodes, drafts(nodes), key_weights=st["w"], **kw)
        assert torch.equal(st["w"], w)


def test_accepting_without_tokens_captured():
    st, past = setup([20, 7]), torch.tensor([20, 7], dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    cum = cum_of([0, 0])
    call = lambda: ep.accept_drafts(st["kc"], st["vc"], cum, past, st["table"], none.int(), none, none)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, lens, after = call()
    for _ in range(3):
        for x in (path, lens, after):
            x.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert path.tolist() == [[-1], [-1]] and lens.tolist() == [0, 0] and after.tolist() == [-1, -1]
