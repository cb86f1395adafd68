"""Trees and accounts on every kernel that serves them: captured and replayed, on two streams at once; what NaN keys
leave alone."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
import test_gpu_accumulating_attention as weigh
import test_gpu_tree_attention as tree
from masked_cases import make_batch
from upkeep_cases import packed, trees

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
# (type, head, pages): fp32 products, coded pages, the VALU kernel, matrix products
KINDS = [(F32, 64, None), (BF16, 128, FP8), (F16, 320, None), (BF16, 128, None)]
# few rows, blocks of them, trees whose bits a kernel of their own makes
BATCHES = [([1, 2, 1], [300, 2000, 100]), ([26, 9, 40], [300, 2000, 100]), ([70, 1, 129], [40, 1500, 300])]


def batch_of(kind, new, past, seed):
    dt, D, pages = kind
    return make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=seed, cache_dtype=pages)


def scales(st):
    return dict(k_scale=st["k_scale"], v_scale=st["v_scale"], k_quant_type=st["quant"], v_quant_type=st["quant"])


def captured(call):
    """A graph of call() after one call on a stream beside."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


@pytest.mark.parametrize("new,past", BATCHES, ids=["few", "rows", "nodes"])
@pytest.mark.parametrize("kind", KINDS, ids=["fp32", "fp8", "large_head", "bf16"])
def test_replays(kind, new, past):
    """Replays over other contexts and trees, eager calls between them, give the eager bits."""
    st = batch_of(kind, new, past, 14)
    held, w = packed(trees(st)), torch.zeros(st["kc"].shape[0], 2, 16, device="cuda")
    out, seen = torch.empty_like(st["q"]), torch.empty_like(st["q"])
    at = (st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"])
    kw = dict(num_heads=8, max_query_len=max(new), max_context_len=max(st["total"]), **scales(st))

    def call(out, seen, w):
        ep.tree_attention(*at, held, local_window_size=500, out=out, **kw)
        ep.accumulating_attention(*at, w, out=seen, **kw)
        return out, seen, w

    graph = captured(lambda: call(out, seen, w))
    for i, less in enumerate((0, 7, 39)):
        st["past_t"].copy_(torch.tensor([max(p - less, 0) for p in past], dtype=torch.int32))
        held.copy_(packed(trees(st, seed=i)))
        start = torch.rand_like(w)
        eager = call(torch.empty_like(out), torch.empty_like(seen), start.clone())
        for _ in range(3):
            w.copy_(start)
            out.fill_(float("nan"))
            seen.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip((out, seen, w), eager))


@pytest.mark.parametrize("kind", KINDS[:3], ids=["fp32", "fp8", "large_head"])
def test_two_streams_at_once(kind):
    sts = [batch_of(kind, *BATCHES[i], 20 + i) for i in (1, 2)]
    weights = [[weigh.account(st) for _ in range(7)] for st in sts]
    nodes = [packed(trees(st)) for st in sts]

    def call(i, w):
        st = sts[i]
        at = (st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"])
        kw = dict(num_heads=8, max_query_len=max(st["new"]), max_context_len=max(st["total"]), **scales(st))
        return ep.tree_attention(*at, nodes[i], **kw), ep.accumulating_attention(*at, w, **kw), w

    want = [call(i, weights[i][0]) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sts], []
    for k in range(1, 7):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, call(i, weights[i][k])))
    torch.cuda.synchronize()
    for i, (t, o, w) in got:
        assert torch.equal(t, want[i][0]) and torch.equal(o, want[i][1])
        assert torch.equal(w.view(torch.int32), want[i][2].view(torch.int32))


@pytest.mark.parametrize("kind", KINDS, ids=["fp32", "fp8", "large_head", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_nan_keys_leave_the_entries_of_nobody(kind, new):
    """Accounts of places that no sequence holds keep their bits."""
    st = batch_of(kind, [new, new], [100, 80], 12)
    j = 100 + new - 1
    at = st["bt"][0, j // 16].long(), j % 16, 0, 3
    if kind[2] is None:
        st["kc"][at] = float("nan")
    else:
        st["kc"].view(torch.uint8)[at] = 0x7f
    w = weigh.account(st)
    old = w.clone()
    out = weigh.run(st, w, window=50).view(-1, 8, kind[1])
    assert torch.isnan(out[new - 1, :4]).all() and torch.isfinite(out[:, 4:]).all() and torch.isfinite(out[new:]).all()
    left = torch.ones_like(w, dtype=torch.bool)
    for b, total in enumerate(st["total"]):
        p = torch.arange(total, device="cuda")
        left[st["bt"][b].long()[p // 16], :, p % 16] = False
    assert bool(left.any()) and torch.equal(w[left].view(torch.int32), old[left].view(torch.int32))
