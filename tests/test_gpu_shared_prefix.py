"""pa_shared_prefix_attention against the definition of plain attention in 64 bits: groups of sequences
whose tables name the same pages for their first keys."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, make_batch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(st, group_cum, shared, *, slopes=None, prefix=None, starts=None, window=-1, softcap=0.0, sink=None,
        causal=1, scale=0.0, **kw):
    dev = st["q"].device
    i32 = lambda x: None if x is None else torch.tensor(list(x), dtype=torch.int32, device=dev)  # noqa: E731
    kw = {"max_query_len": max(st["new"]), "max_context_len": max(st["total"]),
          "max_prefix_len": max(shared), **kw}
    return ep.shared_prefix_attention(
        st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], i32(group_cum), i32(shared),
        num_heads=st["H"], softcap=softcap, local_window_size=window, head_sink=sink, is_causal=causal, scale=scale,
        distance_slopes=None if slopes is None else torch.as_tensor(slopes, dtype=F32).to(dev),
        prefix_lens=i32(prefix), document_starts=i32(starts), k_scale=st["k_scale"], v_scale=st["v_scale"],
        k_quant_type=st["quant"], v_quant_type=st["quant"], **kw)


def compare(st, group_cum, shared, call={}, **forms):
    got = run(st, group_cum, shared, **forms, **call)
    want, tol = attention64(st, **forms)
    check(got[:want.shape[0]], want, tol)
    return got


LAYOUTS = [(BF16, 8, 2, 128, 16), (F16, 8, 1, 64, 32), (BF16, 6, 3, 96, 16), (F16, 4, 1, 256, 16), (BF16, 7, 1, 128, 8),
           (F16, 32, 8, 128, 256), (F32, 4, 2, 64, 16), (BF16, 4, 2, 80, 24)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace("torch.", "") for y in x))
@pytest.mark.parametrize("shape", ["decode", "few", "prompts"])
def test_layouts(layout, shape):
    dt, H, KV, D, block = layout
    P = 6 * block if block < 100 else block
    new = {"decode": [1] * 9, "few": [3, 1, 0, 2, 5, 1, 1, 4, 2], "prompts": [40, 1, 200, 3, 0, 90, 17, 64, 1]}[shape]
    past = [P + 5, P, P + 90, P + 1, P + 33, 2 * P, 2 * P + 700, 2 * P + 3, 44]
    gc, sh = [0, 5, 8], [P, 2 * P]
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, seed=1, shared=sh, group_cum=gc)
    compare(st, gc, sh)


@pytest.mark.parametrize("form", [dict(softcap=4.0), dict(sink=True), dict(slopes=True), dict(window=100), dict(window=500),
                                  dict(prefix=[0, 300, 500, 7, 0, 900]), dict(starts=True), dict(causal=0), dict(scale=-0.07)],
                         ids=lambda f: "-".join(f))
@pytest.mark.parametrize("new", [[1] * 6, [2, 30, 1, 60, 1, 4]], ids=["decode", "mixed"])
def test_forms(form, new):
    gc, sh = [0, 4, 6], [320, 160]
    st = make_batch(new, [330, 320, 700, 400, 160, 1000], H=8, KV=2, D=128, block=16, dtype=BF16, seed=2, shared=sh, group_cum=gc)
    f = dict(form)
    if "sink" in f:
        f["sink"] = torch.linspace(-1, 2, 8).to(BF16).cuda()
    if "slopes" in f:
        f["slopes"] = [2.0 ** -(h + 1) for h in range(8)]
    if "starts" in f:
        f["starts"] = [(7 * i * i) % 900 for i in range(sum(new))]
    compare(st, gc, sh, **f)


def test_long_prefix_many_samples():
    new, past = [1] * 40, [8192 + 13 * i for i in range(40)]
    st = make_batch(new, past, H=16, KV=4, D=128, block=16, dtype=BF16, seed=3, shared=[8192], group_cum=[0, 40])
    compare(st, [0, 40], [8192])


def test_prefix_that_ends_inside_a_page_and_a_tile():
    """Lengths that are no multiple of a page: the pages are the same where the shared keys are."""
    for cut in (1, 17, 63, 65, 100, 127):
        st = make_batch([1, 2, 1], [128, 130, 300], H=8, KV=2, D=128, block=16, dtype=F16, seed=4, shared=[128], group_cum=[0, 3])
        compare(st, [0, 3], [cut])


def test_groups_of_one_of_none_and_sequences_outside():
    st = make_batch([1, 1, 1, 1, 1], [64, 80, 64, 90, 20], H=8, KV=2, D=128, block=16, dtype=F16, seed=5, shared=[0, 64], group_cum=[0, 1, 4])
    compare(st, [0, 1, 4], [64, 64])
    compare(st, [0, 0, 1, 4, 4], [9, 0, 64, 5])
    compare(st, [1, 4], [64])
    compare(st, [0, 5], [0])


def test_prefix_as_long_as_the_context():
    """The new tokens themselves shared (scoring the same prompt's last token again)."""
    st = make_batch([1, 1], [127, 127], H=4, KV=1, D=64, block=16, dtype=F16, seed=6, shared=[128], group_cum=[0, 2])
    compare(st, [0, 2], [128])
    compare(st, [0, 2], [4000], call=dict(max_prefix_len=4000))  # clamped to the keys that are there


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8, torch.uint8])
def test_byte_coded_pages(kind):
    st = make_batch([1, 1, 2], [130, 140, 300], H=8, KV=2, D=128, block=16, dtype=BF16, seed=7, shared=[128], group_cum=[0, 3],
                    cache_dtype=kind)
    compare(st, [0, 3], [128])


def test_values_that_are_not_finite():
    st = make_batch([2, 1], [128, 140], H=4, KV=1, D=128, block=16, dtype=F16, seed=8, shared=[128], group_cum=[0, 2])
    for j, x in ((100, float("inf")), (20, float("nan"))):
        at = st["bt"][0, j // 16].long()
        st["vc"][at, j % 16, 0, 5] = x
        st["vd"][at, j % 16, 0, 5] = x
    compare(st, [0, 2], [128], starts=[21, 101, 0])


def test_rows_behind_the_last_sequence_are_left_alone():
    st = make_batch([1, 1], [200, 300], H=8, KV=2, D=128, block=16, dtype=BF16, seed=9, shared=[192], group_cum=[0, 2], pad_tokens=3)
    out = torch.full_like(st["q"], 7.0)
    compare(st, [0, 2], [192], call=dict(out=out))
    assert bool((out[2:] == 7.0).all())


def test_many_groups_and_sequences():
    n = 400
    gc = list(range(0, n + 1, 4))
    sh = [16 * (1 + i % 5) for i in range(n // 4)]
    past = [sh[b // 4] + b % 37 for b in range(n)]
    st = make_batch([1] * n, past, H=4, KV=2, D=64, block=16, dtype=BF16, seed=10, shared=sh, group_cum=gc)
    compare(st, gc, sh)


def test_bounds_unknown():
    st = make_batch([1] * 5, [64 + i for i in range(5)], H=8, KV=2, D=128, block=16, dtype=BF16, seed=11, shared=[64], group_cum=[0, 5], spare=80)
    compare(st, [0, 5], [64], call=dict(max_query_len=0, max_context_len=0, max_prefix_len=0))


def test_captured_and_replayed():
    st = make_batch([1] * 12, [1030 + 9 * i for i in range(12)], H=8, KV=2, D=128, block=16, dtype=BF16, seed=12, shared=[1024], group_cum=[0, 12])
    gc, sh = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 12], [1024]))
    out = torch.empty_like(st["q"])

    def call(out):
        return ep.shared_prefix_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], gc, sh, num_heads=8,
                                          max_query_len=1, max_context_len=1200, max_prefix_len=1024, out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for prefix, more in ((1024, 0), (512, -3), (0, 0), (1000, -5)):
        sh.fill_(prefix)
        st["past_t"].copy_(torch.tensor([1030 + 9 * i + more for i in range(12)], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
