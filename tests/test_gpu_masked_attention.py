"""pa_masked_attention against its definition in 64 bits: masks by document, prefix, window and
causality, distance biases, softcap, sinks; types, head layouts, page sizes; ragged batches with empty
sequences and rows that see nothing; NaN and infinities in places that nothing reads."""
from __future__ import annotations

import random

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, make_batch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def starts_of(st, lengths, seed=0):
    """Document starts of every packed token, documents of the given lengths in turn."""
    rng, out = random.Random(seed), []
    for new, past in zip(st["new"], st["past"]):
        at, begin = [], 0
        while len(at) < new + past:
            n = rng.choice(lengths)
            at += [begin] * n
            begin += n
        out += at[past:past + new]
    return out


def run(st, *, scale=0.0, softcap=0.0, window=-1, causal=1, sink=None, slopes=None, prefix=None,
        starts=None, **kw):
    dev = st["q"].device
    i32 = lambda x: None if x is None else torch.tensor(list(x), dtype=torch.int32, device=dev)  # noqa: E731
    kw = {"max_query_len": max(st["new"]), "max_context_len": max(st["total"]), **kw}
    return ep.masked_attention(
        st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=st["H"],
        scale=scale, softcap=softcap, local_window_size=window, is_causal=causal, head_sink=sink,
        distance_slopes=None if slopes is None else torch.as_tensor(slopes, dtype=F32).to(dev),
        prefix_lens=i32(prefix), document_starts=i32(starts), k_scale=st["k_scale"],
        v_scale=st["v_scale"], k_quant_type=st["quant"], v_quant_type=st["quant"], **kw)


def compare(st, **forms):
    call = {k: v for k, v in forms.items() if k.startswith("max_")}
    forms = {k: v for k, v in forms.items() if k not in call}
    got = run(st, **forms, **call)
    want, tol = attention64(st, **forms)
    check(got[:want.shape[0]], want, tol)
    return got


def slopes_of(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


LAYOUTS = [(BF16, 8, 2, 128, 16), (F16, 8, 2, 128, 32), (F16, 8, 1, 64, 16), (BF16, 6, 3, 96, 16),
           (BF16, 4, 1, 256, 16), (F16, 4, 2, 256, 256), (BF16, 16, 2, 64, 64), (F16, 7, 1, 128, 8),
           (BF16, 4, 4, 128, 24), (F16, 32, 2, 128, 16), (F32, 4, 2, 64, 16), (BF16, 4, 2, 80, 16),
           (F16, 3, 1, 40, 7), (F32, 2, 1, 256, 16)]
BATCHES = {"decode": ([1, 1, 1, 1, 1], [0, 1, 63, 64, 700]),
           "few": ([2, 0, 5, 1, 3], [9, 100, 31, 511, 1200]),
           "prompts": ([33, 1, 200, 65, 0, 129], [0, 0, 0, 40, 9, 333])}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace("torch.", "") for y in x))
def test_layouts(layout, batch):
    dt, H, KV, D, block = layout
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, seed=1)
    compare(st, slopes=slopes_of(H))
    compare(st, starts=starts_of(st, [1, 7, 40, 90]))


FORMS = {"plain": {}, "slopes": dict(slopes=True), "prefix": dict(prefix=[0, 5, 70, 64, 3, 4000]),
         "documents": dict(starts=[1, 3, 50]), "window": dict(window=17),
         "window_prefix": dict(window=40, prefix=[20, 1, 150, 60, 0, 400]),
         "softcap_sink": dict(softcap=5.0, sink=True),
         "all": dict(slopes=True, prefix=[4, 0, 90, 300, 1, 20], starts=[30, 80], window=100,
                     softcap=20.0, sink=True),
         "both_sides": dict(causal=0, slopes=True), "both_sides_documents": dict(causal=0, starts=[9, 64]),
         "scale": dict(scale=0.3), "negative_scale": dict(scale=-0.1, slopes=True)}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dt", [BF16, F16])
def test_forms(dt, form, batch):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=128, block=16, dtype=dt, seed=2)
    f = dict(FORMS[form])
    if "slopes" in f:
        f["slopes"] = slopes_of(8)
    if "prefix" in f:
        f["prefix"] = f["prefix"][:len(new)]
    if "starts" in f:
        f["starts"] = starts_of(st, f["starts"])
    if "sink" in f:
        f["sink"] = torch.linspace(-1, 2, 8).to(dt).cuda()
    compare(st, **f)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 256)])
def test_rows_that_see_nothing_are_zero(dt, D):
    st = make_batch([1, 40, 1, 3], [5, 0, 900, 70], H=4, KV=2, D=D, block=16, dtype=dt, seed=3)
    starts = [6] + [(100 if i % 3 else 0) for i in range(40)] + [2000] + [73, 0, 73]
    got = compare(st, starts=starts)
    rows = got.view(-1, 4 * D)
    assert not rows[0].any() and not rows[2].any() and not rows[41].any() and not rows[42].any()
    got = compare(st, starts=starts, sink=torch.zeros(4, dtype=dt, device="cuda"))
    assert not got.view(-1, 4 * D)[41].any()


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F16, 256), (F32, 64)])
def test_values_that_are_not_finite_stay_in_the_rows_that_see_them(dt, D):
    """Infinite and NaN values and keys behind a mask change nothing; rows that see them show them."""
    st = make_batch([70, 1, 3], [30, 200, 64], H=4, KV=1, D=D, block=16, dtype=dt, seed=4)
    bs = st["block"]
    for b, j, side, x in ((0, 55, "v", float("inf")), (0, 90, "v", float("nan")), (0, 20, "k", float("nan")),
                          (1, 10, "v", float("inf")), (2, 66, "v", -float("inf"))):
        at = st["bt"][b, j // bs].long(), j % bs, 0
        st[side + "c"][at[0], at[1], 0, 3] = x
        st[side + "d"][at[0], at[1], 0, 3] = x
    compare(st, starts=[0] * 5 + [21] * 30 + [56] * 35 + [11] + [0, 65, 66])
    compare(st, window=30)


def test_one_token_of_one_key():
    for dt in (BF16, F16, F32):
        st = make_batch([1], [0], H=2, KV=1, D=64, block=16, dtype=dt, seed=5)
        compare(st, slopes=[0.5, 0.25])
        # a single key: the output is its value, to the bit
        v = st["vc"][st["bt"][0, 0].long(), 0, 0]
        assert torch.equal(run(st).view(2, 64), v.expand(2, 64))


def test_no_tokens():
    st = make_batch([0, 0], [4, 0], H=4, KV=2, D=64, block=16, dtype=F16, seed=6)
    assert run(st, max_query_len=0).shape == (0, 256)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 64)])
def test_rows_behind_the_last_sequence_are_left_alone(dt, D):
    for new, past in (([1, 2], [600, 3]), ([130, 1], [9, 2000])):
        st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=7, pad_tokens=5)
        out = torch.full_like(st["q"], 7.0)
        got = run(st, slopes=slopes_of(8), out=out)
        want, tol = attention64(st, slopes=slopes_of(8))
        assert got is out and bool((out[sum(new):] == 7.0).all())
        check(out[:sum(new)], want, tol)


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8, torch.uint8])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_byte_coded_pages(dt, kind):
    for new, past in (([1, 1, 1], [0, 77, 600]), ([20, 50], [100, 0])):
        for scales in (("PER_TENSOR", "PER_CHANNEL") if kind != torch.float8_e4m3fn else ("NONE",)):
            st = make_batch(new, past, H=4, KV=2, D=64, block=16, dtype=dt, seed=8, cache_dtype=kind, scales=scales)
            compare(st, slopes=slopes_of(4), starts=starts_of(st, [5, 60]))


@pytest.mark.parametrize("dt,H,KV,D", [(BF16, 32, 8, 128), (F16, 64, 8, 64)])
def test_long_contexts(dt, H, KV, D):
    st = make_batch([1, 1, 2], [9001, 4095, 8192], H=H, KV=KV, D=D, block=16, dtype=dt, seed=9)
    compare(st, slopes=slopes_of(H))
    st = make_batch([300], [6000], H=H, KV=KV, D=D, block=16, dtype=dt, seed=10)
    compare(st, slopes=slopes_of(H), prefix=[6100])
    compare(st, starts=starts_of(st, [100, 2500]), window=3000)


def test_many_sequences():
    rng = random.Random(11)
    new = [rng.choice((0, 1, 1, 2)) for _ in range(700)]
    past = [rng.randrange(0, 90) for _ in range(700)]
    st = make_batch(new, past, H=4, KV=2, D=64, block=16, dtype=BF16, seed=11)
    compare(st, slopes=slopes_of(4))


@pytest.mark.parametrize("batch", ["decode", "prompts"])
def test_bounds_unknown(batch):
    """Without bounds on the lengths the results are the same."""
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=128, block=16, dtype=BF16, seed=12, spare=90)
    compare(st, slopes=slopes_of(8), max_query_len=0, max_context_len=0)


@pytest.mark.parametrize("batch", ["decode", "prompts"])
def test_plain_mask_agrees_with_paged_attention(batch):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=128, block=16, dtype=BF16, seed=13)
    rows = torch.zeros(sum(new), 2 * 128, dtype=BF16, device="cuda")
    a = ep.attention(st["q"], rows, rows, st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=8,
                     max_query_len=max(new), new_rows_in_cache=True)
    want, tol = attention64(st)
    check(a, want, tol)
    check(run(st), want, tol)


def test_captured_and_replayed():
    """A captured call gives the eager bits at every replay, over contexts that grow in between."""
    st = make_batch([1, 1, 40], [300, 5000, 100], H=8, KV=2, D=128, block=16, dtype=BF16, seed=14)
    slopes = torch.tensor(slopes_of(8), device="cuda")
    out = torch.empty_like(st["q"])

    def call(out):
        return ep.masked_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=8,
                                   distance_slopes=slopes, max_query_len=40, max_context_len=5001, out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for past in ([300, 5000, 100], [299, 4000, 20], [0, 1, 0], [300, 4999, 99]):
        st["past_t"].copy_(torch.tensor(past, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_two_streams_at_once():
    sts = [make_batch([1] * 8, [400 * (i + 1)] * 8, H=8, KV=2, D=128, block=16, dtype=BF16, seed=20 + i)
           for i in range(2)]
    want = [run(st, slopes=slopes_of(8)) for st in sts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sts]
    got = [[], []]
    for _ in range(20):
        for i, (st, s) in enumerate(zip(sts, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(st, slopes=slopes_of(8)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_same_bits_every_time():
    st = make_batch([1, 30, 1], [3000, 700, 10], H=8, KV=2, D=128, block=16, dtype=F16, seed=30)
    first = run(st, slopes=slopes_of(8))
    for _ in range(5):
        assert torch.equal(run(st, slopes=slopes_of(8)), first)
