"""pa_accumulating_attention against its definition in 64 bits: outputs and accounts; types, heads, pages; steps,
prompts and mixed batches; rows that count; windows, softcaps, sinks; new tokens' slots that held anything."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import check, make_batch
from upkeep_cases import attention64, causal_seen

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def account(st, seed=0):
    """An account whose keys weigh something; the slots of new tokens, and all that no sequence holds, are NaN."""
    g = torch.Generator().manual_seed(seed)
    w = torch.full((st["kc"].shape[0], st["KV"], st["block"]), float("nan"))
    for b, past in enumerate(st["past"]):
        p = torch.arange(past)
        w[st["bt"][b].cpu().long()[p // st["block"]], :, p % st["block"]] = torch.rand(past, st["KV"], generator=g)
    return w.cuda()


def run(st, w, *, observed=0, scale=0.0, softcap=0.0, window=-1, causal=1, sink=None, **kw):
    kw = {"max_query_len": max(st["new"]), "max_context_len": max(st["total"]), **kw}
    return ep.accumulating_attention(
        st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], w, num_heads=st["H"], observed_rows=observed,
        scale=scale, softcap=softcap, local_window_size=window, is_causal=causal, head_sink=sink,
        k_scale=st["k_scale"], v_scale=st["v_scale"], k_quant_type=st["quant"], v_quant_type=st["quant"], **kw)


def compare(st, *, observed=0, window=-1, causal=1, call=None, **forms):
    w = account(st)
    old = w.clone()
    got = run(st, w, observed=observed, window=window, causal=causal, **forms, **(call or {}))
    seen = [causal_seen(n, p, window, causal) for n, p in zip(st["new"], st["past"])]
    want, tol, weights = attention64(st, seen, observed=observed, **forms)
    check(got[:want.shape[0]], want, tol)
    left = torch.ones_like(w, dtype=torch.bool)
    for b, (added, bound) in enumerate(weights):
        if st["new"][b] == 0:
            continue
        p = torch.arange(st["total"][b], device="cuda")
        at = st["bt"][b].long()[p // st["block"]], slice(None), p % st["block"]
        before = torch.where((p < st["past"][b])[:, None], old[at].double(), 0.0)
        exact = before + added.T
        check(w[at], exact, bound.T + 2.0 ** -23 * exact + 1e-30)
        left[at] = False
    assert torch.equal(w[left].view(torch.int32), old[left].view(torch.int32))  # nobody else's entries
    return got, w


LAYOUTS = [(BF16, 8, 2, 128, 16), (F16, 8, 2, 128, 32), (F16, 8, 1, 64, 16), (BF16, 6, 3, 96, 16),
           (BF16, 4, 1, 256, 16), (F16, 4, 2, 256, 256), (BF16, 16, 2, 64, 64), (F16, 7, 1, 128, 8),
           (BF16, 4, 4, 128, 24), (F16, 32, 2, 128, 16), (F32, 4, 2, 64, 16), (BF16, 4, 2, 80, 16),
           (F16, 3, 1, 40, 7), (F32, 2, 1, 256, 16)]
BATCHES = {"decode": ([1, 1, 1, 1, 1], [0, 1, 63, 64, 700]),
           "few": ([2, 0, 4, 1, 3], [9, 100, 31, 511, 1200]),
           "prompts": ([33, 1, 200, 65, 0, 129], [0, 0, 0, 40, 9, 333])}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace("torch.", "") for y in x))
def test_layouts(layout, batch):
    dt, H, KV, D, block = layout
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, seed=1)
    for observed in (0, 1, 3):
        compare(st, observed=observed)


FORMS = {"window_one": dict(window=1), "window": dict(window=17), "window_observed": dict(window=90, observed=7),
         "softcap": dict(softcap=5.0), "softcap_mid": dict(softcap=50.0), "softcap_large": dict(softcap=100.0),
         "sink": dict(sink=True), "both_sides": dict(causal=0), "both_sides_window": dict(causal=0, window=30),
         "scale": dict(scale=0.3), "negative_scale": dict(scale=-0.1), "more_observed": dict(observed=10000)}


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_forms(dt, D, form, batch):
    new, past = BATCHES[batch]
    st = make_batch(new, past, H=8, KV=2, D=D, block=16, dtype=dt, seed=2)
    f = dict(FORMS[form])
    if "sink" in f:
        f["sink"] = torch.linspace(-1, 2, 8).to(dt).cuda()
    compare(st, **f)


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8, torch.uint8])
def test_byte_coded_pages(kind):
    for new, past in (([1, 1, 1], [0, 77, 600]), ([20, 50], [100, 0])):
        for scales in (("PER_TENSOR", "PER_CHANNEL") if kind != torch.float8_e4m3fn else ("NONE",)):
            st = make_batch(new, past, H=4, KV=2, D=64, block=16, dtype=BF16, seed=8, cache_dtype=kind, scales=scales)
            compare(st, observed=30)


def test_long_steps_and_prompts():
    st = make_batch([1, 1, 2], [9001, 4095, 8192], H=32, KV=8, D=128, block=16, dtype=BF16, seed=9)
    compare(st)
    st = make_batch([1500, 700], [300, 2000], H=8, KV=2, D=128, block=16, dtype=F16, seed=10)
    compare(st)
    compare(st, observed=32)
    compare(st, window=400)
    st = make_batch([1200], [100], H=2, KV=1, D=256, block=16, dtype=BF16, seed=11)
    compare(st, softcap=30.0)


def test_bounds_unknown_and_rows_behind_the_last_sequence():
    for dt, D, new in ((BF16, 128, [1, 2]), (BF16, 128, [3, 40]), (F32, 64, [3, 40])):
        st = make_batch(new, [600, 3], H=8, KV=2, D=D, block=16, dtype=dt, seed=7, pad_tokens=5)
        out = torch.full_like(st["q"], 7.0)
        got, _ = compare(st, call=dict(max_query_len=0, max_context_len=0, out=out))
        assert got is out and bool((out[sum(new):] == 7.0).all())


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 64)])
@pytest.mark.parametrize("new", [1, 40])
def test_keys_that_are_not_finite(dt, D, new):
    """A NaN key makes the rows that see it NaN, and the accounts of what they see; nothing else."""
    st = make_batch([new, new], [100, 80], H=4, KV=2, D=D, block=16, dtype=dt, seed=12)
    j = 100 + new - 1
    st["kc"][st["bt"][0, j // 16].long(), j % 16, 0, 3] = float("nan")
    w = account(st)
    old = w.clone()
    out = run(st, w, window=50).view(-1, 4, D)
    assert torch.isnan(out[new - 1, :2]).all() and torch.isfinite(out[:new - 1]).all() and torch.isfinite(out[new:]).all()
    assert torch.isfinite(out[:, 2:]).all()
    p = torch.arange(100 + new, device="cuda")
    mine = w[st["bt"][0].long()[p // 16], :, p % 16]
    assert torch.isnan(mine[max(0, j - 49):, 0]).all() and torch.isfinite(mine[:max(0, j - 49), 0]).all()
    assert torch.isfinite(mine[:, 1]).all()
    p = torch.arange(80 + new, device="cuda")
    assert torch.isfinite(w[st["bt"][1].long()[p // 16], :, p % 16]).all()
    assert old.shape == w.shape


def test_values_that_are_not_finite_leave_the_account():
    for new in (1, 50):
        st = make_batch([new], [100], H=8, KV=2, D=128, block=16, dtype=BF16, seed=13)
        w0, w1 = account(st), account(st)
        run(st, w0)
        st["vc"][st["bt"][0, 2].long(), 5, 1, 7] = float("inf")
        out = run(st, w1)
        assert not torch.isfinite(out).all()
        p = torch.arange(100 + new, device="cuda")
        at = st["bt"][0].long()[p // 16], slice(None), p % 16
        assert torch.allclose(w0[at], w1[at], rtol=1e-5, atol=0.0)


def test_rows_of_the_account_add_up():
    """What a step adds to all keys is the rows' whole weight: one per row and head, without a sink."""
    for new, past in (([1] * 6, [0, 5, 100, 900, 64, 2000]), ([300, 20], [0, 700])):
        st = make_batch(new, past, H=8, KV=2, D=128, block=16, dtype=BF16, seed=15)
        w = torch.zeros(st["kc"].shape[0], 2, 16, device="cuda")
        run(st, w)
        assert abs(float(w.double().sum()) / (8 * sum(new)) - 1) < 1e-5


@pytest.mark.parametrize("new,past", [([1, 1, 2], [300, 5000, 100]), ([1, 300], [300, 100])])
def test_captured_and_replayed(new, past):
    st = make_batch(new, past, H=8, KV=2, D=128, block=16, dtype=BF16, seed=14)
    out, w = torch.empty_like(st["q"]), torch.zeros(st["kc"].shape[0], 2, 16, device="cuda")

    def call(out, w):
        return ep.accumulating_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], w, num_heads=8,
                                         max_query_len=max(new), max_context_len=max(st["total"]), out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out, w)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, w)
    for less in (0, 7, 99):
        st["past_t"].copy_(torch.tensor([p - less for p in past], dtype=torch.int32))
        start = torch.rand_like(w)
        eager_w = start.clone()
        eager = call(torch.empty_like(out), eager_w)
        for _ in range(2):
            w.copy_(start)
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(w, eager_w)


def test_two_streams_at_once_same_bits():
    sts = [make_batch([1] * 4 if i else [90, 1], [400 * (i + 1)] * (4 if i else 2), H=8, KV=2, D=128, block=16,
                      dtype=BF16, seed=20 + i) for i in range(2)]
    want = []
    for st in sts:
        w = account(st)
        want.append((run(st, w), w))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sts], [[], []]
    fresh = [[account(st) for _ in range(10)] for st in sts]
    torch.cuda.synchronize()
    for k in range(10):
        for i, (st, s) in enumerate(zip(sts, streams)):
            with torch.cuda.stream(s):
                got[i].append((run(st, fresh[i][k]), fresh[i][k]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, w in got[i]:
            assert torch.equal(o, want[i][0])
            assert torch.equal(w.view(torch.int32), want[i][1].view(torch.int32))


def test_steps_behind_long_tables():
    """More scores than are held: the keys are read again instead."""
    st = make_batch([1] * 4, [100, 50, 900, 3], H=32, KV=2, D=64, block=16, dtype=F16, seed=16, spare=140000)
    compare(st, call=dict(max_context_len=0))
    compare(st, call=dict(max_context_len=0), observed=1)
