"""pa_multi_axis_rotary_append against its definition in 64 bits, and the path it feeds: images and text
appended with three-axis positions, a prompt under a prefix mask, then samples over the shared prompt.

Error bound of a finished element a c - b s (a, b normalised): u |x| for the one rounding, and
(|a c| + |b s|) (D + 16) 2^-24 for the fp32 norm (a sum of D squares, a root, a division, two products)
and the rotation's own roundings, times 1.01 for the products of these."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, half_step, make_batch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def axis_list(sections, interleaved):
    half, axes = sum(sections), len(sections)
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [(i % axes if i < axes * sections[i % axes] else 0) for i in range(half)]


def turned64(x, heads, st, w, eps):
    """Rows in 64 bits and their bound, [T, heads, D]."""
    T, D = x.shape[0], st["D"]
    x = x.double().reshape(T, heads, D)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half, off = sum(st["sections"]), st["offset"]
    idx = torch.arange(half, device=x.device)
    e1 = off + 2 * idx if st["pairs"] else off + idx
    e2 = e1 + 1 if st["pairs"] else e1 + half
    ids = st["positions"][torch.tensor(axis_list(st["sections"], st["turns"]), device=x.device)].T  # [T, half]
    ok = ((ids >= 0) & (ids < st["cos"].shape[0]))[:, None]
    ids = ids.clamp(0, st["cos"].shape[0] - 1)
    c, s = (st[n][ids, idx].double()[:, None] for n in ("cos", "sin"))
    a, b = x[..., e1], x[..., e2]
    y, m = x.clone(), x.abs()
    y[..., e1] = torch.where(ok, a * c - b * s, a)
    y[..., e2] = torch.where(ok, b * c + a * s, b)
    m[..., e1] = torch.where(ok, (a * c).abs() + (b * s).abs(), a.abs())
    m[..., e2] = torch.where(ok, (b * c).abs() + (a * s).abs(), b.abs())
    tol = half_step(st["dtype"]) * y.abs() + m * (D + 16) * 2.0 ** -24 * 1.01
    return y, tol + torch.finfo(st["dtype"]).smallest_normal * half_step(st["dtype"]) * 2


def make(new, past, *, H, KV, D, block, dtype, sections, turns=False, pairs=0, offset=0, norm=False, table=None,
         seed=0, packed=False, cache_dtype=None, pad_tokens=0, axes_pos=200, scales="PER_TENSOR"):
    st = make_batch(new, past, H=H, KV=KV, D=D, block=block, dtype=dtype, seed=seed, cache_dtype=cache_dtype,
                    pad_tokens=pad_tokens, scales=scales)
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(new) + pad_tokens
    st.update(sections=sections, turns=turns, pairs=pairs, offset=offset)
    rows = torch.randn(T, (H + 2 * KV) * D, generator=g).to(dtype).cuda()
    q, k, v = rows.split([H * D, KV * D, KV * D], 1)
    st["q"], st["k"], st["v"] = (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())
    half = sum(sections)
    ang = torch.rand(axes_pos, half, generator=g, dtype=torch.float64) * 6.3
    st["cos"], st["sin"] = ang.cos().to(table or dtype).cuda(), ang.sin().to(table or dtype).cuda()
    st["positions"] = torch.randint(0, axes_pos, (len(sections), T), generator=g).cuda()
    st["qn"] = st["kn"] = None
    if norm:
        st["qn"], st["kn"] = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2))
    return st


def call(st, **kw):
    return ep.multi_axis_rotary_append(
        st["q"], st["k"], st["v"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], st["positions"], st["cos"],
        st["sin"], num_heads=st["H"], axis_sections=st["sections"], axes_interleaved=st["turns"],
        rotary_interleaved=st["pairs"], rotary_offset=st["offset"], q_norm_weight=st["qn"], k_norm_weight=st["kn"],
        qk_norm_epsilon=1e-6, k_scale=st["k_scale"], v_scale=st["v_scale"], k_quant_type=st["quant"],
        v_quant_type=st["quant"], **kw)


def places(st):
    """Page and row of every packed token."""
    out = []
    for b, (n, p) in enumerate(zip(st["new"], st["past"])):
        for i in range(n):
            out.append((int(st["bt"][b, (p + i) // st["block"]]), (p + i) % st["block"]))
    pages = torch.tensor([o[0] for o in out], device="cuda"), torch.tensor([o[1] for o in out], device="cuda")
    return pages


def compare(st, **kw):
    T, H, KV, D = sum(st["new"]), st["H"], st["KV"], st["D"]
    want_q, tol_q = turned64(st["q"], H, st, st["qn"], 1e-6)
    want_k, tol_k = turned64(st["k"], KV, st, st["kn"], 1e-6)
    before_k, before_v = st["kc"].clone(), st["vc"].clone()
    v = st["v"].clone().reshape(-1, KV, D)
    q = call(st, **kw)
    check(q.view(-1, H, D)[:T], want_q[:T], tol_q[:T])
    at = places(st)
    check(st["kc"][at], want_k[:T], tol_k[:T])
    assert torch.equal(st["vc"][at], v[:T])
    # nothing else of the pages changes
    before_k[at], before_v[at] = st["kc"][at], st["vc"][at]
    assert torch.equal(before_k.view(torch.uint8), st["kc"].view(torch.uint8))
    assert torch.equal(before_v.view(torch.uint8), st["vc"].view(torch.uint8))
    return q


LAYOUTS = [
    (BF16, 32, 8, 128, 16, (16, 24, 24), {}), (F16, 28, 4, 128, 16, (16, 24, 24), dict(turns=True, norm=True)),
    (F16, 24, 4, 256, 256, (8, 12, 12), dict(turns=True, norm=True)), (BF16, 8, 2, 64, 32, (8, 12, 12), dict(norm=True)),
    (BF16, 6, 3, 96, 16, (16, 16, 16), {}), (F16, 4, 2, 128, 16, (3, 20, 41), dict(pairs=1, turns=True)),
    (BF16, 4, 2, 128, 16, (16, 8, 8), dict(offset=64)), (F16, 4, 2, 128, 16, (5, 4, 3), dict(offset=7, norm=True)),
    (F32, 4, 2, 64, 16, (8, 12, 12), dict(norm=True)), (BF16, 3, 1, 80, 24, (10, 15, 15), dict(norm=True)),
    (F16, 2, 1, 33, 16, (5, 6), {}), (BF16, 4, 1, 512, 16, (32, 32, 32, 32), dict(norm=True)),
    (F16, 2, 2, 640, 16, (320,), dict(norm=True)), (BF16, 8, 2, 128, 16, (16, 24, 24), dict(table=F32, norm=True)),
    (F16, 8, 2, 64, 16, (0, 16, 16), dict(table=F32, pairs=1, norm=True))]


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace("torch.", "") for y in x[:5]))
@pytest.mark.parametrize("packed", [False, True], ids=["dense", "packed"])
@pytest.mark.parametrize("distinct", [False, True], ids=["any_slots", "distinct"])
def test_layouts(layout, packed, distinct):
    dt, H, KV, D, block, sections, more = layout
    for new, past in (([1], [5]), ([1] * 9, [17 * i for i in range(9)]), ([40, 0, 3, 100], [0, 9, 700, 31])):
        st = make(new, past, H=H, KV=KV, D=D, block=block, dtype=dt, sections=sections, packed=packed, seed=len(new), **more)
        compare(st, slots_distinct=distinct)


@pytest.mark.parametrize("dt,D,norm", [(BF16, 128, True), (F16, 64, False), (F16, 96, False), (F32, 64, True)])
def test_in_place_queries(dt, D, norm):
    h = D // 2
    st = make([50, 1], [3, 90], H=6, KV=2, D=D, block=16, dtype=dt, sections=(h - 2 * (h // 3), h // 3, h // 3), norm=norm)
    q = compare(st, q_out=st["q"], slots_distinct=True)
    assert q.data_ptr() == st["q"].data_ptr()


def test_positions_outside_the_table_leave_the_pair():
    st = make([20], [0], H=4, KV=2, D=128, block=16, dtype=BF16, sections=(16, 24, 24))
    st["positions"][0, 3], st["positions"][1, 4], st["positions"][2, 5] = -1, 200, 1 << 40
    compare(st, slots_distinct=True)
    compare(st)


@pytest.mark.parametrize("distinct", [False, True])
def test_wider_position_rows_and_rows_behind_the_last_sequence(distinct):
    st = make([7, 2], [10, 1], H=4, KV=2, D=128, block=16, dtype=BF16, sections=(16, 24, 24), pad_tokens=4)
    wide = torch.zeros(3, 40, dtype=torch.int64, device="cuda")
    wide[:, 5:18] = st["positions"]
    st["positions"] = wide[:, 5:18]
    out = torch.full((13, 512), 7.0, dtype=BF16, device="cuda")
    compare(st, q_out=out, slots_distinct=distinct)
    assert bool((out[9:] == 7.0).all())


@pytest.mark.parametrize("kind,scales", [(torch.float8_e4m3fn, "NONE"), (torch.int8, "PER_TENSOR"), (torch.int8, "PER_CHANNEL"),
                                         (torch.uint8, "PER_TENSOR"), (torch.uint8, "PER_CHANNEL")])
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 80)])
@pytest.mark.parametrize("distinct", [False, True])
def test_byte_coded_pages(kind, scales, dt, D, distinct):
    """A code stands for the finished row's value to half a step: half a scale (integers, inside their
    range), half of 2^-3 of the value or of the smallest step 2^-9 (e4m3)."""
    h = D // 2
    st = make([30, 1, 5], [3, 64, 100], H=4, KV=2, D=D, block=16, dtype=dt, sections=(h - 2 * (h // 3), h // 3, h // 3),
              norm=True, cache_dtype=kind, scales=scales)
    st["k_scale"].mul_(0.3)  # some rows saturate
    want, tol = turned64(st["k"], 2, st, st["kn"], 1e-6)
    plain = {s: st[s + "c"].clone() for s in "kv"}
    call(st, slots_distinct=distinct)
    at = places(st)
    for side, rows, t in (("k", want, tol), ("v", st["v"].double().reshape(-1, 2, D), None)):
        codes, sc = st[side + "c"][at], st[side + "_scale"].double()
        if kind == torch.float8_e4m3fn:
            s = sc[at[0]][:, :, None]
            val, top = codes.double() * s, 448 * s
            step = torch.maximum(rows.abs() * 2.0 ** -4, s * 2.0 ** -10)
        else:
            s = sc if scales == "PER_CHANNEL" else sc.view(1, 1)
            if kind == torch.int8:
                val, lo, hi = codes.double() * s, -128, 127
            else:
                val = torch.stack([(codes & 15).double() - 8, (codes >> 4).double() - 8], -1).flatten(-2)[..., :D] * s
                lo, hi = -8, 7
            step = (s / 2).expand_as(rows)
            rows = rows.clamp(lo * s, hi * s) if scales == "PER_TENSOR" else torch.minimum(torch.maximum(rows, lo * s), hi * s)
            top = torch.full_like(rows, torch.inf)
        rows = torch.minimum(torch.maximum(rows, -top.expand_as(rows)), top.expand_as(rows))
        off = (val - rows).abs() - (step * (1 + 1e-6) + (0 if t is None else t) * (1 + 2.0 ** -4))
        assert float(off.max()) <= 0, float(off.max())
    # values are the plain append's codes, to the bit
    other = {s: plain[s].clone() for s in "kv"}
    ep.reshape_and_cache(st["k"].contiguous(), st["v"].contiguous(), other["k"], other["v"], st["cum"], st["past_t"], st["bt"],
                         k_scale=st["k_scale"], v_scale=st["v_scale"], k_quant_type=st["quant"], v_quant_type=st["quant"])
    assert torch.equal(other["v"].view(torch.uint8), st["vc"].view(torch.uint8))


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 64)])
def test_slot_mapping_and_tokens_that_share_a_slot(dt, D):
    st = make([6, 3], [2, 40], H=4, KV=2, D=D, block=16, dtype=dt, sections=(D // 2,))
    slots = torch.tensor([5, -1, 9, 5, 17, 9, 16, 5, -1], dtype=torch.int32, device="cuda")
    want, tol = turned64(st["k"], 2, st, None, 0)
    before = st["kc"].clone()
    q = call(st, slot_mapping=slots)
    wq, tq = turned64(st["q"], 4, st, None, 0)
    check(q.view(-1, 4, D), wq, tq)
    flat = st["kc"].view(-1, 2, D)
    for slot, t in ((5, 7), (9, 5), (17, 4), (16, 6)):  # the last token of each slot
        check(flat[slot], want[t], tol[t])
        assert torch.equal(st["vc"].view(-1, 2, D)[slot], st["v"].reshape(-1, 2, D)[t])
    keep = [i for i in range(flat.shape[0]) if i not in (5, 9, 16, 17)]
    assert torch.equal(flat[keep].view(torch.uint8), before.view(-1, 2, D)[keep].view(torch.uint8))


def test_keys_and_values_alone():
    st = make([30], [7], H=4, KV=2, D=128, block=16, dtype=BF16, sections=(16, 24, 24), norm=True)
    want, tol = turned64(st["k"], 2, st, st["kn"], 1e-6)
    st["q"] = None
    assert call(st, slots_distinct=True) is None
    check(st["kc"][places(st)], want, tol)


def test_no_norm_and_unturned_rows_are_copied():
    st = make([33], [0], H=4, KV=2, D=128, block=16, dtype=F16, sections=(16, 24, 24))
    st["positions"].fill_(-1)
    q = call(st, slots_distinct=True)
    assert torch.equal(q, st["q"]) and torch.equal(st["kc"][places(st)].reshape(33, -1), st["k"])


def test_captured_and_replayed():
    st = make([1] * 6, [9 * i for i in range(6)], H=8, KV=2, D=128, block=16, dtype=BF16, sections=(16, 24, 24), norm=True)
    out = torch.empty(6, 1024, dtype=BF16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(st, q_out=out, slots_distinct=True)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(st, q_out=out, slots_distinct=True)
    for step in range(3):
        st["positions"].copy_(torch.randint(0, 200, (3, 6)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, pages = out.clone(), st["kc"].clone()
        eager = call(st, slots_distinct=True)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        assert torch.equal(pages.view(torch.uint8), st["kc"].view(torch.uint8))


@pytest.mark.parametrize("dt", [BF16, F16])
def test_picture_prompt_then_samples(dt):
    """Append with three axes, the prompt under its prefix mask, then samples over the shared prompt."""
    H, KV, D, bs, P = 8, 2, 128, 16, 160
    st = make([P], [0], H=H, KV=KV, D=D, block=bs, dtype=dt, sections=(16, 24, 24), turns=True, norm=True, seed=5)
    # the prompt: 100 picture tokens and the question, seen from both sides, the rest causal
    q = call(st, slots_distinct=True)
    st["kd"], st["vd"] = st["kc"].double(), st["vc"].double()
    got = ep.masked_attention(q, st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=H, max_query_len=P,
                              prefix_lens=torch.tensor([120], dtype=torch.int32, device="cuda"))
    want, tol = attention64({**st, "q": q}, prefix=[120])
    check(got, want, tol)
    # six samples of it: the prompt's pages in front, pages of their own behind
    n, steps = 6, 20
    spare = torch.randn(n * 2, bs, KV, D).to(dt).cuda()
    kc, vc = torch.cat([st["kc"], spare]), torch.cat([st["vc"], spare])
    mine = st["kc"].shape[0] + torch.arange(n * 2, device="cuda").view(n, 2)
    bt = torch.cat([st["bt"][:, :P // bs].expand(n, -1), mine.int()], 1).contiguous()
    cum = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    gc, sh = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [P]))
    for step in range(steps):
        new = make([1] * n, [P + step] * n, H=H, KV=KV, D=D, block=bs, dtype=dt, sections=(16, 24, 24), turns=True,
                   norm=True, seed=100 + step)
        new.update(kc=kc, vc=vc, bt=bt)
        q = call(new, slots_distinct=True)
        got = ep.shared_prefix_attention(q, kc, vc, cum, new["past_t"], bt, gc, sh, num_heads=H, max_query_len=1,
                                         max_context_len=P + steps, max_prefix_len=P)
        if step in (0, 1, 15, 16, steps - 1):
            want, tol = attention64({**new, "q": q, "kd": kc.double(), "vd": vc.double()})
            check(got, want, tol)
