"""pa_evict_keys against its rule, to the bit: which keys stay, and their rows in place and in other pages."""
from __future__ import annotations

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from upkeep_cases import staying

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn,
         "int8": torch.int8, "int4": torch.uint8}


def setup(lens, *, KV=2, D=64, block=16, kind="bf16", seed=0, extra=0, weights=None):
    """Caches of random bytes (finite), their account, tables; `extra` rows of table for other pages."""
    g = torch.Generator().manual_seed(seed)
    mb = max(1, max(-(-n // block) for n in lens)) + 1
    nb = 2 * mb * len(lens) + 3
    order = torch.randperm(nb, generator=g).to(torch.int32)
    table = order[:mb * len(lens)].view(len(lens), mb).cuda()
    other = order[mb * len(lens):2 * mb * len(lens)].view(len(lens), mb).cuda()
    dt = KINDS[kind]
    width = (D + 1) // 2 if kind == "int4" else D
    if dt in (torch.int8, torch.uint8):
        mk = lambda: torch.randint(0, 127, (nb, block, KV, width), generator=g).to(dt).cuda()  # noqa: E731
    else:
        mk = lambda: torch.randn(nb, block, KV, width, generator=g).to(dt).cuda()  # noqa: E731
    st = dict(lens=lens, KV=KV, block=block, kc=mk(), vc=mk(), table=table, other=other, kw={},
              w=torch.rand(nb, KV, block, generator=g).cuda(),
              lens_t=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if kind == "fp8":
        st["kw"] = dict(k_scale=(torch.rand(nb, KV, generator=g) + 0.5).cuda(),
                        v_scale=(torch.rand(nb, KV, generator=g) + 0.5).cuda())
    if weights is not None:
        for b, n in enumerate(lens):
            for h in range(KV):
                at = places(st, b, range(n))
                st["w"][at[0], h, at[1]] = torch.as_tensor(weights(n, b, h), dtype=torch.float32).cuda()
    return st


def places(st, b, positions, table="table"):
    p = torch.tensor(list(positions), dtype=torch.long, device="cuda")
    return st[table][b].long()[p // st["block"]], p % st["block"]


def recoded(codes, a, b):
    """fp8 rows of scale a written for scale b, as the append rounds."""
    x = codes.float() * a[:, None]
    y = (x / b[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.where((a == b)[:, None], codes.view(torch.uint8), y.view(torch.uint8))


def raw(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x.view(torch.int16) if x.element_size() == 2 else x


def verify(st, budget, sinks=0, recent=0, out=False, **kw):
    before = {s: st[s].clone() for s in ("kc", "vc", "w")}
    kept, left = ep.evict_keys(st["kc"], st["vc"], st["w"], st["lens_t"], st["table"], budget=budget, sinks=sinks,
                               recent=recent, block_table_out=st["other"] if out else None, **st["kw"], **kw)
    want = {s: before[s].clone() for s in before}
    touched = torch.zeros(st["kc"].shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(st["lens"]):
        m = min(n, budget)
        assert int(left[b]) == m
        dst = places(st, b, range(m), "other" if out else "table")
        if out or n > budget:
            touched[places(st, b, range(m if out else n), "other" if out else "table")] = True
        at_all = places(st, b, range(n))
        for h in range(st["KV"]):
            stay = staying(before["w"][at_all[0], h, at_all[1]].tolist(), budget, sinks, recent)
            assert kept[b, h].tolist() == stay + [-1] * (budget - m), (b, h)
            src = places(st, b, stay)
            for s in ("kc", "vc"):
                rows = before[s][src[0], src[1], h]
                if st["kw"]:
                    sc = st["kw"][s[0] + "_scale"]
                    rows = recoded(rows, sc[src[0], h], sc[dst[0], h])
                    want[s].view(torch.uint8)[dst[0], dst[1], h] = rows
                else:
                    want[s][dst[0], dst[1], h] = rows
            want["w"][dst[0], h, dst[1]] = before["w"][src[0], h, src[1]]
            for s in ("kc", "vc"):
                assert torch.equal(raw(st[s])[dst[0], dst[1], h], raw(want[s])[dst[0], dst[1], h]), (s, b, h)
            assert torch.equal(st["w"][dst[0], h, dst[1]].view(torch.int32), want["w"][dst[0], h, dst[1]].view(torch.int32))
    for s in ("kc", "vc"):  # nobody else's rows
        assert torch.equal(raw(st[s])[~touched], raw(before[s])[~touched])
    return kept, left


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "other_pages"])
@pytest.mark.parametrize("kind,D,block", [("bf16", 64, 16), ("f16", 128, 32), ("f32", 40, 7), ("bf16", 256, 256),
                                          ("f16", 3, 16), ("int8", 96, 16), ("int4", 65, 16), ("int4", 128, 24),
                                          ("fp8", 64, 16), ("fp8", 30, 8)])
def test_rows(kind, D, block, out):
    verify(setup([100, 0, 1, 37, 400, 300], D=D, block=block, kind=kind), 37, 3, 10, out)


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "other_pages"])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 32, 32), (200, 0, 0), (513, 4, 100),
                                                 (1999, 0, 0), (2000, 7, 0), (2001, 0, 0), (5000, 4, 9)])
def test_budgets(budget, sinks, recent, out):
    verify(setup([2000, 1500, 513], KV=3, seed=1), budget, sinks, recent, out)


TIES = {"all": lambda n, b, h: [0.0] * n, "few": lambda n, b, h: [float((j * 7 + h) % 3) for j in range(n)],
        "rising": lambda n, b, h: [j / n for j in range(n)], "falling": lambda n, b, h: [-j / n for j in range(n)],
        "zeros": lambda n, b, h: [(-0.0, 0.0)[j % 2] for j in range(n)],
        "near": lambda n, b, h: [1.0 + (j * 37 % n) * 2.0 ** -23 for j in range(n)],
        "odd": lambda n, b, h: [(float("nan"), float("inf"), -float("inf"), 1e-40, -1e-40, 3.0, -3.0)[(j + h) % 7] for j in range(n)]}


@pytest.mark.parametrize("tie", list(TIES))
def test_ties_and_odd_weights(tie):
    for budget in (10, 300, 1000):
        verify(setup([1000, 777], weights=TIES[tie], seed=2), budget, 2, 5)


@pytest.mark.parametrize("n,budget", [(8192 + 600, 4000), (33000, 1000), (40000, 30000)])
def test_long_sequences(n, budget):
    verify(setup([n, 50], KV=1, D=16, seed=3), budget, 4, 64)
    verify(setup([n], KV=1, D=16, seed=3, weights=TIES["few"]), budget, 0, 0, True)


def test_again_and_again():
    """A cache cut down over several rounds, as it grows in between."""
    st = setup([900, 1000], seed=4)
    for n, budget in ((1000, 600), (640, 500), (500, 500), (501, 500), (500, 20)):
        st["lens"] = [min(n, 900), n]
        st["lens_t"] = torch.tensor(st["lens"], dtype=torch.int32, device="cuda")
        verify(st, budget, 4, 16)


def test_bound_on_the_lengths():
    st = setup([500, 200], seed=5)
    verify(st, 100, 4, 16, max_context_len=500)


def test_captured_and_replayed():
    st = setup([3000, 700, 64], KV=4, D=128, seed=6)
    start = {s: st[s].clone() for s in ("kc", "vc", "w")}

    def call():
        return ep.evict_keys(st["kc"], st["vc"], st["w"], st["lens_t"], st["table"], budget=256, sinks=4, recent=32)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, left = call()
    for lens in ([3000, 700, 64], [2000, 257, 0], [256, 300, 1]):
        st["lens_t"].copy_(torch.tensor(lens, dtype=torch.int32))
        seen = []
        for how in (call, None, None):
            for x in start:
                st[x].copy_(start[x])
            k, n = how() if how else (graph.replay(), (kept, left))[1]
            torch.cuda.synchronize()
            seen.append([x.clone() for x in (k, n, st["kc"], st["vc"], st["w"])])
        for other in seen[1:]:
            assert all(torch.equal(a, b) for a, b in zip(seen[0], other))
