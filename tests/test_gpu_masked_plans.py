"""Masked attention's shares of work: documents from the queue, whole items and stretches of them, batches of more
sequences than a plan scans at a time, caches that the matrix-core kernel does not take."""
from __future__ import annotations

import random

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import attention64, check, make_batch
from test_gpu_masked_attention import BF16, F16, compare, run, slopes_of, starts_of

pytestmark = pytest.mark.gpu


def many(n, low, high, ones, seed):
    """n sequences of low .. high new tokens, the first `ones` of one token, some empty."""
    rng = random.Random(seed)
    new = [rng.randint(low, high) for _ in range(n)]
    new[:ones] = [1] * ones
    new[ones + 3] = new[-2] = 0
    rng.shuffle(new)
    return new, [rng.choice([0, 5, 63, 200]) for _ in range(n)]


# Rows * heads that give every workgroup several items (512 workgroups, 768 at head 64, 256 at head 256).
QUEUED = [(BF16, 16, 4, 128, 300, 20, 60), (F16, 32, 4, 64, 270, 20, 40), (BF16, 16, 2, 256, 40, 60, 200),
          (F16, 12, 3, 96, 20, 400, 900)]


@pytest.mark.parametrize("dt,H,KV,D,n,low,high", QUEUED)
def test_documents_from_the_queue(dt, H, KV, D, n, low, high):
    new, past = many(n, low, high, n // 4, seed=D)
    st = make_batch(new, past, H=H, KV=KV, D=D, block=16, dtype=dt, seed=D)
    compare(st, starts=starts_of(st, [1, 7, 30, 64, 150], seed=3))


def test_documents_from_the_queue_with_every_mask():
    new, past = many(24, 100, 500, 6, seed=1)
    st = make_batch(new, past, H=32, KV=8, D=128, block=32, dtype=BF16, seed=8)
    sink = torch.randn(32, device="cuda").to(BF16)
    compare(st, starts=starts_of(st, [5, 90, 200], seed=2), slopes=slopes_of(32), softcap=3.0, window=70, sink=sink,
            prefix=[min(t, 40) for t in st["total"]])


def test_documents_from_the_queue_captured_and_replayed():
    """Every replay starts from queues of its own, also beside eager calls."""
    new, past = many(40, 60, 200, 8, seed=5)
    st = make_batch(new, past, H=32, KV=8, D=64, block=16, dtype=F16, seed=9)
    starts = starts_of(st, [3, 50, 130], seed=4)
    want, tol = attention64(st, starts=starts)
    starts_t = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def call(out):
        return ep.masked_attention(st["q"], st["kc"], st["vc"], st["cum"], st["past_t"], st["bt"], num_heads=32,
                                   document_starts=starts_t, max_query_len=max(new), max_context_len=max(st["total"]),
                                   out=out)

    out = torch.empty_like(st["q"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    eager = call(torch.empty_like(out))
    torch.cuda.synchronize()
    check(eager[:want.shape[0]], want, tol)
    for _ in range(4):
        out.fill_(float("nan"))
        graph.replay()
        other = call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(other, eager)


# One item per workgroup and fewer, several turns of whole ones, stretches beside single tokens, one long sequence.
SHARES = [([130], [0]), ([600], [0]), ([1500], [100]), ([900] * 6, [0] * 6), ([64] * 40, [0] * 40),
          ([257, 1, 1, 1, 1], [3000, 4000, 10, 0, 2000]), ([1] * 40 + [700], [900] * 40 + [2])]


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("share", range(len(SHARES)))
def test_shares(share, D, causal):
    new, past = SHARES[share]
    st = make_batch(new, past, H=8, KV=4, D=D, block=64, dtype=BF16, seed=30 + share)
    compare(st, causal=causal, slopes=slopes_of(8) if share % 2 else None)


@pytest.mark.parametrize("dt,D,H,KV", [(BF16, 128, 8, 2), (F16, 64, 4, 4), (BF16, 256, 4, 1)])
def test_distance_biases_on_both_sides(dt, D, H, KV):
    """Without a causal mask, and behind a prefix, rows see keys on both sides of them."""
    st = make_batch([150, 1, 33, 300], [0, 90, 200, 31], H=H, KV=KV, D=D, block=16, dtype=dt, seed=D)
    compare(st, causal=0, slopes=slopes_of(H))
    compare(st, causal=0, slopes=slopes_of(H), softcap=5.0)
    compare(st, prefix=[100, 91, 220, 331], slopes=slopes_of(H))
    compare(st, slopes=[-s for s in slopes_of(H)], softcap=2.0)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_caches_at_odd_addresses(dt):
    """Caches that do not begin at 16 bytes go to the kernel without matrix cores, with the same answer."""
    st = make_batch([40, 1, 0, 7], [3, 200, 5, 90], H=8, KV=2, D=128, block=16, dtype=dt, seed=2)
    for name in ("kc", "vc"):
        c = st[name]
        room = torch.empty(c.numel() + 4, dtype=c.dtype, device="cuda")
        st[name] = room[4:].view(c.shape).copy_(c)
        assert st[name].data_ptr() % 16 == 8
    compare(st, slopes=slopes_of(8), window=100)


def test_rows_at_odd_addresses_are_refused():
    st = make_batch([3, 1], [3, 200], H=8, KV=2, D=128, block=16, dtype=BF16, seed=2)
    q = st["q"]
    room = torch.empty(q.numel() + 4, dtype=BF16, device="cuda")
    st["q"] = room[4:].view(q.shape).copy_(q)
    with pytest.raises(Exception, match="16-byte aligned"):
        run(st)
    st["q"] = q
    with pytest.raises(Exception, match="16-byte aligned"):
        run(st, out=room[4:].view(q.shape))
