"""A cache kept at work over a while, as a server does: prompts whose last rows say what stays, eviction, steps that go
on weighing, drafted trees checked and accepted, eviction again -- every attention and every account against lists of
the rows that each (sequence, kv-head) should hold, in 64 bits, and the pages against them to the bit."""
from __future__ import annotations

import random

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from masked_cases import check, half_step
from upkeep_cases import PAIR, accepted, lines, packed, staying, tree

pytestmark = pytest.mark.gpu

BS, WORDS = 16, 3


class Cache:
    """The pages with their account, and beside them the rows of every head as they should be."""

    def __init__(self, B, H, KV, D, dt, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.B, self.H, self.KV, self.D, self.dt = B, H, KV, D, dt
        nb, mb = B * 20 + 3, 20
        self.kc, self.vc = (torch.full((nb, BS, KV, D), float("nan"), dtype=dt, device="cuda") for _ in range(2))
        self.w = torch.full((nb, KV, BS), float("nan"), device="cuda")
        self.bt = torch.randperm(nb, generator=self.g)[:B * mb].view(B, mb).to(torch.int32).cuda()
        self.held = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.text = [0] * B  # tokens of the text so far
        self.rows = [[dict(k=torch.zeros(0, D, dtype=torch.float64, device="cuda"),
                           v=torch.zeros(0, D, dtype=torch.float64, device="cuda"),
                           w=torch.zeros(0, dtype=torch.float64, device="cuda"),
                           tol=torch.zeros(0, dtype=torch.float64, device="cuda")) for _ in range(KV)] for _ in range(B)]
        f = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
        self.cos, self.sin = f.cos().to(dt).cuda(), f.sin().to(dt).cuda()

    def place(self, b, j):
        return self.bt[b].long()[j // BS], j % BS

    def append(self, new, places):
        """Rows of new tokens at `places` of their texts into the slots behind what is held; the turned queries."""
        T, kv = sum(new), self.KV * self.D
        rnd = lambda n: torch.randn(T, n, generator=self.g).to(self.dt).cuda()  # noqa: E731
        cum = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        q = ep.multi_axis_rotary_append(rnd(self.H * self.D), rnd(kv), rnd(kv), self.kc, self.vc, cum, self.held, self.bt,
                                        torch.tensor([places], device="cuda"), self.cos, self.sin, num_heads=self.H,
                                        axis_sections=(self.D // 2,), slots_distinct=True)
        return q, cum

    def now(self, b, n):
        """Rows of every head with n new ones, as the pages hold them."""
        held = int(self.held[b])
        p = torch.arange(held, held + n, device="cuda")
        page, off = self.place(b, p)
        return [{s: torch.cat([self.rows[b][h][s], c[page, off, h].double()]) for s, c in (("k", self.kc), ("v", self.vc))}
                for h in range(self.KV)]

    def attend(self, q, new, seen, observed=None):
        """Definition and bound of the outputs; with observed the accounts grow, too."""
        out, t0, u, s = [], 0, half_step(self.dt), PAIR[self.dt]
        for b, n in enumerate(new):
            rows, g = self.now(b, n), self.H // self.KV
            qs = q[t0:t0 + n].double().view(n, self.H, self.D)
            o, tol = torch.zeros(2, n, self.H, self.D, dtype=torch.float64, device="cuda")
            vis = seen[b].cuda()
            for h in range(self.KV):
                r, keys = rows[h], rows[h]["k"].shape[0]
                add, addtol = torch.zeros(2, keys, dtype=torch.float64, device="cuda")
                for j in range(h * g, (h + 1) * g):
                    x = (qs[:, j] @ r["k"].T * self.D ** -0.5).masked_fill(~vis, -torch.inf)
                    M = (qs[:, j].abs() @ r["k"].abs().T * self.D ** -0.5).amax(1, keepdim=True)
                    p = torch.softmax(x, 1)
                    d = (self.D + 24) * 2.0 ** -24 * M
                    o[:, j], A = p @ r["v"], p @ r["v"].abs()
                    tol[:, j] = u * o[:, j].abs() + A * (2 * s + 4 * d + (keys + 64) * 2.0 ** -23) * 1.01 + 1e-12
                    counts = slice(0 if not observed else max(0, n - observed), n)
                    add += p[counts].sum(0)
                    # (64: the constants of the softmax in log2 units stay below it here)
                    addtol += (p * (4 * d + (keys + 128) * 2.0 ** -23))[counts].sum(0) * 1.01
                if observed is not None:
                    mine = self.rows[b][h]
                    zero = torch.zeros(n, dtype=torch.float64, device="cuda")
                    mine["w"] = torch.cat([mine["w"], zero]) + add
                    mine["tol"] = torch.cat([mine["tol"], zero]) + addtol + 2.0 ** -23 * (mine["w"] + (n * g + 8) * add)
            out.append((o.view(n, -1), tol.view(n, -1)))
            t0 += n
        return torch.cat([o for o, _ in out]), torch.cat([t for _, t in out])

    def keep_new(self, new, which=None):
        """New rows (those of `which`) become held ones."""
        for b, n in enumerate(new):
            rows = self.now(b, n)
            held = int(self.held[b])
            for h in range(self.KV):
                pick = list(range(held)) + [held + r for r in (range(n) if which is None else which[b])]
                for s in ("k", "v"):
                    self.rows[b][h][s] = rows[h][s][pick]

    def verify(self):
        for b in range(self.B):
            n = int(self.held[b])
            page, off = self.place(b, torch.arange(n, device="cuda"))
            for h in range(self.KV):
                r = self.rows[b][h]
                assert torch.equal(self.kc[page, off, h].double(), r["k"]) and torch.equal(self.vc[page, off, h].double(), r["v"])
                assert r["w"].shape[0] == n
                check(self.w[page, h, off], r["w"], r["tol"] + 1e-12)


def causal(n, held):
    return torch.arange(held + n) <= held + torch.arange(n)[:, None]


@pytest.mark.parametrize("B,H,KV,D,dt", [(3, 8, 2, 64, torch.bfloat16), (2, 7, 1, 128, torch.float16),
                                         (2, 4, 2, 80, torch.bfloat16), (2, 4, 4, 64, torch.float32)])
def test_a_cache_at_work(B, H, KV, D, dt):
    c, rng = Cache(B, H, KV, D, dt, seed=B), random.Random(H)
    kw = dict(num_heads=H)

    def step(new, observed):
        places = [t + i for t, n in zip(c.text, new) for i in range(n)]
        q, cum = c.append(new, places)
        got = ep.accumulating_attention(q, c.kc, c.vc, cum, c.held, c.bt, c.w, observed_rows=observed,
                                        max_query_len=max(new), **kw)
        want, tol = c.attend(q, new, [causal(n, int(c.held[b])) for b, n in enumerate(new)], observed)
        check(got, want, tol)
        c.keep_new(new)
        c.held += torch.tensor(new, dtype=torch.int32, device="cuda")
        c.text = [t + n for t, n in zip(c.text, new)]
        c.verify()

    def evict(budget, sinks, recent):
        # (who stays goes by the accounts as the pages hold them)
        for b in range(B):
            n = int(c.held[b])
            page, off = c.place(b, torch.arange(n, device="cuda"))
            for h in range(KV):
                stay = staying(c.w[page, h, off].tolist(), budget, sinks, recent)
                for s in ("k", "v", "w", "tol"):
                    c.rows[b][h][s] = c.rows[b][h][s][stay]
        _, c.held = ep.evict_keys(c.kc, c.vc, c.w, c.held, c.bt, budget=budget, sinks=sinks, recent=recent)
        c.verify()

    def draft(nodes):
        parents = [tree(rng, n, 0.6) for n in nodes]
        depth = [lines(p)[1].tolist() for p in parents]
        q, cum = c.append(nodes, [t + d for t, ds in zip(c.text, depth) for d in ds])
        got = ep.tree_attention(q, c.kc, c.vc, cum, c.held, c.bt, packed(parents), max_query_len=max(nodes), **kw)
        seen = [torch.cat([torch.ones(n, int(c.held[b]), dtype=torch.bool), lines(parents[b])[0]], 1)
                for b, n in enumerate(nodes)]
        want, tol = c.attend(q, nodes, seen)
        check(got, want, tol)
        words = lambda: [[rng.randrange(WORDS) for _ in p] for p in parents]  # noqa: E731
        tokens, targets = words(), words()
        paths = [accepted(*x) for x in zip(parents, tokens, targets)]
        c.keep_new(nodes, paths)
        i64 = lambda x: torch.tensor(sum(x, []), dtype=torch.int64, device="cuda")  # noqa: E731
        path, lens, _ = ep.accept_drafts(c.kc, c.vc, cum, c.held, c.bt, packed(parents), i64(tokens), i64(targets),
                                         max_query_len=max(nodes), key_weights=c.w)
        assert [path[b, :int(lens[b])].tolist() for b in range(B)] == paths
        # what was accepted begins weighing nothing
        for b in range(B):
            for h in range(KV):
                for s in ("w", "tol"):
                    zero = torch.zeros(int(lens[b]), dtype=torch.float64, device="cuda")
                    c.rows[b][h][s] = torch.cat([c.rows[b][h][s], zero])
        c.held += lens
        c.text = [t + len(p) for t, p in zip(c.text, paths)]
        c.verify()

    step([90, 37, 60][:B], 16)
    evict(48, 2, 16)
    for _ in range(3):
        step([1] * B, 0)
    draft([26, 9, 40][:B])
    step([1] * B, 0)
    evict(40, 2, 8)
    draft([5, 33, 1][:B])
    step([3] * B, 0)
    evict(30, 0, 0)
    step([1] * B, 0)
