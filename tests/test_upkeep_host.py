"""Layouts, refusals and workspace sizes of the entries for drafted trees, accounts and eviction, on the host: every
call here is turned down before any device work (the pointers are not memory)."""
from __future__ import annotations

import ctypes as C
import json
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import onnxruntime_ep_mlx_amd as ep
from onnxruntime_ep_mlx_amd import _capi as capi
from onnxruntime_ep_mlx_amd import ops
from test_masked_host import BF16, FAKE, attn, batch, cache, error

HEADER = Path(__file__).resolve().parent.parent / "include" / "pa_mi355x_upkeep.h"
MIRRORS = {"pa_drafts": capi.PaDrafts, "pa_eviction": capi.PaEviction}
F32 = capi.PA_DTYPE_FLOAT32


def test_mirrors_have_the_headers_layout(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc is not available")
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    fields = {m.group(1): [n.split()[-1].lstrip("*") for d in m.group(2).split(";") if d.strip() for n in d.split(",")]
              for m in re.finditer(r"typedef struct (\w+) \{(.*?)\} \1;", text, flags=re.S)}
    assert set(fields) == set(MIRRORS)
    body = "".join(f'printf("%s\\"{s}.{f}\\": %zu", n++ ? "," : "{{", offsetof({s}, {f}));'
                   for s, fs in fields.items() for f in fs)
    body += "".join(f'printf(",\\"{s}\\": %zu", sizeof({s}));' for s in fields)
    body += 'printf(",\\"nodes\\": %d", PA_MAX_TREE_NODES);'
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pa_mi355x_upkeep.h"\n'
                   f'int main(void) {{ int n = 0; {body} printf("}}\\n"); return 0; }}\n')
    subprocess.run([gcc, "-std=c11", "-Wall", f"-I{HEADER.parent}", str(src), "-o", str(tmp_path / "l")], check=True)
    lay = json.loads(subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout)
    assert lay["nodes"] == capi.PA_MAX_TREE_NODES
    for s, mirror in MIRRORS.items():
        assert [f[0] for f in mirror._fields_] == fields[s]
        assert C.sizeof(mirror) == lay[s]
        for f in fields[s]:
            assert getattr(mirror, f).offset == lay[f"{s}.{f}"], (s, f)


def tree(c=None, b=None, a=None, parents=FAKE, q=FAKE, out=8 * FAKE, ws=FAKE, n=1 << 40, act=BF16):
    return capi.load().pa_tree_attention(C.byref(c or cache()), C.byref(b or batch()), C.byref(a or attn()), parents,
                                         act, q, out, ws, n, None)


def weigh(c=None, b=None, a=None, w=FAKE, observed=0, q=FAKE, out=8 * FAKE, ws=FAKE, n=1 << 40, act=BF16):
    return capi.load().pa_accumulating_attention(C.byref(c or cache()), C.byref(b or batch()), C.byref(a or attn()), w,
                                                 observed, act, q, out, ws, n, None)


def accept(c=None, b=None, **kw):
    d = dict(parents=FAKE, tokens=FAKE, targets=FAKE, path=FAKE, lens=FAKE, after=None, most=4, w=None)
    d.update(kw)
    return capi.load().pa_accept_drafts(C.byref(c or cache()), C.byref(b or batch()),
                                        C.byref(capi.PaDrafts(*d.values())), None)


def evict(c=None, b=None, **kw):
    d = dict(w=FAKE, budget=16, sinks=2, recent=4, out=None, blocks=0, kept=FAKE, lens=2 * FAKE)
    d.update(kw)
    return capi.load().pa_evict_keys(C.byref(c or cache()), C.byref(b or batch()),
                                     C.byref(capi.PaEviction(*d.values())), None)


INVALID, UNSUPPORTED = capi.PA_ERR_INVALID_ARGUMENT, capi.PA_ERR_UNSUPPORTED
ATTENTION = [("latent", dict(c=cache(v=None)), UNSUPPORTED, "SEPARATE"),
             ("slots", dict(b=batch(slots=FAKE)), INVALID, "slot_mapping"),
             ("window", dict(a=attn(window=0)), INVALID, "local_window_size"),
             ("scale", dict(a=attn(scale=float("nan"))), INVALID, "scale"),
             ("softcap", dict(a=attn(softcap=-1.0)), INVALID, "softcap"),
             ("heads", dict(a=attn(heads=7)), INVALID, "num_heads"),
             ("values", dict(a=attn(vh=64)), INVALID, "value head"),
             ("type", dict(act=capi.PA_DTYPE_FLOAT16), UNSUPPORTED, "dtype"),
             ("workspace", dict(n=0), INVALID, "workspace too small"),
             ("no_workspace", dict(ws=None), INVALID, "workspace too small"),
             ("workspace_place", dict(ws=FAKE + 8), INVALID, "16-byte"),
             ("query_place", dict(q=FAKE + 2), INVALID, "16-byte"),
             ("no_query", dict(q=None), INVALID, "NULL"),
             ("out_on_query", dict(out=FAKE + 64), INVALID, "overlap"),
             ("batch", dict(b=batch(batch=0)), INVALID, "batch")]


@pytest.mark.parametrize("call", [tree, weigh], ids=["tree", "weigh"])
@pytest.mark.parametrize("name,kw,code,word", ATTENTION, ids=[x[0] for x in ATTENTION])
def test_attention_refusals(call, name, kw, code, word):
    assert call(**kw) == code
    assert word in error()


def test_tree_refusals():
    assert tree(parents=None) == INVALID and "parents" in error()
    assert tree(a=attn(causal=0)) == INVALID and "is_causal" in error()
    assert tree(b=batch(tokens=9000, mq=4097)) == UNSUPPORTED and "4096" in error()
    # rows of other types need no alignment of their own
    c = cache(dt=F32)
    assert tree(c=c, q=FAKE + 4, act=F32, n=0) == INVALID and "workspace too small" in error()


def test_account_refusals():
    assert weigh(w=None) == INVALID and "key_weights" in error()
    assert weigh(w=FAKE + 2) == INVALID and "key_weights" in error()
    assert weigh(observed=-1) == INVALID and "observed_rows" in error()
    assert weigh(b=batch(tokens=1 << 30, mq=1)) == UNSUPPORTED and "rows" in error()


def test_no_tokens_are_fine_without_pointers():
    assert tree(b=batch(tokens=0), parents=None, q=None, out=None, ws=None, n=0) == capi.PA_OK
    assert weigh(b=batch(tokens=0), w=None, q=None, out=None, ws=None, n=0) == capi.PA_OK


ROWS = [("latent", dict(c=cache(v=None)), UNSUPPORTED, "SEPARATE"),
        ("scales", dict(c=cache(dt=capi.PA_DTYPE_FP8_E4M3)), INVALID, "scale"),
        ("geometry", dict(c=cache(bs=0)), INVALID, "geometry"),
        ("batch", dict(b=batch(batch=0)), INVALID, "batch"),
        ("many", dict(b=batch(batch=65536)), INVALID, "batch"),
        ("table", dict(b=batch(bt=None)), INVALID, "metadata"),
        ("past", dict(b=batch(past=None)), INVALID, "metadata")]


@pytest.mark.parametrize("call", [accept, evict], ids=["accept", "evict"])
@pytest.mark.parametrize("name,kw,code,word", ROWS, ids=[x[0] for x in ROWS])
def test_row_refusals(call, name, kw, code, word):
    assert call(**kw) == code
    assert word in error()


def test_accept_refusals():
    assert accept(b=batch(cum=None)) == INVALID and "metadata" in error()
    assert accept(b=batch(slots=FAKE)) == INVALID and "slot_mapping" in error()
    assert accept(b=batch(mq=4097)) == UNSUPPORTED and "4096" in error()
    for kw in (dict(path=None), dict(lens=None), dict(most=0)):
        assert accept(**kw) == INVALID and "path" in error()
    for kw in (dict(parents=None), dict(tokens=None), dict(targets=None)):
        assert accept(**kw) == INVALID and "together" in error()
    assert accept(w=FAKE + 2) == INVALID and "key_weights" in error()
    assert accept(parents=None, tokens=None, targets=None, after=FAKE) == INVALID and "next_tokens" in error()


def test_evict_refusals():
    for kw in (dict(w=None), dict(w=FAKE + 1), dict(kept=None), dict(lens=None)):
        assert evict(**kw) == INVALID and "required" in error()
    for kw in (dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(sinks=9, recent=8)):
        assert evict(**kw) == INVALID and "budget" in error()
    assert evict(out=FAKE, blocks=1) == INVALID and "other pages" in error()  # (FAKE: the table itself)
    assert evict(out=3 * FAKE, blocks=0) == INVALID and "min(budget" in error()
    assert evict(out=3 * FAKE, blocks=1, budget=17) == INVALID and "min(budget" in error()
    assert evict(lens=FAKE) == INVALID and "lens_out" in error()
    assert evict(b=batch(batch=60000), budget=1 << 20, out=None) == UNSUPPORTED and "2^31" in error()


def sizes(c, b, a, act, observed=0):
    lib, args = capi.load(), (C.byref(c), C.byref(b), C.byref(a))
    return (lib.pa_tree_attention_workspace_bytes(*args, act),
            lib.pa_accumulating_attention_workspace_bytes(*args, observed, act),
            lib.pa_masked_attention_workspace_bytes(*args, None, act))


def test_workspaces():
    """The masked entry's own, and a tree's bits, an account's scores or sums beside it."""
    a = attn(heads=8)
    c, b = cache(nb=1000), batch(tokens=64, batch=64, mb=256, mq=1, ctx=4000)
    t, w, m = sizes(c, b, a, BF16)
    assert t == m + 256  # one lag to each of 64 nodes
    wide = sizes(c, batch(tokens=66, batch=2, mb=256, mq=65, ctx=4000), a, BF16)
    assert wide[0] == wide[2] + 1024 + 512  # three words and one lag to each of 66
    # other types: 64 x 2 blocks of rows in 8 chunks of 512 keys, their partial rows of 128 elements and (m, l)
    f32, rows = sizes(cache(nb=1000, dt=F32), batch(tokens=64, batch=64, mb=256, mq=1, ctx=4000), a, F32), 64 * 8 * 8
    assert f32[0] == 256 + 256 + rows * 128 * 4 + rows * 2 * 4
    assert f32[1] == 64 * 8 * 4 + 64 * 8 * 4032 * 4 + rows * 128 * 4 + rows * 2 * 4
    assert w == m + 64 * 8 * 4 + 64 * 8 * 4032 * 4  # constants, scores of 4000 keys in tiles of 64
    # a longer bound than a GiB of scores: sums of chunks instead
    far = batch(tokens=64, batch=64, mb=1 << 18, mq=1, ctx=600000)
    assert sizes(cache(nb=1 << 20), far, a, BF16)[1] - sizes(cache(nb=1 << 20), far, a, BF16)[2] < 1 << 29
    # many rows, some of which count: the sums of one chunk
    p = batch(tokens=2000, batch=2, mb=256, mq=1000, ctx=4000)
    t, w, m = sizes(c, p, a, BF16, observed=32)
    assert t == m + 2000 * 32 * 4 + (2000 * 4 + 255) // 256 * 256  # 32 words to each node
    assert w == m + (2000 * 8 * 4 + 255) // 256 * 256 + 2 * 2 * 4032 * 4
    assert sizes(c, batch(tokens=0), a, BF16)[:2] == (0, 0)


@pytest.fixture
def tensors(monkeypatch):
    """Arguments of the wrappers on the host; the library's calls are not made."""
    monkeypatch.setattr(ops, "_need_cuda", lambda name, t: None)
    monkeypatch.setattr(ops, "_on_device", lambda index, call, *args: capi.PA_OK)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pages = lambda: torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16)  # noqa: E731
    return dict(kc=pages(), vc=pages(), cum=i32(0, 3, 4), past=i32(5, 6), bt=torch.zeros(2, 3, dtype=torch.int32),
                q=torch.zeros(4, 4 * 64, dtype=torch.bfloat16), w=torch.zeros(6, 2, 16), parents=i32(-1, 0, 0, -1),
                tokens=torch.zeros(4, dtype=torch.int64), i32=i32)


def test_wrappers_take_what_fits(tensors):
    t = tensors
    assert ep.tree_attention(t["q"], t["kc"], t["vc"], t["cum"], t["past"], t["bt"], t["parents"], num_heads=4).shape == (4, 256)
    assert ep.accumulating_attention(t["q"], t["kc"], t["vc"], t["cum"], t["past"], t["bt"], t["w"], num_heads=4).shape == (4, 256)
    path, lens, after = ep.accept_drafts(t["kc"], t["vc"], t["cum"], t["past"], t["bt"], t["parents"], t["tokens"], t["tokens"])
    assert path.shape == (2, 4) and lens.shape == (2,) and after.dtype == torch.int64
    kept, lens = ep.evict_keys(t["kc"], t["vc"], t["w"], t["past"], t["bt"], budget=5)
    assert kept.shape == (2, 2, 5) and lens.dtype == torch.int32


def test_wrappers_refuse(tensors):
    t, i32 = tensors, tensors["i32"]
    at = (t["kc"], t["vc"], t["cum"], t["past"], t["bt"])

    def refused(word, f, *args, **kw):
        with pytest.raises((ValueError, TypeError), match=word):
            f(*args, **kw)

    refused("parents", ep.tree_attention, t["q"], *at, t["parents"].long(), num_heads=4)
    refused("parents", ep.tree_attention, t["q"], *at, t["parents"][:3], num_heads=4)
    refused("query", ep.tree_attention, t["q"], *at, t["parents"], num_heads=3)
    refused("out", ep.tree_attention, t["q"], *at, t["parents"], num_heads=4, out=t["q"][:3])
    refused("contiguous", ep.tree_attention, t["q"], *at, i32(-1, 0, 0, -1, 0, 0, 0, 0)[::2], num_heads=4)
    refused("key_weights", ep.accumulating_attention, t["q"], *at, t["w"].half(), num_heads=4)
    refused("key_weights", ep.accumulating_attention, t["q"], *at, t["w"].transpose(1, 2), num_heads=4)
    refused("key_weights", ep.evict_keys, t["kc"], t["vc"], t["w"][:5], t["past"], t["bt"], budget=5)
    refused("int32", ep.evict_keys, t["kc"], t["vc"], t["w"], t["past"].long(), t["bt"], budget=5)
    refused("int32", ep.evict_keys, t["kc"], t["vc"], t["w"], t["past"], t["bt"][:1], budget=5)
    refused("block_table_out", ep.evict_keys, t["kc"], t["vc"], t["w"], t["past"], t["bt"], budget=5,
            block_table_out=t["bt"][0])
    refused("SEPARATE", ep.evict_keys, t["kc"], None, t["w"], t["past"], t["bt"], budget=5)
    refused("key_weights", ep.accept_drafts, *at, t["parents"], t["tokens"], t["tokens"], key_weights=t["w"][1:])
    refused("give", ep.accept_drafts, *at)
    refused("give", ep.accept_drafts, *at, t["parents"], t["tokens"], t["tokens"], path=t["bt"], path_lens=t["past"])
    refused("give", ep.accept_drafts, *at, path=t["bt"])
    refused("int64", ep.accept_drafts, *at, t["parents"], t["tokens"].int(), t["tokens"])
    refused("int64", ep.accept_drafts, *at, t["parents"], t["tokens"], t["tokens"][:2])
    refused("int32", ep.accept_drafts, *at, path=t["bt"].long(), path_lens=t["past"])
    refused("cumulative", ep.accept_drafts, t["kc"], t["vc"], t["cum"][:2], t["past"], t["bt"], t["parents"], t["tokens"], t["tokens"])
