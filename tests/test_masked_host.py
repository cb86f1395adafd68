"""Refusals and layouts of the masked, shared-prefix and multi-axis entries, on the host: every call here
is turned down before any device work (the pointers are not memory)."""
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

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "pa_mi355x_ext.h"
MIRRORS = {"pa_axis_rotary": capi.PaAxisRotary, "pa_mask": capi.PaMask,
           "pa_shared_prefix": capi.PaSharedPrefix}
FAKE = 1 << 20
BF16 = capi.PA_DTYPE_BFLOAT16


def header_fields() -> dict[str, list[str]]:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    out = {}
    for m in re.finditer(r"typedef struct (\w+) \{(.*?)\} \1;", text, flags=re.S):
        out[m.group(1)] = [re.sub(r"\[.*$", "", n).split()[-1].lstrip("*")
                           for d in m.group(2).split(";") if d.strip() for n in d.split(",")]
    return out


def test_mirrors_have_the_headers_layout(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc is not available")
    fields = header_fields()
    assert set(fields) == set(MIRRORS)
    body = "".join(f'printf("%s\\"{s}.{f}\\": %zu", n++ ? "," : "{{", offsetof({s}, {f}));'
                   for s, fs in fields.items() for f in fs)
    body += "".join(f'printf(",\\"{s}\\": %zu", sizeof({s}));' for s in fields)
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pa_mi355x_ext.h"\n'
                   f'int main(void) {{ int n = 0; {body} printf("}}\\n"); return 0; }}\n')
    subprocess.run([gcc, "-std=c11", "-Wall", f"-I{HEADER.parent}", str(src), "-o", str(tmp_path / "l")], check=True)
    lay = json.loads(subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout)
    for s, mirror in MIRRORS.items():
        assert [f[0] for f in mirror._fields_] == fields[s]
        assert C.sizeof(mirror) == lay[s]
        for f in fields[s]:
            assert getattr(mirror, f).offset == lay[f"{s}.{f}"], (s, f)


def cache(**kw):
    c = dict(k=FAKE, v=FAKE, ks=None, vs=None, nb=10, bs=16, kv=2, d=128, dt=BF16, kq=0, vq=0)
    c.update(kw)
    return capi.PaCache(*c.values())


def batch(tokens=4, slots=None, flags=0, **kw):
    b = dict(cum=FAKE, past=FAKE, bt=FAKE, slots=slots, batch=2, mb=4, tokens=tokens, mq=4, flags=flags, ctx=0)
    b.update(kw)
    return capi.PaBatch(*b.values())


def attn(heads=8, **kw):
    a = dict(scale=0.0, softcap=0.0, window=-1, causal=1, sink=None, vh=0)
    a.update(kw)
    return capi.PaAttn(heads, *a.values())


def masked(c=None, b=None, a=None, q=FAKE, out=FAKE, ws=FAKE, n=1 << 40, act=BF16):
    return capi.load().pa_masked_attention(C.byref(c or cache()), C.byref(b or batch()), C.byref(a or attn()),
                                           C.byref(capi.PaMask()), act, q, out, ws, n, None)


def error() -> str:
    return capi.load().pa_last_error().decode()


@pytest.mark.parametrize("kw,code,text", [
    (dict(c=cache(v=None)), capi.PA_ERR_UNSUPPORTED, "SEPARATE"),
    (dict(b=batch(slots=FAKE)), capi.PA_ERR_INVALID_ARGUMENT, "slot_mapping"),
    (dict(c=cache(nb=0)), capi.PA_ERR_INVALID_ARGUMENT, "block geometry"),
    (dict(c=cache(d=641)), capi.PA_ERR_UNSUPPORTED, "head_dim"),
    (dict(c=cache(dt=capi.PA_DTYPE_FLOAT16)), capi.PA_ERR_UNSUPPORTED, "cache dtype"),
    (dict(c=cache(dt=capi.PA_DTYPE_FP8_E4M3)), capi.PA_ERR_INVALID_ARGUMENT, "k_scale"),
    (dict(b=batch(cum=None)), capi.PA_ERR_INVALID_ARGUMENT, "metadata"),
    (dict(b=batch(batch=0)), capi.PA_ERR_INVALID_ARGUMENT, "batch"),
    (dict(a=attn(heads=7)), capi.PA_ERR_INVALID_ARGUMENT, "num_heads"),
    (dict(a=attn(scale=float("nan"))), capi.PA_ERR_INVALID_ARGUMENT, "scale"),
    (dict(a=attn(softcap=-1.0)), capi.PA_ERR_INVALID_ARGUMENT, "softcap"),
    (dict(a=attn(softcap=float("inf"))), capi.PA_ERR_INVALID_ARGUMENT, "softcap"),
    (dict(a=attn(vh=64)), capi.PA_ERR_INVALID_ARGUMENT, "head sizes"),
    (dict(q=None), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(out=None), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(b=batch(mb=4000), ws=None, n=0), capi.PA_ERR_INVALID_ARGUMENT, "workspace"),
    (dict(b=batch(mb=4000), n=64), capi.PA_ERR_INVALID_ARGUMENT, "workspace"),
], ids=lambda x: x if isinstance(x, str) else None)
def test_masked_attention_refuses(kw, code, text):
    assert masked(**kw) == code
    assert text in error()


@pytest.mark.parametrize("kw", [dict(q=FAKE + 8), dict(out=FAKE + 2), dict(ws=FAKE + 8)])
def test_rows_and_workspaces_at_odd_addresses_are_refused(kw):
    assert masked(**kw) == capi.PA_ERR_INVALID_ARGUMENT
    assert "16-byte aligned" in error()


def test_null_descriptors_are_refused():
    lib, c, b, a = capi.load(), cache(), batch(), attn()
    for i in range(3):
        args = [C.byref(c), C.byref(b), C.byref(a)]
        args[i] = None
        assert lib.pa_masked_attention(*args, None, BF16, FAKE, FAKE, FAKE, 1 << 40, None) == capi.PA_ERR_INVALID_ARGUMENT
        assert lib.pa_masked_attention_workspace_bytes(*args, None, BF16) == 0


@pytest.mark.parametrize("share", [None, (None, FAKE, 1, 0), (FAKE, None, 1, 0), (FAKE, FAKE, 0, 0), (FAKE, FAKE, 1, -1)])
def test_shared_prefix_refuses(share):
    s = None if share is None else C.byref(capi.PaSharedPrefix(*share))
    rc = capi.load().pa_shared_prefix_attention(C.byref(cache()), C.byref(batch()), C.byref(attn()), s, None, BF16, FAKE, FAKE,
                                                FAKE, 1 << 40, None)
    assert rc == capi.PA_ERR_INVALID_ARGUMENT and "shared prefix" in error()


def test_no_tokens_is_no_work():
    assert masked(b=batch(tokens=0)) == capi.PA_OK
    assert axes(b=batch(tokens=0)) == capi.PA_OK


def rotary(**kw):
    r = dict(positions=FAKE, stride=0, axes=3, sections=(C.c_int32 * 4)(16, 24, 24, 0), turns=0, cos=FAKE, sin=FAKE, table=BF16,
             npos=100, half=64, off=0, pairs=0)
    r.update(kw)
    return capi.PaAxisRotary(*r.values())


def axes(c=None, b=None, r=None, heads=8, act=BF16, q=FAKE, ql=0, k=FAKE * 4, kl=0, v=FAKE * 5, vl=0, qn=None, kn=None, out=FAKE * 6):
    return capi.load().pa_multi_axis_rotary_append(C.byref(c or cache()), C.byref(b or batch()), heads, act, q, ql, k, kl, v, vl,
                                                   C.byref(r or rotary()), qn, kn, 1e-6, out, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(c=cache(v=None)), capi.PA_ERR_UNSUPPORTED, "SEPARATE"),
    (dict(r=rotary(axes=0)), capi.PA_ERR_INVALID_ARGUMENT, "axes"),
    (dict(r=rotary(axes=5)), capi.PA_ERR_INVALID_ARGUMENT, "axes"),
    (dict(r=rotary(half=63)), capi.PA_ERR_INVALID_ARGUMENT, "sections"),
    (dict(r=rotary(axes=2)), capi.PA_ERR_INVALID_ARGUMENT, "sections"),
    (dict(r=rotary(sections=(C.c_int32 * 4)(90, -2, -24, 0))), capi.PA_ERR_INVALID_ARGUMENT, "negative"),
    (dict(r=rotary(off=1)), capi.PA_ERR_INVALID_ARGUMENT, "head_size"),
    (dict(r=rotary(off=-1)), capi.PA_ERR_INVALID_ARGUMENT, "head_size"),
    (dict(r=rotary(npos=0)), capi.PA_ERR_INVALID_ARGUMENT, "head_size"),
    (dict(r=rotary(table=capi.PA_DTYPE_FLOAT16)), capi.PA_ERR_INVALID_ARGUMENT, "tables"),
    (dict(r=rotary(stride=3)), capi.PA_ERR_INVALID_ARGUMENT, "position_stride"),
    (dict(r=rotary(cos=None)), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(r=rotary(positions=None)), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(k=None), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(v=None), capi.PA_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(qn=FAKE), capi.PA_ERR_INVALID_ARGUMENT, "together"),
    (dict(out=None), capi.PA_ERR_INVALID_ARGUMENT, "together"),
    (dict(q=None), capi.PA_ERR_INVALID_ARGUMENT, "together"),
    (dict(heads=0), capi.PA_ERR_INVALID_ARGUMENT, "num_heads"),
    (dict(ql=1023), capi.PA_ERR_INVALID_ARGUMENT, "strides"),
    (dict(kl=255), capi.PA_ERR_INVALID_ARGUMENT, "strides"),
    (dict(vl=-256), capi.PA_ERR_INVALID_ARGUMENT, "strides"),
    (dict(out=FAKE + 2), capi.PA_ERR_INVALID_ARGUMENT, "apart"),
    (dict(out=FAKE, ql=2048), capi.PA_ERR_INVALID_ARGUMENT, "apart"),
    (dict(out=FAKE * 4 + 64), capi.PA_ERR_INVALID_ARGUMENT, "apart"),
    (dict(c=cache(dt=capi.PA_DTYPE_INT8)), capi.PA_ERR_INVALID_ARGUMENT, "quantization"),
], ids=lambda x: x if isinstance(x, str) else None)
def test_multi_axis_append_refuses(kw, code, text):
    assert axes(**kw) == code
    assert text in error()


def test_wrappers_refuse_what_is_not_on_the_device():
    q = torch.zeros(2, 256, dtype=torch.bfloat16)
    kc = torch.zeros(4, 16, 1, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    bt = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ep.masked_attention(q, kc, kc, i, i[:1], bt, num_heads=2)
    with pytest.raises(ValueError, match="device tensor"):
        ep.shared_prefix_attention(q, kc, kc, i, i[:1], bt, i, i[:1], num_heads=2)
    with pytest.raises(ValueError, match="int32"):
        ep.shared_prefix_attention(q, kc, kc, i, i[:1], bt, i.long(), i[:1], num_heads=2)
    with pytest.raises(ValueError, match="one element more"):
        ep.shared_prefix_attention(q, kc, kc, i, i[:1], bt, i, i, num_heads=2)
    with pytest.raises(ValueError, match="device tensor"):
        ep.multi_axis_rotary_append(q, q[:, :128], q[:, :128], kc, kc, i, i[:1], bt, torch.zeros(1, 2, dtype=torch.int64), q, q,
                                    num_heads=2, axis_sections=(64,))
