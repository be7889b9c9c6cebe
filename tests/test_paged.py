"""Paged cache on the CPU: the descriptor's layout, the C entry points' refusals
(they fail before anything reaches a device) and the Python ones'."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import ma_attn
import paged_attention as pa

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_desc_layout_matches_header(tmp_path):
    names = [f[0] for f in pa._Desc._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ma_paged.h"\nint main(void) {\n'
                   + "".join(f'  printf("{n} %zu\\n", offsetof(ma_paged_desc, {n}));\n' for n in names)
                   + '  printf("sizeof %zu\\n", sizeof(ma_paged_desc));\n  return 0;\n}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                       text=True).stdout.splitlines())
    for n in names:
        assert int(got[n]) == getattr(pa._Desc, n).offset, n
    assert int(got["sizeof"]) == ctypes.sizeof(pa._Desc)


def test_declared_functions_are_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "ma_paged.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(ma_paged_\w+)\s*\(", text))
    assert len(names) == 4
    for n in names:
        assert hasattr(ma_attn.LIB, n), n


def _desc(**kw):
    base = dict(batch=2, num_tokens=3, num_heads=4, num_kv_heads=2, head_dim=64, num_pages=8, page_size=16,
                table_width=4, dtype=ma_attn.BF16, left=-1, num_selected=0, local_pages=1)
    base.update(kw)
    return pa._Desc(**base)


A = 4096  # a pointer-like aligned value; nothing dereferences it


def _append(d, **kw):
    p = dict(key=A, value=A, query=A, query_out=A, ck=A, cv=A, sums=None, table=A, start=A, counts=None, freq=A)
    p.update(kw)
    return ma_attn.LIB.ma_paged_append(ctypes.byref(d), *p.values(), None)


def _decode(d, **kw):
    p = dict(query=A, ck=A, cv=A, table=A, lengths=A, pages=None, out=A, lse=None, ws=A, nbytes=1 << 30)
    p.update(kw)
    return ma_attn.LIB.ma_paged_decode(ctypes.byref(d), *p.values(), None)


def _select(d, **kw):
    p = dict(query=A, sums=A, table=A, lengths=A, pages=A)
    p.update(kw)
    return ma_attn.LIB.ma_paged_select(ctypes.byref(d), *p.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=5), "dtype"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"),
    (dict(num_heads=3), "multiple"), (dict(num_kv_heads=0), "multiple"), (dict(batch=-1), "negative"),
    (dict(num_pages=1 << 30, page_size=64), "2\\^31"), (dict(table_width=1 << 30, page_size=64), "2\\^31"),
    (dict(batch=1 << 30), "batch"),
])
def test_every_call_refuses_bad_sizes(kw, msg):
    for call, extra in ((_append, {}), (_decode, {}), (_select, dict(num_selected=4))):
        assert call(_desc(**extra, **kw)) != 0
        assert re.search(msg, ma_attn.last_error()), (call, ma_attn.last_error())


@pytest.mark.parametrize("dkw,kw,msg", [
    (dict(rotary_dim=8), {}, "rotary_dim"), (dict(rotary_dim=80), {}, "rotary_dim"),
    (dict(rotary_dim=32), dict(freq=None), "null"), ({}, dict(key=None), "null"), ({}, dict(start=None), "null"),
    ({}, dict(query_out=None), "null"), ({}, dict(cv=None), "null"), ({}, dict(table=None), "null"),
    ({}, dict(key=A + 2), "aligned"), ({}, dict(ck=A + 8), "aligned"),
    (dict(num_tokens=1 << 30), {}, "num_tokens"), (dict(num_tokens=1 << 29, batch=1 << 20), {}, "batch"),
])
def test_append_refuses(dkw, kw, msg):
    assert _append(_desc(**dkw), **kw) != 0
    assert msg in ma_attn.last_error()


@pytest.mark.parametrize("dkw,kw,msg", [
    (dict(num_selected=4), {}, "go together"), ({}, dict(pages=A), "go together"),
    (dict(num_selected=65), dict(pages=A), "64"), (dict(num_selected=4, left=3), dict(pages=A), "window"),
    (dict(num_global=2), {}, "num_global"), (dict(left=4, num_global=-1), {}, "num_global"),
    (dict(scale=-1.0), {}, "scale"), (dict(scale=float("inf")), {}, "scale"), (dict(scale=float("nan")), {}, "scale"),
    ({}, dict(out=None), "null"), ({}, dict(lengths=None), "null"), (dict(num_pages=0), {}, "no page"),
    ({}, dict(query=A + 4), "aligned"),
    (dict(table_width=4096), dict(nbytes=16), "workspace"), (dict(table_width=4096), dict(ws=None), "workspace"),
])
def test_decode_refuses(dkw, kw, msg):
    assert _decode(_desc(**dkw), **kw) != 0
    assert msg in ma_attn.last_error(), ma_attn.last_error()


@pytest.mark.parametrize("dkw,kw,msg", [
    (dict(num_selected=0), {}, "num_selected"), (dict(num_selected=65), {}, "num_selected"),
    (dict(local_pages=0), {}, "local_pages"), (dict(first_pages=4), {}, "fit"), (dict(first_pages=-1), {}, "first"),
    (dict(table_width=16385), {}, "16384"), ({}, dict(sums=None), "null"), ({}, dict(pages=None), "null"),
    ({}, dict(sums=A + 4), "aligned"),
])
def test_select_refuses(dkw, kw, msg):
    assert _select(_desc(**{"num_selected": 4, **dkw}), **kw) != 0
    assert msg in ma_attn.last_error()


def test_empty_batches_do_nothing():
    assert _append(_desc(batch=0), key=None) == 0 and _append(_desc(num_tokens=0), key=None) == 0
    assert _decode(_desc(batch=0), query=None) == 0
    assert _select(_desc(batch=0, num_selected=2), query=None) == 0


def test_decode_workspace_grows_with_the_split():
    size = lambda **kw: ma_attn.LIB.ma_paged_decode_workspace_size(ctypes.byref(_desc(**kw)))  # noqa: E731
    assert size(table_width=4) == 0  # one pass
    assert size(table_width=4096) > 0
    assert size(table_width=4096, left=63) == 0  # a short window is one pass however long the cache
    assert size(table_width=4096, num_selected=2) == 0


def test_python_refuses_host_tensors_and_bad_objects():
    x = torch.zeros(2, 16, 2, 64)
    with pytest.raises(RuntimeError, match="device tensor"):
        pa.PagedCache.from_tensors(x, x)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        pa.PagedCache.from_tensors(None, x)
    for call in (lambda: pa.paged_append(x, x, x, x, x), lambda: pa.paged_decode(x, x, x, x),
                 lambda: pa.paged_select(x, x, x, x, 4)):
        with pytest.raises(RuntimeError, match="PagedCache"):
            call()


@pytest.mark.parametrize("dim", [0, 8, 24, -16])
def test_rotation_refuses_dims(dim):
    with pytest.raises(RuntimeError, match="multiple of 16"):
        pa.Rotation(dim, device="cpu")


def test_rotation_frequencies():
    r = pa.Rotation(32, base=500.0, device="cpu")
    assert r.inv_freq.dtype == torch.float64 and r.inv_freq.shape == (16,)
    assert abs(float(r.inv_freq[5]) - 500.0 ** (-10 / 32)) < 1e-15
    given = pa.Rotation(16, inv_freq=torch.arange(8.0), device="cpu")
    assert given.inv_freq.tolist() == list(range(8))
    with pytest.raises(RuntimeError, match="frequencies"):
        pa.Rotation(16, inv_freq=torch.arange(7.0), device="cpu")
    with pytest.raises(RuntimeError, match="base"):
        pa.Rotation(16, base=0.0, device="cpu")
