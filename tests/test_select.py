"""Block selection and the attention over selected blocks on the CPU: descriptor
layout and the C entry points' refusals (they fail before anything reaches a
device)."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import ma_attn
import sparse_attention_cuda as ext

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_desc_layout_matches_header(tmp_path):
    names = [f[0] for f in ext._SelectDesc._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ma_select.h"\nint main(void) {\n'
                   + "".join(f'  printf("{n} %zu\\n", offsetof(ma_select_desc, {n}));\n' for n in names)
                   + '  printf("sizeof %zu\\n", sizeof(ma_select_desc));\n  return 0;\n}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                       text=True).stdout.splitlines())
    for n in names:
        assert int(got[n]) == getattr(ext._SelectDesc, n).offset, n
    assert int(got["sizeof"]) == ctypes.sizeof(ext._SelectDesc)


def test_declared_functions_are_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "ma_select.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(ma_select\w+)\s*\(", text))
    assert len(names) == 6
    for n in names:
        assert hasattr(ma_attn.LIB, n), n


def _desc(**kw):
    base = dict(batch=2, seq_len=300, num_heads=4, num_kv_heads=2, head_dim=64, block_size=64, num_selected=4,
                dtype=ma_attn.BF16, causal=1, local_blocks=1)
    base.update(kw)
    return ext._SelectDesc(**base)


A = 4096  # a pointer-like aligned value; nothing dereferences it
NPTR = {"select_blocks": 3, "selected_forward": 6, "selected_backward": 10}


def _run(name, d, ws=A, nbytes=1 << 40, **at):
    ptrs = [A] * NPTR[name]
    for i, v in at.items():
        ptrs[int(i[1:])] = v
    return getattr(ma_attn.LIB, "ma_" + name)(ctypes.byref(d), *ptrs, ws, nbytes, None)


@pytest.mark.parametrize("name", NPTR)
@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=5), "dtype"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(block_size=48), "block_size"), (dict(block_size=128), "block_size"), (dict(block_size=0), "block_size"),
    (dict(num_selected=0), "num_selected"), (dict(num_selected=65), "num_selected"),
    (dict(num_heads=3), "multiple"), (dict(num_kv_heads=0), "multiple"), (dict(seq_len=-1), "negative"),
    (dict(seq_len=16385 * 64), "blocks"), (dict(seq_len=16384 * 16 + 1, block_size=16), "blocks"),
    (dict(batch=1 << 30), "large"), (dict(batch=1 << 20, seq_len=1 << 19), "large"),
])
def test_every_call_refuses_bad_sizes(name, kw, msg):
    assert _run(name, _desc(**kw)) != 0
    assert msg in ma_attn.last_error(), ma_attn.last_error()


@pytest.mark.parametrize("name", NPTR)
def test_every_call_refuses_pointers_and_workspaces(name):
    assert _run(name, _desc(), p0=None) != 0 and "null" in ma_attn.last_error()
    assert _run(name, _desc(), p1=A + 8) != 0 and "aligned" in ma_attn.last_error()
    need = getattr(ma_attn.LIB, f"ma_{name}_workspace_size")(ctypes.byref(_desc()))
    assert need > 0
    assert _run(name, _desc(), nbytes=need - 1) != 0 and "workspace" in ma_attn.last_error()
    assert _run(name, _desc(), ws=None) != 0 and "workspace" in ma_attn.last_error()
    assert _run(name, _desc(), ws=A + 4) != 0 and "workspace" in ma_attn.last_error()
    for kw in (dict(batch=0), dict(seq_len=0)):  # nothing to do
        assert _run(name, _desc(**kw), p0=None) == 0


@pytest.mark.parametrize("kw", [dict(local_blocks=0), dict(first_blocks=-1), dict(first_blocks=4),
                                dict(local_blocks=5), dict(first_blocks=1 << 62, local_blocks=1 << 62)])
def test_select_refuses_forced_blocks_that_do_not_fit(kw):
    assert _run("select_blocks", _desc(**kw)) != 0
    assert "fit" in ma_attn.last_error()


@pytest.mark.parametrize("name", ["selected_forward", "selected_backward"])
@pytest.mark.parametrize("scale", [-1.0, float("inf"), float("nan")])
def test_attention_refuses_scales(name, scale):
    assert _run(name, _desc(scale=scale)) != 0
    assert "scale" in ma_attn.last_error()


def test_workspace_is_bounded_by_the_heads_that_run_together():
    """Past 1 GiB of partial rows the heads run one group after another."""
    size = lambda **kw: ma_attn.LIB.ma_selected_forward_workspace_size(ctypes.byref(_desc(**kw)))  # noqa: E731
    one = size(batch=1, num_heads=1, num_kv_heads=1, seq_len=65536, num_selected=16)
    many = size(batch=1, num_heads=64, num_kv_heads=64, seq_len=65536, num_selected=16)
    assert one < many < 16 * one


def test_python_refuses_host_tensors():
    x = torch.zeros(1, 64, 2, 64)
    for call in (lambda: ext.select_blocks(x, x, 2), lambda: ext.selected_forward(x, x, x, x),
                 lambda: ext.selected_backward(x, x, x, x, x)):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()
