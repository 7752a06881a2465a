"""CPU: attention and rotary refuse what they cannot run, before anything is launched (no GPU needed): status codes of the C ABI,
exceptions of the Python front end, and the argument structs' layout against the header."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from segquant_b200 import _lib as L
from segquant_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "segquant_b200.h")


@pytest.mark.parametrize("name,mirror", [("sq_attention_args", L.AttentionArgs), ("sq_rotary_args", L.RotaryArgs)])
def test_struct_layout_matches_header(tmp_path, name, mirror):
    fields = [f[0] for f in mirror._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){", f'printf("size %zu\\n", sizeof({name}));']
    lines += [f'printf("{f} %zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n") if line)
    assert int(got["size"]) == ctypes.sizeof(mirror)
    for f in fields:
        assert int(got[f]) == getattr(mirror, f).offset, f
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), open(HEADER).read(), re.S).group(1)
    assert len(re.findall(r"\w+(?:\[\w+\])?\s*[,;]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))) == len(fields)


def _attention_args(**kw):
    a = L.AttentionArgs()
    a.q_dev = a.k_dev = a.v_dev = a.out_dev = 4096
    a.dtype, a.batch, a.Tq, a.Tk, a.Hq, a.Hkv, a.D, a.scale = L.SQ_BF16, 2, 300, 400, 4, 2, 64, 0.125
    for pre, t, h in (("q", 300, 4), ("k", 400, 2), ("v", 400, 2), ("out", 300, 4)):
        setattr(a, pre + "_head_stride", 64)
        setattr(a, pre + "_token_stride", 64 * h)
        setattr(a, pre + "_batch_stride", 64 * h * t)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=L.SQ_F32), L.SQ_ERR_UNSUPPORTED), (dict(dtype=17), L.SQ_ERR_UNSUPPORTED), (dict(D=60), L.SQ_ERR_ALIGNMENT),
    (dict(D=136), L.SQ_ERR_UNSUPPORTED), (dict(D=0), L.SQ_ERR_UNSUPPORTED), (dict(Hkv=3), L.SQ_ERR_INVALID_ARG), (dict(Hkv=0), L.SQ_ERR_INVALID_ARG),
    (dict(scale=0.0), L.SQ_ERR_INVALID_ARG), (dict(scale=-1.0), L.SQ_ERR_INVALID_ARG), (dict(scale=float("inf")), L.SQ_ERR_INVALID_ARG),
    (dict(scale=float("nan")), L.SQ_ERR_INVALID_ARG), (dict(Tq=-1), L.SQ_ERR_INVALID_ARG), (dict(batch=-1), L.SQ_ERR_INVALID_ARG),
    (dict(q_offsets_dev=4096), L.SQ_ERR_INVALID_ARG), (dict(kv_offsets_dev=4096), L.SQ_ERR_INVALID_ARG),
    (dict(q_offsets_dev=4096, kv_offsets_dev=4096, kv_lens_dev=4096), L.SQ_ERR_INVALID_ARG),
    (dict(q_dev=None), L.SQ_ERR_INVALID_ARG), (dict(v_dev=None), L.SQ_ERR_INVALID_ARG), (dict(out_dev=None), L.SQ_ERR_INVALID_ARG),
    (dict(k_dev=4104), L.SQ_ERR_ALIGNMENT), (dict(out_dev=4098), L.SQ_ERR_ALIGNMENT), (dict(k_token_stride=132), L.SQ_ERR_ALIGNMENT),
    (dict(q_head_stride=0), L.SQ_ERR_ALIGNMENT), (dict(v_batch_stride=-64), L.SQ_ERR_ALIGNMENT), (dict(Tk=1 << 31), L.SQ_ERR_TOO_LARGE),
    (dict(batch=1 << 20, Tq=1 << 20), L.SQ_ERR_TOO_LARGE),
    (dict(batch=1, Tq=1, Tk=9000), L.SQ_ERR_INVALID_ARG),        # cut into parts: scratch is missing
])
def test_attention_status_codes(native_lib, change, status):
    assert native_lib.sq_attention(ctypes.byref(_attention_args(**change)), None) == status
    assert native_lib.sq_last_error()


def test_attention_scratch_bytes(native_lib):
    size = lambda **kw: native_lib.sq_attention_scratch_bytes(ctypes.byref(_attention_args(**kw)))  # noqa: E731
    assert size(batch=64, Tq=4096, Tk=4096) == 0
    assert size(batch=0) == 0 and size(Tq=0) == 0
    assert size(D=60) == L.SQ_ERR_ALIGNMENT
    one = size(batch=1, Tq=1, Tk=9000)                            # a part is a row of D values and a logarithm in fp32
    assert one > 0 and one % (4 * (64 + 1) * 4) == 0
    assert native_lib.sq_attention(None, None) == L.SQ_ERR_INVALID_ARG
    assert native_lib.sq_attention_scratch_bytes(None) == L.SQ_ERR_INVALID_ARG
    # nothing to do: no pointer is looked at
    for kw in (dict(batch=0), dict(Tq=0), dict(Hq=0)):
        assert native_lib.sq_attention(ctypes.byref(_attention_args(q_dev=None, k_dev=None, v_dev=None, out_dev=None, **kw)), None) == 0


def _rotary_args(**kw):
    a = L.RotaryArgs()
    a.q_dev = a.k_dev = a.q_out_dev = a.k_out_dev = a.positions_dev = 4096
    a.dtype, a.batch, a.tokens, a.heads_q, a.heads_k, a.D, a.num_axes, a.theta, a.eps = L.SQ_F32, 1, 4, 2, 1, 64, 2, 1e4, 1e-6
    a.axes[0], a.axes[1] = 16, 24
    for pre in ("q", "k", "q_out", "k_out"):
        setattr(a, pre + "_head_stride", 64)
        setattr(a, pre + "_token_stride", 128)
    for k, v in kw.items():
        if k == "axes":
            for i, w in enumerate(v):
                a.axes[i] = w
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), L.SQ_ERR_INVALID_ARG), (dict(pairing=2), L.SQ_ERR_INVALID_ARG), (dict(D=0), L.SQ_ERR_UNSUPPORTED), (dict(D=258), L.SQ_ERR_UNSUPPORTED),
    (dict(num_axes=0), L.SQ_ERR_INVALID_ARG), (dict(num_axes=9), L.SQ_ERR_INVALID_ARG), (dict(axes=(16, 50)), L.SQ_ERR_INVALID_ARG),
    (dict(axes=(15, 24)), L.SQ_ERR_INVALID_ARG), (dict(axes=(0, 24)), L.SQ_ERR_INVALID_ARG), (dict(theta=0.0), L.SQ_ERR_INVALID_ARG),
    (dict(theta=float("nan")), L.SQ_ERR_INVALID_ARG), (dict(tokens=-1), L.SQ_ERR_INVALID_ARG), (dict(positions_dev=None), L.SQ_ERR_INVALID_ARG),
    (dict(q_dev=None), L.SQ_ERR_INVALID_ARG), (dict(k_out_dev=None), L.SQ_ERR_INVALID_ARG), (dict(norm_q_dev=4096), L.SQ_ERR_INVALID_ARG),
    (dict(q_dev=4098), L.SQ_ERR_ALIGNMENT), (dict(batch=1 << 30, tokens=1 << 30), L.SQ_ERR_TOO_LARGE),
])
def test_rotary_status_codes(native_lib, change, status):
    assert native_lib.sq_rotary(ctypes.byref(_rotary_args(**change)), None) == status
    assert native_lib.sq_last_error()


def test_rotary_nothing_to_do(native_lib):
    assert native_lib.sq_rotary(None, None) == L.SQ_ERR_INVALID_ARG
    for kw in (dict(tokens=0), dict(batch=0), dict(heads_q=0, heads_k=0)):
        assert native_lib.sq_rotary(ctypes.byref(_rotary_args(q_dev=None, k_dev=None, positions_dev=None, **kw)), None) == 0


def test_no_cpu_path():
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.attention(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.rotary(x, x, torch.zeros(4, 1, dtype=torch.int32), (64,))
