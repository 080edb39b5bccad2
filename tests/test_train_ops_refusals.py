"""Refusals of the training operators that need no GPU: C entry points with arguments that no kernel may see, Python entry
points with tensors that are not on a GPU, and the descriptor's layout."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tensor(**kw):
    import nsr_hip
    d = dict(params=4096, grad=4096, exp_avg=4096, exp_avg_sq=4096, n=100, lr=0.1, weight_decay=0.0, dtype=0, state_bits=32)
    t = nsr_hip.NsrAdamwTensor()
    for k, v in {**d, **kw}.items():
        setattr(t, k, v)
    return (nsr_hip.NsrAdamwTensor * 1)(t)


@pytest.mark.parametrize("kw,said", [
    (dict(params=None), "NULL pointer"), (dict(grad=None), "NULL gradient"), (dict(exp_avg=None), "NULL pointer"),
    (dict(dtype=3), "dtype 3"), (dict(state_bits=16), "16 bits"), (dict(state_bits=8), "scales"), (dict(n=1 << 35), "2^35"),
    (dict(index0=100), "index0"), (dict(grad=4097), "misaligned"), (dict(params=4098), "misaligned"),
    (dict(exp_avg=4097), "misaligned"), (dict(image=4097), "misaligned"), (dict(lr_dev=4096), "lr_dev"),
    (dict(state_bits=8, scales_m=4098, scales_r=4096), "misaligned")])
def test_adamw_tensors_refuses(kw, said):
    import nsr_hip
    lib = nsr_hip.lib
    assert lib.nsr_adamw_tensors(_tensor(**kw), 1, 0.9, 0.99, 1e-15, 1, None, 1.0, 0, None) < 0
    assert said in lib.nsr_last_error().decode()


def test_adamw_scalars_are_checked():
    import nsr_hip
    lib = nsr_hip.lib
    none = _tensor(n=0)
    assert lib.nsr_adamw_tensors(none, 1, 0.9, 0.99, 1e-15, 1, None, 1.0, 0, None) == 0  # nothing to launch
    assert lib.nsr_adamw_tensors(None, 0, 0.9, 0.99, 1e-15, 1, None, 1.0, 0, None) == 0
    for b1, b2, eps, step in ((1.0, 0.9, 0.0, 1), (0.9, -0.1, 0.0, 1), (0.9, 0.9, -1.0, 1), (0.9, 0.9, 0.0, 0),
                              (float("nan"), 0.9, 0.0, 1)):
        assert lib.nsr_adamw_tensors(none, 1, b1, b2, eps, step, None, 1.0, 0, None) < 0
    assert lib.nsr_adamw_tensors(None, 1, 0.9, 0.9, 0.0, 1, None, 1.0, 0, None) < 0
    assert lib.nsr_adamw_begin(None, None, 0.9, 0.9, None, 0, 1.0, None, None, None) < 0
    assert lib.nsr_adamw_begin(4096, 4096, 0.9, 0.9, 4096, 1, 0.0, None, None, None) < 0
    assert lib.nsr_adamw_begin(4096, 4096, 0.9, 1.5, None, 1, 1.0, None, None, None) < 0
    got = ctypes.c_uint32(7)
    assert lib.nsr_grad_squares(none, 1, None, 10, ctypes.byref(got), None) < 0
    assert lib.nsr_grad_squares(none, 1, 4096, 10, ctypes.byref(got), None) == 0 and got.value == 0
    big = _tensor(n=1 << 30)
    assert lib.nsr_grad_squares(big, 1, 4096, 10, ctypes.byref(got), None) < 0  # too little room, refused before the launch
    assert lib.nsr_grad_squares_capacity(big, 1) >= 1024


@pytest.mark.parametrize("bad", [dict(width=0), dict(dtype=3), dict(affine=1), dict(x=None), dict(y=None), dict(eps=-1.0),
                                 dict(stride=31), dict(x=4097), dict(y=4098), dict(weight=4098), dict(mean=4096),
                                 dict(rows=1 << 40)])
def test_layer_norm_forward_refuses(bad):
    import nsr_hip
    a = dict(x=4096, stride=32, weight=4096, bias=None, y=4096, mean=None, rstd=None, rows=4, width=32, dtype=0, affine=0, eps=1e-5)
    a.update(bad)
    assert nsr_hip.lib.nsr_layer_norm_forward(a["x"], a["stride"], a["weight"], a["bias"], a["y"], a["mean"], a["rstd"], a["rows"],
                                              a["width"], a["dtype"], a["affine"], a["eps"], None) < 0
    assert b"nsr_layer_norm_forward" in nsr_hip.lib.nsr_last_error()


@pytest.mark.parametrize("bad", [dict(width=0), dict(dtype=3), dict(affine=2), dict(x=None), dict(dy=None), dict(ws=None),
                                 dict(stride=31), dict(dy=4097), dict(dx=4098), dict(dw=4097), dict(mean=None), dict(ws=4098)])
def test_layer_norm_backward_refuses(bad):
    import nsr_hip
    a = dict(dy=4096, stride=32, x=4096, weight=4096, mean=4096, rstd=4096, dx=4096, dw=4096, db=4096, ws=4096, rows=4, width=32,
             dtype=0, affine=0)
    a.update(bad)
    assert nsr_hip.lib.nsr_layer_norm_backward(a["dy"], a["stride"], a["x"], 32, a["weight"], a["mean"], a["rstd"], a["dx"], a["dw"],
                                               a["db"], a["ws"], a["rows"], a["width"], a["dtype"], a["affine"], None) < 0
    assert b"nsr_layer_norm_backward" in nsr_hip.lib.nsr_last_error()


def test_python_entry_points_refuse_cpu_tensors():
    import nsr.optim
    from nsr.layers import LayerNorm
    from nsr_hip import NsrError, ops
    x = torch.zeros(2, 8)
    with pytest.raises(NsrError):
        ops.layer_norm(x)
    with pytest.raises(NsrError):
        LayerNorm(8)(x)
    with pytest.raises(ValueError):
        LayerNorm(9)(x)
    with pytest.raises(ValueError):
        LayerNorm(0)
    p = torch.nn.Parameter(x)
    with pytest.raises(NsrError):
        nsr.optim.AdamW([p])
    for kw in (dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=float("inf")), dict(rounding_seed=-1)):
        with pytest.raises(ValueError):
            nsr.optim.AdamW([p], **kw)


def test_descriptor_layout(tmp_path):
    import nsr_hip
    cls = nsr_hip.NsrAdamwTensor
    src = tmp_path / "layout.c"
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "nsr_hip.h"', 'int main(void) {',
             '  printf("%zu\\n", sizeof(NsrAdamwTensor));']
    lines += [f'  printf("%zu\\n", offsetof(NsrAdamwTensor, {f[0]}));' for f in cls._fields_] + ['  return 0;', '}']
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)])
    got = [int(v) for v in subprocess.check_output([str(exe)], text=True).split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]


def test_begin_clipped_refuses():
    import nsr_hip
    call = nsr_hip.lib.nsr_adamw_begin_clipped
    t = _tensor()
    good = (t, 1, 4096, 10000, 4096, 4096, 0.9, 0.99, 1.0, None, None, None)
    for at, bad in ((0, None), (2, None), (4, None), (5, None), (6, 1.0), (7, -0.1), (8, 0.0), (8, float("nan"))):
        args = list(good)
        args[at] = bad
        assert call(*args) < 0, at
    assert call(_tensor(grad=None), *good[1:]) < 0 and call(_tensor(dtype=7), *good[1:]) < 0
    assert call(_tensor(n=1 << 30), 1, 4096, 10, *good[4:]) < 0  # too little room for the sums, refused before a launch
