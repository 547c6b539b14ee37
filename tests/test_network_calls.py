"""Calls of gather_rows, norm_rotate and attention that are settled before any CUDA call."""
import ctypes
import math

import pytest
import torch
from test_network_refusals import Side, attention_args


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwAD

    import pytorch_cluster_b200  # noqa: F401

    ops = torch.ops.torch_cluster
    h, pos, freq, w, slope = (torch.rand(*s) for s in ((4, 2, 8), (4, 2), (2, 4), (8,), (2,)))
    calls = [(lambda x: ops.gather_rows(x, torch.tensor([0]), 1.0), [h[:, 0]]),
             (lambda q, k, p, pk, f, wq, wk: ops.norm_rotate(q, k, p, pk, f, wq, wk, 1e-6), [h, h, pos, pos, freq, w, w]),
             (lambda q, k, v, p, pk, s: ops.attention(q, k, v, None, None, p, pk, s, 1.0, 0.0),
              [h, h, h, pos, pos, slope])]
    for call, args in calls:
        for i in range(len(args)):
            for wants in (False, True):
                with fwAD.dual_level():
                    mine = list(args)
                    primal = mine[i].clone().requires_grad_(wants)
                    mine[i] = fwAD.make_dual(primal, torch.ones_like(primal))
                    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                        call(*mine)
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            call(*args)


@pytest.mark.parametrize("changes, message", [
    (dict(cap=math.inf), b"finite"), (dict(cap=-math.inf), b"finite"), (dict(cap=math.nan), b"finite"),
    (dict(scale=math.inf), b"finite"), (dict(scale=-math.inf), b"finite"),
    (dict(cap=1e-39), b"cap"), (dict(cap=1e-38, scale=-1.2), b"cap"), (dict(cap=1e-20, scale=1e20), b"cap"),
])
def test_attention_caps_and_scales_that_are_refused(changes, message):
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    a, p = attention_args(**changes), 1 << 20  # never followed
    assert lib.b200c_attention_forward(ctypes.byref(a), p, None, None, None, 0, None) == 1
    assert message in lib.b200c_last_error()
    assert lib.b200c_attention_backward(ctypes.byref(a), p, None, p, p, p, p, p, None, 0, None) == 1
    assert message in lib.b200c_last_error()
    assert lib.b200c_attention_workspace_bytes(ctypes.byref(a)) == 0


def test_attention_of_more_segments_than_can_be_bisected_is_refused():
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    a, p = attention_args(ptr_q=1 << 20, ptr_k=1 << 20, num_segments=(1 << 30) + 1), 1 << 20
    assert lib.b200c_attention_forward(ctypes.byref(a), p, None, None, None, 0, None) == 1
    assert b"2^30 segments" in lib.b200c_last_error()
    assert lib.b200c_attention_backward(ctypes.byref(a), p, None, p, p, p, p, p, None, 0, None) == 1
    assert b"2^30 segments" in lib.b200c_last_error()


def test_the_word_that_waits_report_to():
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    before = lib.b200c_attention_report()
    word = ctypes.c_int32(0)
    lib.b200c_attention_set_report(ctypes.byref(word))
    assert ctypes.addressof(lib.b200c_attention_report().contents) == ctypes.addressof(word)
    lib.b200c_attention_set_report(before)
    assert bool(lib.b200c_attention_report()) == bool(before)


def test_functions_can_be_scripted():
    import pytorch_cluster_b200 as pc

    h = torch.rand(4, 2, 8)
    pos, freq = torch.rand(4, 2), torch.rand(2, 4)
    for f, args in ((pc.gather_rows, (h[:, 0], torch.tensor([0]))), (pc.norm_rotate, (h, h, pos, pos, freq)),
                    (pc.attention, (h, h, h))):
        with pytest.raises(torch.jit.Error, match="must be CUDA tensor"):
            torch.jit.script(f)(*args)


def test_workspaces_of_sizes_that_are_refused_are_empty():
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    far = (1 << 63) - 1
    for rows, edges, channels in ((far, 10, 8), (1 << 31, 10, 8), (-1, 10, 8), (10, -1, 8), (10, far, 8), (10, 1 << 31, 8),
                                  (10, 10, 0), (10, 10, -8), (10, 10, 65537), (10, 0, 8)):
        assert lib.b200c_gather_rows_workspace_bytes(rows, edges, channels) == 0, (rows, edges, channels)
    assert lib.b200c_gather_rows_workspace_bytes(10, 10, 8) > 0
    assert lib.b200c_norm_rotate_workspace_bytes(-2) == 0 and lib.b200c_norm_rotate_workspace_bytes(258) == 0
    assert lib.b200c_norm_rotate_workspace_bytes(256) > 0


@pytest.mark.parametrize("dtype", [0, 2, 3])  # fp32, fp16, bf16
def test_pointers_between_two_elements_are_refused(dtype):
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    p, odd = 1 << 20, (1 << 20) + 1  # never followed

    def refused(status):
        assert status == 1 and b"misaligned" in lib.b200c_last_error()

    for name in ("q", "k", "v", "ptr_q", "ptr_k", "pos_q", "pos_k", "slope"):
        a = attention_args(**{**dict(dtype=dtype, dims=2, ptr_q=p, ptr_k=p, pos_q=p, pos_k=p, slope=p), name: odd})
        refused(lib.b200c_attention_forward(ctypes.byref(a), p, None, None, None, 0, None))
        refused(lib.b200c_attention_backward(ctypes.byref(a), p, None, p, p, p, p, p, None, 0, None))
    a = ctypes.byref(attention_args(dtype=dtype))
    for i in range(3):
        refused(lib.b200c_attention_forward(a, *(odd if i == j else p for j in range(3)), None, 0, None))
    for i in range(7):
        refused(lib.b200c_attention_backward(a, *(odd if i == j else p for j in range(7)), None, 0, None))

    def rotate(direction, side={}, freq=p, **flags):
        s = Side(**{**dict(x=p, rows=4, row_stride=8, head_stride=8, heads=1, pos=p, weight=p, y=p, dy=p, dx=p, dweight=p),
                    **side})
        args = (ctypes.byref(s), ctypes.byref(s), freq, 1, 8, flags.get("pos_f64", 0), flags.get("freq_f64", 0), 1e-6, dtype)
        return lib.b200c_norm_rotate(*args, None) if direction == "forward" else \
            lib.b200c_norm_rotate_backward(*args, None, 0, None)

    for direction, names in (("forward", ("x", "pos", "weight", "y")),
                             ("backward", ("x", "pos", "weight", "dy", "dx", "dweight"))):
        for name in names:
            refused(rotate(direction, {name: odd}))
        refused(rotate(direction, freq=odd))
        refused(rotate(direction, {"pos": p + 4}, pos_f64=1))
        refused(rotate(direction, freq=p + 4, freq_f64=1))
