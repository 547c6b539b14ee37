"""What gather_rows, norm_rotate and attention refuse, without a GPU: CPU tensors, and through the C ABI every
argument check (they come before any CUDA call)."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import pytorch_cluster_b200 as pc

    x, i = torch.rand(4, 8), torch.tensor([0, 1])
    h = torch.rand(4, 2, 8)
    with pytest.raises(RuntimeError, match="x must be CUDA tensor"):
        pc.gather_rows(x, i)
    with pytest.raises(RuntimeError, match="x must be CUDA tensor"):
        pc.gather_rows(x.requires_grad_(), i)
    with pytest.raises(RuntimeError, match="q must be CUDA tensor"):
        pc.norm_rotate(h, h, torch.rand(4, 1), torch.rand(4, 1), torch.rand(1, 4))
    with pytest.raises(RuntimeError, match="q must be CUDA tensor"):
        pc.attention(h, h, h)
    for op in ("gather_rows", "norm_rotate", "attention"):
        assert hasattr(torch.ops.torch_cluster, op)


class Attention(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + \
        [(n, ctypes.c_int64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")] + \
        [("ptr_q", ctypes.c_void_p), ("ptr_k", ctypes.c_void_p), ("num_segments", ctypes.c_int64),
         ("pos_q", ctypes.c_void_p), ("pos_k", ctypes.c_void_p), ("slope", ctypes.c_void_p),
         ("m", ctypes.c_int64), ("n", ctypes.c_int64)] + \
        [(n, ctypes.c_int) for n in ("heads", "groups", "channels", "dims")] + \
        [("scale", ctypes.c_float), ("cap", ctypes.c_float), ("dtype", ctypes.c_int)]


def attention_args(**changes):
    p = 1 << 20  # never followed: every case below is refused first
    a = dict(q=p, k=p, v=p, q_row=64, q_head=32, k_row=64, k_head=32, v_row=64, v_head=32, num_segments=1, m=4, n=4,
             heads=2, groups=2, channels=32, dims=0, scale=1.0, cap=0.0, dtype=0)
    a.update(changes)
    return Attention(**a)


@pytest.mark.parametrize("changes, message", [
    (dict(dtype=1), b"unsupported dtype"),
    (dict(dtype=7), b"unsupported dtype"),
    (dict(channels=0), b"channels"),
    (dict(channels=129), b"channels"),
    (dict(heads=3), b"heads"),
    (dict(heads=1), b"heads"),
    (dict(groups=0), b"heads"),
    (dict(heads=2048, groups=1), b"heads"),
    (dict(dims=9), b"coordinates"),
    (dict(dims=-1), b"coordinates"),
    (dict(dims=2), b"null pointer"),
    (dict(m=-1), b"rows"),
    (dict(n=1 << 31), b"rows"),
    (dict(num_segments=2), b"Input mismatch"),
    (dict(ptr_q=1 << 20), b"Input mismatch"),
    (dict(ptr_q=1 << 20, ptr_k=1 << 20, num_segments=0), b"Input mismatch"),
    (dict(q=0), b"null pointer"),
    (dict(v=0), b"null pointer"),
    (dict(q=(1 << 20) + 1), b"misaligned"),
    (dict(scale=float("nan")), b"numbers"),
])
def test_attention_argument_checks(changes, message):
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    a = attention_args(**changes)
    for call in (lambda: lib.b200c_attention_forward(ctypes.byref(a), 1 << 20, None, None, None, 0, None),
                 lambda: lib.b200c_attention_backward(ctypes.byref(a), 1 << 20, None, 1 << 20, 1 << 20, 1 << 20, 1 << 20,
                                                      1 << 20, None, 0, None)):
        assert call() == 1 and message in lib.b200c_last_error()
    assert lib.b200c_attention_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.b200c_attention_forward(None, 1 << 20, None, None, None, 0, None) == 1


def test_misaligned_workspaces_are_refused():
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    p, odd, a = 1 << 20, (1 << 20) + 8, attention_args()
    assert lib.b200c_attention_forward(ctypes.byref(a), p, None, None, odd, 1 << 30, None) == 1
    assert b"misaligned workspace" in lib.b200c_last_error()
    assert lib.b200c_attention_backward(ctypes.byref(a), p, None, p, p, p, p, p, odd, 1 << 30, None) == 1
    assert b"misaligned workspace" in lib.b200c_last_error()
    assert lib.b200c_gather_rows(p, p + 4, 4, 4, 8, 1.0, 0, p, None) == 1 and b"misaligned" in lib.b200c_last_error()


class Side(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("rows", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("heads", ctypes.c_int), ("pos", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("y", ctypes.c_void_p), ("dy", ctypes.c_void_p), ("dx", ctypes.c_void_p),
                ("dweight", ctypes.c_void_p)]


@pytest.mark.parametrize("channels, dims, dtype, side, message", [
    (7, 1, 0, {}, b"even"), (258, 1, 0, {}, b"even"), (0, 1, 0, {}, b"even"), (8, 0, 0, {}, b"coordinates"),
    (8, 9, 0, {}, b"coordinates"), (8, 1, 1, {}, b"dtype"), (8, 1, 0, dict(heads=0), b"heads"),
    (8, 1, 0, dict(rows=1 << 31), b"rows"), (8, 1, 0, dict(x=0), b"null"), (8, 1, 0, dict(pos=0), b"null"),
    (8, 1, 0, dict(y=0, dx=0), b"null"),
])
def test_norm_rotate_argument_checks(channels, dims, dtype, side, message):
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    p = 1 << 20
    s = Side(**{**dict(x=p, rows=4, row_stride=8, head_stride=8, heads=1, pos=p, y=p, dy=p, dx=p), **side})
    args = (ctypes.byref(s), ctypes.byref(s), p, dims, channels, 0, 0, 1e-6, dtype)
    assert lib.b200c_norm_rotate(*args, None) == 1 and message in lib.b200c_last_error()
    assert lib.b200c_norm_rotate_backward(*args, None, 0, None) == 1 and message in lib.b200c_last_error()


@pytest.mark.parametrize("rows, edges, channels, dtype, x, message", [
    (-1, 4, 8, 0, 1 << 20, b"mismatch"), (4, 1 << 31, 8, 0, 1 << 20, b"2^31-1"), (4, 4, 0, 0, 1 << 20, b"mismatch"),
    (4, 4, 1 << 20, 0, 1 << 20, b"channels"), (4, 4, 8, 1, 1 << 20, b"dtype"), (4, 4, 8, 0, 0, b"null"),
    (4, 4, 8, 2, (1 << 20) + 1, b"misaligned"),
])
def test_gather_rows_argument_checks(rows, edges, channels, dtype, x, message):
    from pytorch_cluster_b200 import _native

    lib = _native.cabi()
    p = 1 << 20
    assert lib.b200c_gather_rows(x, p, rows, edges, channels, 1.0, dtype, p, None) == 1
    assert message in lib.b200c_last_error()
    assert lib.b200c_gather_rows_backward(x, p, rows, edges, channels, 1.0, dtype, p, None, 0, None) == 1
    assert message in lib.b200c_last_error()


@pytest.mark.gpu
def test_mismatched_cuda_tensors_are_refused():
    import pytorch_cluster_b200 as pc

    d = dict(device="cuda")
    q, k = torch.rand(6, 4, 32, **d), torch.rand(5, 2, 32, **d)
    ok = torch.zeros(6, dtype=torch.long, **d)
    with pytest.raises(RuntimeError, match="float, half and bfloat16"):
        pc.attention(q.double(), k.double(), k.double())
    with pytest.raises(RuntimeError, match="mismatch"):
        pc.attention(q, k.half(), k.half())
    with pytest.raises(RuntimeError, match="mismatch"):
        pc.attention(q, k, k[:4])
    with pytest.raises(RuntimeError, match="mismatch"):
        pc.attention(q, k[..., :16], k[..., :16])
    with pytest.raises(RuntimeError, match="mismatch"):
        pc.attention(q[0], k, k)
    with pytest.raises(RuntimeError, match="multiple"):
        pc.attention(q[:, :3], k, k)
    with pytest.raises(RuntimeError, match="128 channels"):
        pc.attention(*(torch.rand(3, 1, 136, **d) for _ in range(3)))
    with pytest.raises(AssertionError):
        pc.attention(q, k, k, ok)
    with pytest.raises(AssertionError):
        pc.attention(q, k, k, ok, ok)
    with pytest.raises(ValueError, match="positive"):
        pc.attention(q, k, k, cap=0.0)
    with pytest.raises(ValueError, match="finite"):
        pc.attention(q, k, k, cap=float("inf"))
    with pytest.raises(ValueError, match="together"):
        pc.attention(q, k, k, pos_q=torch.rand(6, 3, **d))
    p = dict(pos_q=torch.rand(6, 3, **d), pos_k=torch.rand(5, 3, **d), slope=torch.rand(4, **d))
    for name, bad in (("pos_q", torch.rand(5, 3, **d)), ("pos_k", torch.rand(5, 2, **d)), ("slope", torch.rand(2, **d)),
                      ("slope", torch.rand(4))):
        with pytest.raises(RuntimeError, match="mismatch"):
            pc.attention(q, k, k, **{**p, name: bad})
    for name in p:
        with pytest.raises(RuntimeError, match="receives no gradient"):
            pc.attention(q, k, k, **{**p, name: p[name].clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="coordinates"):
        pc.attention(q, k, k, pos_q=torch.rand(6, 9, **d), pos_k=torch.rand(5, 9, **d), slope=p["slope"])
    x, e = torch.rand(6, 8, **d).requires_grad_(), torch.zeros(4, dtype=torch.long, **d)
    # linear: where the outer gradient is a constant, so is the inner one; where it is not, there is no second one
    assert not torch.autograd.grad(pc.gather_rows(x, e).sum(), x, create_graph=True)[0].requires_grad
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(torch.autograd.grad(pc.gather_rows(x, e).square().sum(), x, create_graph=True)[0].sum(), x)
    out = pc.attention(q.requires_grad_(), k, k)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(torch.autograd.grad(out.square().sum(), q, create_graph=True)[0].sum(), q)

    f = torch.rand(1, 16, **d)
    pos = torch.rand(6, 1, **d)
    for args in ((q, k, pos, pos, f), (q, k, pos, pos[:5], f[:, :8]), (q, k, pos, pos[:5], torch.rand(2, 16, **d)),
                 (q, k.half(), pos, pos[:5], f), (q, k, pos, pos[:5], f.half()), (q.double(), k.double(), pos, pos[:5], f),
                 (q, k, pos, pos[:5], f, torch.rand(31, **d)), (q, k, pos, pos[:5], f.cpu())):
        with pytest.raises(RuntimeError):
            pc.norm_rotate(*args)
    with pytest.raises(RuntimeError, match="receives no gradient"):
        pc.norm_rotate(q, k, pos.clone().requires_grad_(), pos[:5], f)
    x = torch.rand(6, 8, **d)
    for args in ((x.double(), ok), (x, ok.int()), (x, ok.cpu()), (x[0], ok), (x, ok[None])):
        with pytest.raises(RuntimeError):
            pc.gather_rows(*args)
