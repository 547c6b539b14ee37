"""gather_rows, norm_rotate and attention where values lie far apart or rows belong to nothing: against their definitions
in 64 bits, with the tolerances of test_gpu_network."""
import math

import pytest
import torch
from test_gpu_network import DTYPES, assert_close, attention_plain, gen, ids, rand, rotate_plain

pytestmark = pytest.mark.gpu


def gradients(ts, dout, *args, **kwargs):
    import pytorch_cluster_b200 as pc

    ts = [t.detach().clone().requires_grad_() for t in ts]
    out = pc.attention(*ts, *args, **kwargs)
    return [out.detach(), *torch.autograd.grad(out, ts, dout)]


# ---- rows of no example --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
# rows of two examples and behind them; channels: 128-row tiles, of twice the width, 16-row tiles
@pytest.mark.parametrize("lens, channels", [([150, 90, 60], 64), ([150, 90, 60], 128), ([100, 90, 20], 32),
                                            ([1, 3, 500], 64)])
def test_gradients_of_rows_of_no_example_are_zero(dtype, lens, channels):
    g = gen(51)
    n, b = sum(lens), ids(lens)
    ts = [rand(g, n, 2, channels, dtype=dtype) for _ in range(4)]
    healthy, outside = b == 0, b == 2
    want = attention_plain(*(t[:lens[0]] for t in ts[:3]), lens[:1], lens[:1], dout=ts[3][:lens[0]])
    for which in range(4):
        for value in (math.nan, math.inf):
            bad = [t.clone() for t in ts]
            bad[which][b == 1] = value
            bad[(which + 1) % 4][outside] = value  # and what stands in the rows themselves
            got = gradients(bad[:3], bad[3], b, b, batch_size=2)
            for name, t in zip(("out", "dq", "dk", "dv"), got):
                assert (t[outside] == 0).all(), (name, which, value)
                assert_close(t[healthy], *want[name], (name, which, value))


# ---- fp16 gradients of unlike magnitudes ---------------------------------------------------------------------

@pytest.mark.parametrize("lens, channels", [([3000, 40], 64), ([100] * 24 + [40], 32), ([700, 40], 128)])
# which: v, the gradient of the output; a row of the example itself is part of the others' dk and dv, not of their dq
@pytest.mark.parametrize("which, value, place", [(w, x, p) for w in (2, 3) for x in (math.inf, math.nan, 6e4)
                                                 for p in ("example", "outside")] +
                         [(3, math.inf, "row"), (3, math.nan, "row")])
def test_fp16_gradients_do_not_depend_on_other_examples_magnitudes(lens, channels, which, value, place):
    g = gen(52)
    n, b = sum(lens), ids(lens)
    ts = [rand(g, n, 2, channels, dtype=torch.float16) for _ in range(3)]
    ts.append(rand(g, n, 2, channels, dtype=torch.float16, scale=1e-4))
    first = n - lens[-1]
    want = attention_plain(*(t[:first] for t in ts[:3]), lens[:-1], lens[:-1], dout=ts[3][:first])
    if place == "row":
        ts[3][5] = value
        got = gradients(ts[:3], ts[3], b, b, batch_size=len(lens))
        keep = torch.arange(first, device="cuda") != 5
        assert_close(got[1][:first][keep], want["dq"][0][keep], want["dq"][1][keep], "dq")
        return
    ts[which][first + 7] = value
    got = gradients(ts[:3], ts[3], b, b, batch_size=len(lens) - (place == "outside"))
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert_close(t[:first], *want[name], name)


@pytest.mark.parametrize("rows, groups, channels, gaps", [(2, 16, 32, 1), (3, 8, 16, 4), (40, 4, 24, 1), (300, 2, 64, 2)])
def test_fp16_gradients_of_many_examples_of_their_own_magnitudes(rows, groups, channels, gaps):
    """Output gradients from 1e-4 to 1e4, another size for every example and key head; empty examples between them."""
    g = gen(59)
    examples = 70000 // rows
    n = examples * rows
    b = torch.arange(examples, device="cuda").repeat_interleave(rows) * gaps
    ts = [rand(g, n, h, channels, dtype=torch.float16) for h in (16, groups, groups)]
    size = 10 ** (8 * torch.rand(examples, groups, generator=g, device="cuda") - 4)
    do = torch.randn(n, 16, channels, generator=g, device="cuda")
    do = (do * size.repeat_interleave(rows, 0).repeat_interleave(16 // groups, 1)[..., None]).half().clamp(-6e4, 6e4)
    got = gradients(ts, do, b, b, batch_size=examples * gaps)
    some = torch.randperm(examples, generator=g, device="cuda")[:30].sort().values
    at = (some[:, None] * rows + torch.arange(rows, device="cuda")).flatten()
    want = attention_plain(*(t[at] for t in ts), [rows] * 30, [rows] * 30, dout=do[at])
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert_close(t[at], *want[name], name)


# ---- derivatives that do not exist are refused ---------------------------------------------------------------

def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwAD

    import pytorch_cluster_b200 as pc

    g = gen(55)
    h = rand(g, 10, 2, 16, dtype=torch.float32)
    pos, freq, w = rand(g, 10, 2, dtype=torch.float32), rand(g, 2, 8, dtype=torch.float32), torch.ones(16, device="cuda")
    slope = torch.ones(2, device="cuda")
    edges = torch.tensor([1, 2, 3], device="cuda")
    calls = [(lambda x: pc.gather_rows(x, edges), [h[:, 0]]),
             (lambda q, k, p, f, wq: pc.norm_rotate(q, k, p, p, f, wq), [h, h, pos, freq, w]),
             (lambda q, k, v, p, s: pc.attention(q, k, v, pos_q=p, pos_k=pos, slope=s), [h, h, h, pos, slope])]
    for call, args in calls:
        for i in range(len(args)):
            for wants in (False, True):
                with fwAD.dual_level():
                    mine = list(args)
                    primal = mine[i].clone().requires_grad_(wants)
                    mine[i] = fwAD.make_dual(primal, torch.ones_like(primal))
                    with pytest.raises(RuntimeError, match="forward-mode|receives no gradient"):
                        call(*mine)
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                        call(*mine)
        with fwAD.dual_level():
            call(*args)  # without tangents nothing is refused


# ---- weights far below a row's largest -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("below", [21.86, 26.0])  # powers of two
# tiles; tiles split over the keys; short examples; few queries
@pytest.mark.parametrize("queries, keys, examples, channels, train", [
    (300, 5000, 1, 64, True), (300, 5000, 1, 128, True), (200, 3000, 1, 64, False), (100, 120, 30, 32, True),
    (1, 40000, 2, 64, False), (2, 3000, 4, 40, True), (1, 40000, 2, 7, False)])
def test_attention_adds_up_small_weights(dtype, below, queries, keys, examples, channels, train):
    """One key takes nearly all the weight and has the value zero: the result is what the others add."""
    import pytorch_cluster_b200 as pc

    g = gen(53)
    m, n = queries * examples, keys * examples
    q, k = torch.zeros(m, 1, channels, device="cuda"), torch.zeros(n, 1, channels, device="cuda")
    q[..., 0], k[..., 0] = 4.0, -below * math.log(2) / 4
    v = 1 + torch.rand(n, 1, channels, generator=g, device="cuda")
    top = torch.arange(examples, device="cuda") * keys + keys // 3
    k[top], v[top] = 0.0, 0.0
    ts = [t.to(dtype).requires_grad_(train) for t in (q, k, v)]
    lens_q, lens_k = [queries] * examples, [keys] * examples
    out = pc.attention(*ts, ids(lens_q), ids(lens_k), scale=1.0, batch_size=examples)
    o, tol = attention_plain(*(t.detach() for t in ts), lens_q, lens_k, scale=1.0)["out"]
    if dtype == torch.float16:
        # a weight is held in fp16 times 2^9 or more, of which 2^-25 is half the smallest step; v is below 2
        tol = tol + keys * 2.0 ** -34 * 2
    assert_close(out.detach(), o, tol, "out")


# ---- rows far from unit size ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels", [64, 6])
@pytest.mark.parametrize("size, eps", [(1e16, 1e-6), (1e-14, 1e-30)])
def test_norm_rotate_gradients_of_large_and_small_rows(dtype, channels, size, eps):
    import pytorch_cluster_b200 as pc

    g = gen(54)
    q, k = (rand(g, 100, 2, channels, dtype=dtype, scale=size).requires_grad_() for _ in range(2))
    pos, freq = rand(g, 100, 2, dtype=torch.float32), rand(g, 2, channels // 2, dtype=torch.float32)
    w = (1 + 0.2 * torch.randn(channels, generator=g, device="cuda")).requires_grad_()
    dy = [rand(g, *q.shape, dtype=dtype) for _ in range(2)]
    out = pc.norm_rotate(q, k, pos, pos, freq, w, w, eps=eps)
    grads = torch.autograd.grad(out, (q, k, w), dy)
    want_w, tol_w = 0.0, 0.0
    for i, x in enumerate((q, k)):
        y, ty, dx, tx, dw, tw = rotate_plain(x.detach(), pos, freq, w.detach(), eps, dy[i])
        assert_close(out[i].detach(), y, ty, "y")
        assert_close(grads[i], dx, tx, "dx")
        want_w, tol_w = want_w + dw, tol_w + tw + 2.0 ** -24 * dw.abs()
    assert_close(grads[2], want_w, tol_w + 2.0 ** -24 * want_w.abs(), "dw")


# ---- caps and scales that 32 bits do not hold -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_caps_and_scales_beyond_32_bits_are_refused(dtype):
    import pytorch_cluster_b200 as pc

    h = rand(gen(56), 70, 2, 16, dtype=dtype)
    for extra in (dict(cap=1e39), dict(cap=1e-50), dict(cap=1e-39, scale=1.0), dict(cap=1.2e-38, scale=2.0),
                  dict(scale=math.inf), dict(scale=1e39), dict(scale=math.nan)):
        with pytest.raises((RuntimeError, ValueError), match="cap|scale"):
            pc.attention(h, h, h, **extra)
    for cap in (math.inf, math.nan, 1e-50, 1e39):
        with pytest.raises(RuntimeError, match="cap"):
            torch.ops.torch_cluster.attention(h, h, h, None, None, None, None, None, 1.0, cap)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, channels", [(70, 16), (300, 64), (70, 7), (1, 40), (1, 7)])
def test_the_largest_and_smallest_caps(dtype, queries, channels):
    g = gen(56)
    ts = [rand(g, n, 2, channels, dtype=dtype) for n in (queries, 300, 300)]
    ts[1][::3, :, ::2] = 0  # products that vanish
    ts[1][::9] = 0
    do = rand(g, queries, 2, channels, dtype=dtype)
    for cap in (3e38, 1e35, 1e30, 1e25, 1e-29, 1e-37):
        want = attention_plain(*ts, [queries], [300], cap=cap, scale=0.25, dout=do)
        got = gradients(ts, do, cap=cap, scale=0.25)
        for name, t in zip(("out", "dq", "dk", "dv"), got):
            assert_close(t, *want[name], (cap, name))


# ---- waits that run out ----------------------------------------------------------------------------------------

def test_a_wait_that_ran_out_is_reported_at_the_next_call():
    """The kernels' part, setting the word, takes a hang; here the host sets it."""
    import pytorch_cluster_b200 as pc
    from pytorch_cluster_b200 import _native

    h = rand(gen(60), 300, 2, 64, dtype=torch.bfloat16).requires_grad_()
    graph = torch.cuda.CUDAGraph()
    out = pc.attention(h, h, h)
    word = _native.cabi().b200c_attention_report()
    assert word and word[0] == 0
    word[0] = 1
    with pytest.raises(RuntimeError, match="wait"):
        pc.attention(h, h, h)
    word[0] = 1
    with pytest.raises(RuntimeError, match="wait"):
        torch.autograd.grad(out.sum(), h, retain_graph=True)
    # said once, and nothing else has changed
    torch.autograd.grad(out.sum(), h)
    with torch.no_grad():
        want = pc.attention(h, h, h)
        with torch.cuda.graph(graph):
            again = pc.attention(h, h, h)
    graph.replay()
    assert torch.equal(again, want) and word[0] == 0


# ---- scripted --------------------------------------------------------------------------------------------------

def test_scripted_functions_give_the_same():
    import pytorch_cluster_b200 as pc

    g = gen(57)
    h, b = rand(g, 50, 2, 32, dtype=torch.bfloat16), ids([20, 30])
    pos, slope = rand(g, 50, 3, dtype=torch.float32), torch.tensor([1.0, 0.5], device="cuda")
    freq = rand(g, 3, 16, dtype=torch.float32)
    attention, rotate, gather = (torch.jit.script(f) for f in (pc.attention, pc.norm_rotate, pc.gather_rows))
    assert torch.equal(attention(h, h, h, b, b, pos, pos, slope), pc.attention(h, h, h, b, b, pos, pos, slope))
    assert torch.equal(attention(h, h, h, cap=3.0), pc.attention(h, h, h, cap=3.0))
    for places in ((pos, pos), (pos, pos.double()), (pos[:, 0], pos[:, 0].clone())):
        f = freq if places[0].dim() == 2 else freq[:1]
        assert all(torch.equal(x, y) for x, y in zip(rotate(h, h, *places, f), pc.norm_rotate(h, h, *places, f)))
    edges = torch.tensor([3, 1, 49], device="cuda")
    assert torch.equal(gather(h[:, 0], edges, 2.0), pc.gather_rows(h[:, 0], edges, 2.0))


# ---- segment pointers ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows, segments", [(0, 1), (1, 1), (33, 5), (1000, 4000), (100000, 7), (100000, 3000),
                                            (70001, 200000), (1000003, 65536), (3000, 100000),
                                            (50000, 16384), (50000, 16385)])
def test_segment_pointers_of_few_and_many_examples(rows, segments):
    g = gen(58)
    batch = torch.randint(0, segments, (rows,), generator=g, device="cuda").sort().values
    for shift in (0, -segments // 3, segments // 3):  # ids below zero and at or above the number of examples
        got = torch.ops.torch_cluster.segment_ptr(batch + shift, segments)
        assert torch.equal(got, torch.searchsorted(batch + shift, torch.arange(segments + 1, device="cuda")))


# ---- small calls, split over the columns -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens_q, lens_k", [([300, 500, 400], [300, 500, 400]), ([40, 30, 50], [700, 900, 300]),
                                            ([90, 0, 20], [400, 600, 800])])
@pytest.mark.parametrize("channels, dims", [(64, 0), (128, 3)])
def test_attention_split_over_columns_keeps_nan_in_its_example(dtype, lens_q, lens_k, channels, dims):
    import pytorch_cluster_b200 as pc

    g = gen(61)
    after = 70  # rows of no example
    bq, bk = ids([*lens_q, after]), ids([*lens_k, after])
    m, n = sum(lens_q), sum(lens_k)
    q, k, v = (rand(g, r + after, 2, channels, dtype=dtype) for r in (m, n, n))
    extra = {}
    if dims:
        extra = dict(pos_q=rand(g, m + after, dims, dtype=torch.float32), pos_k=rand(g, n + after, dims, dtype=torch.float32),
                     slope=torch.tensor([1.0, 0.3], device="cuda"))
    rows = {name: t[:m] if name == "pos_q" else t[:n] if name == "pos_k" else t for name, t in extra.items()}
    want, tol = attention_plain(q[:m], k[:n], v[:n], lens_q, lens_k, **rows)["out"]
    for bad_example in (0, 1, 2, 3):
        for value in (math.nan, math.inf):
            v2, k2 = v.clone(), k.clone()
            at = (bk == bad_example).nonzero().flatten()
            v2[at[::50]], k2[at[::70]] = value, value
            out = pc.attention(q, k2, v2, bq, bk, batch_size=3, **extra)
            keep = (bq != bad_example)[:m]
            assert_close(out[:m][keep], want[keep], tol[keep], (bad_example, value))
            assert (out[m:] == 0).all()
