"""gather_rows, norm_rotate and attention against their definitions in 64 bits.

Tolerances are sums of what each rounding can add, element by element: ``u`` is half a step of the type
(``finfo.eps / 2``), ``U`` that of fp32.  They hold for operands of attention's second products rounded to the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def grid(dtype):  # half the distance of the smallest numbers: rounding there is absolute
    return {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134,
            torch.float64: 0.0}[dtype]


def assert_close(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = int((off / tol.clamp(min=1e-300)).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance; worst at {i}: got "
                             f"{got.flatten()[i].item()}, want {want.flatten()[i].item()}, tol {tol.flatten()[i].item()}")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ---- attention -----------------------------------------------------------------------------------------------

def ids(lens):
    return torch.arange(len(lens), device="cuda").repeat_interleave(torch.tensor(lens, device="cuda"))


def attention_plain(q, k, v, lens_q, lens_k, pos_q=None, pos_k=None, slope=None, scale=None, cap=None, dout=None):
    """Outputs, gradients and tolerances (all in 64 bits) of one call."""
    dt, u = q.dtype, half_step(q.dtype)
    q, k, v = q.double(), k.double(), v.double()
    m, h, c = q.shape
    n, g, _ = k.shape
    scale = c ** -0.5 if scale is None else scale
    zero = torch.zeros_like
    o, to = zero(q), zero(q)
    dq, dk, dv, tq, tk, tv = zero(q), zero(k), zero(v), zero(q), zero(k), zero(v)
    i = j = 0
    for mq, nk in zip(lens_q, lens_k):
        if mq and nk:
            qs = q[i:i + mq].transpose(0, 1)
            ks, vs = (t[j:j + nk].transpose(0, 1).repeat_interleave(h // g, 0) for t in (k, v))
            t = scale * qs @ ks.transpose(1, 2)
            # rounding of the scores: the sum over the channels, scale, cap and bias, the change to base 2
            dz = (c + 8) * U * abs(scale) * (qs.abs() @ ks.abs().transpose(1, 2))
            bend = torch.ones_like(t)
            if cap:
                w = torch.tanh(t / cap)
                t, bend = cap * w, 1 - w * w
                dz = dz + 8 * U * cap
            if slope is not None:
                far = (pos_q[i:i + mq].double()[:, None] - pos_k[j:j + nk].double()[None]).square().sum(-1).sqrt()
                b = slope.double()[:, None, None] * far
                t = t - b
                dz = dz + 16 * U * b.abs()
            dz = dz + 8 * U * t.abs()
            p = torch.softmax(t, -1)
            out = p @ vs
            # p: its score's error and the largest score's, the exponential, the sum of nk terms
            rel = 2 * dz.amax(-1, keepdim=True) + (nk + 32) * U
            pv = p @ vs.abs()
            o[i:i + mq] = out.transpose(0, 1)
            to[i:i + mq] = (u * out.abs() + (u + rel) * pv).transpose(0, 1)
            if dout is not None:
                do = dout[i:i + mq].double().transpose(0, 1)
                dp = do @ vs.transpose(1, 2)
                d = (do * out).sum(-1, keepdim=True)
                ds = scale * p * (dp - d) * bend
                # errors of dp and D (the result enters rounded), then of their product with p and of ds itself
                big = do.abs() @ vs.abs().transpose(1, 2) + (do.abs() * pv).sum(-1, keepdim=True)
                e = abs(scale) * p * (big * ((c + 16) * U + rel) + u * (dp - d).abs() +
                                 (do.abs() * (u * out.abs() + (u + rel) * pv)).sum(-1, keepdim=True) +
                                 (16 * U + 2 * dz) * big)
                sum_q = 4 * (mq * h // g + 32) * U  # the sums over queries and heads, and over keys
                sum_k = 4 * (nk + 32) * U
                fold = lambda x: x.reshape(g, h // g, nk, c).sum(1).transpose(0, 1)  # noqa: E731
                dq[i:i + mq] = (ds @ ks).transpose(0, 1)
                tq[i:i + mq] = (e @ ks.abs() + sum_k * (ds.abs() @ ks.abs())).transpose(0, 1)
                dk[j:j + nk] = fold(ds.transpose(1, 2) @ qs)
                tk[j:j + nk] = fold((e + sum_q * ds.abs()).transpose(1, 2) @ qs.abs())
                dv[j:j + nk] = fold(p.transpose(1, 2) @ do)
                tv[j:j + nk] = fold((p * (u + rel + sum_q)).transpose(1, 2) @ do.abs())
        i, j = i + mq, j + nk
    tiny = grid(dt)
    return dict(out=(o, to + tiny), dq=(dq, tq + u * dq.abs() + tiny), dk=(dk, tk + u * dk.abs() + tiny),
                dv=(dv, tv + u * dv.abs() + tiny))


def check_attention(dtype, lens_q, lens_k, heads, groups, channels, dims=0, cap=None, seed=0, train=True, qscale=1.5,
                    dscale=1.0, slope_scale=0.7, scale=None):
    import pytorch_cluster_b200 as pc

    g = gen(seed)
    m, n = sum(lens_q), sum(lens_k)
    q = rand(g, m, heads, channels, dtype=dtype, scale=qscale).requires_grad_(train)
    k = rand(g, n, groups, channels, dtype=dtype).requires_grad_(train)
    v = rand(g, n, groups, channels, dtype=dtype).requires_grad_(train)
    extra = {}
    if dims:
        extra = dict(pos_q=rand(g, m, dims, dtype=torch.float32), pos_k=rand(g, n, dims, dtype=torch.float32),
                     slope=slope_scale * (1 + torch.rand(heads, generator=g, device="cuda")))
        if lens_q == lens_k:
            extra["pos_k"] = extra["pos_q"]
    dout = rand(g, m, heads, channels, dtype=dtype, scale=dscale) if train else None
    out = pc.attention(q, k, v, ids(lens_q), ids(lens_k), cap=cap, scale=scale, batch_size=len(lens_q), **extra)
    assert out.dtype == dtype and out.shape == q.shape
    want = attention_plain(q.detach(), k.detach(), v.detach(), lens_q, lens_k, cap=cap, scale=scale, dout=dout, **extra)
    assert_close(out.detach(), *want["out"], "out")
    if train:
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)):
            assert got.dtype == dtype
            assert_close(got, *want[name], name)


SHAPES = [
    # queries, keys per example; heads, key heads, channels; coordinates; cap
    ([1], [1], 1, 1, 8, 0, None),
    ([1], [1], 2, 1, 64, 3, 10.0),
    ([5], [7], 2, 2, 16, 1, None),
    ([128], [64], 1, 1, 64, 0, None),
    ([129], [65], 2, 1, 64, 2, None),
    ([300], [300], 2, 2, 128, 3, None),
    ([257], [511], 4, 2, 32, 0, 5.0),
    ([64, 1, 200], [64, 1, 200], 4, 4, 32, 3, None),
    ([30, 0, 17, 60, 5], [12, 40, 0, 60, 1], 3, 1, 24, 3, None),
    ([0, 0, 3], [5, 0, 9], 2, 2, 40, 4, 20.0),
    ([7] * 40, [9] * 40, 2, 1, 72, 8, None),
    ([31, 33, 64, 63, 65, 1, 1, 2], [31, 33, 64, 63, 65, 1, 1, 2], 2, 2, 96, 5, 3.0),
    ([100, 28], [640, 1], 6, 2, 128, 0, None),
    ([50], [50], 2, 2, 5, 2, None),      # channels that no 16-byte access fits
    ([40, 90], [90, 40], 1, 1, 1, 0, None),
    ([700, 500], [700, 500], 2, 2, 64, 3, None),
    ([33, 1, 47, 16, 15, 0, 70], [33, 1, 47, 16, 15, 0, 70], 5, 5, 64, 3, 8.0),
    ([12] * 30, [12] * 30, 8, 2, 16, 1, None),
    ([2] * 100, [150] + [1] * 99, 4, 1, 48, 0, None),
    ([40] * 7, [3] * 7, 6, 6, 32, 8, None),
    ([30, 0, 17, 60, 5], [12, 40, 0, 60, 1], 3, 1, 80, 3, None),  # short examples with more channels
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_and_gradients(shape, dtype):
    lens_q, lens_k, heads, groups, channels, dims, cap = SHAPES[shape]
    check_attention(dtype, lens_q, lens_k, heads, groups, channels, dims, cap, seed=shape)


FEW = [
    ([1], [1000], 1, 1, 64, 0, None),
    ([1], [20011], 8, 2, 64, 3, None),
    ([1, 1, 1], [300, 0, 5000], 4, 4, 32, 1, 30.0),
    ([2, 0, 3], [900, 100, 2000], 4, 1, 128, 3, None),
    ([1] * 8, [333] * 8, 2, 2, 24, 0, None),
    ([3], [2048], 4, 4, 40, 2, None),
    ([1], [777], 3, 1, 7, 8, 9.0),
    ([1, 7], [4000, 129], 16, 16, 128, 0, None),
    ([16], [1000], 1, 1, 64, 0, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(FEW)))
def test_attention_of_few_queries(shape, dtype):
    lens_q, lens_k, heads, groups, channels, dims, cap = FEW[shape]
    check_attention(dtype, lens_q, lens_k, heads, groups, channels, dims, cap, seed=100 + shape)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dscale", [1e-4, 300.0])
def test_attention_gradients_of_other_magnitudes(dtype, dscale):
    check_attention(dtype, [200, 90], [200, 90], 2, 2, 64, 3, seed=7, dscale=dscale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores(dtype):
    # nearly one-hot rows and a steep bias: the running maximum moves from tile to tile
    check_attention(dtype, [400], [400], 2, 2, 32, 1, seed=9, qscale=12.0)
    check_attention(dtype, [400], [400], 2, 2, 32, 3, seed=10, slope_scale=40.0)
    check_attention(dtype, [130], [130], 2, 2, 32, 0, seed=11, scale=-0.5)
    check_attention(dtype, [300], [300], 2, 2, 64, 2, seed=12, qscale=12.0)
    # a cap that bends nothing, and one that bends all
    check_attention(dtype, [140, 30], [140, 30], 2, 2, 64, 0, cap=5000.0, seed=13)
    check_attention(dtype, [1], [900], 2, 2, 64, 0, cap=5000.0, seed=14)
    check_attention(dtype, [140, 30], [140, 30], 2, 2, 64, 0, cap=0.01, seed=15)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [32, 64, 128])  # 16 rows at a time, 128, and 128 of twice the width
def test_attention_keeps_nan_and_infinities_in_their_example(dtype, channels):
    import pytorch_cluster_b200 as pc

    lens = [20, 45, 3, 90, 130, 7]
    g = gen(3)
    n, b = sum(lens), ids(lens)
    q, k, v, do = (rand(g, n, 2, channels, dtype=dtype) for _ in range(4))
    pos = rand(g, n, 3, dtype=torch.float32)
    slope = torch.tensor([0.5, 1.0], device="cuda")

    def run(*ts):
        ts = [t.clone().requires_grad_() for t in ts]
        out = pc.attention(*ts, b, b, pos, pos, slope)
        return [out.detach(), *torch.autograd.grad(out, ts, do)]

    clean = run(q, k, v)
    # two results within tolerance of the same value
    apart = attention_plain(q, k, v, lens, lens, pos, pos, slope, dout=do)
    apart = [2 * apart[n][1] for n in ("out", "dq", "dk", "dv")]
    others = [b != e for e in range(len(lens))]
    for bad_example, value in ((1, math.nan), (3, math.inf), (5, -math.inf)):
        for which in range(3):
            ts = [q.clone(), k.clone(), v.clone()]
            ts[which][b == bad_example] = value
            keep = others[bad_example]
            for c, got, tol in zip(clean, run(*ts), apart):
                assert_close(got[keep], c[keep].double(), tol[keep], (bad_example, which))
            assert not torch.isfinite(run(*ts)[0][b == bad_example]).all()
    # positions
    pos2 = pos.clone()
    pos2[b == 4] = math.nan
    out = pc.attention(q, k, v, b, b, pos2, pos2, slope)
    assert_close(out[b != 4], clean[0][b != 4].double(), apart[0][b != 4], "positions")
    assert torch.isnan(out[b == 4]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_without_keys(dtype):
    import pytorch_cluster_b200 as pc

    g = gen(4)
    q, k, v = (rand(g, 50, 2, 64, dtype=dtype).requires_grad_() for _ in range(3))
    # no example has both; ids at or above batch_size belong to none
    bq, bk = ids([20, 0, 30]), ids([0, 50, 0])
    out = pc.attention(q, k, v, bq, bk)
    assert (out == 0).all()
    assert all((t == 0).all() for t in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)))
    b = ids([20, 10, 20])
    out = pc.attention(q, k, v, b, b, batch_size=2)
    assert (out[30:] == 0).all() and (out[:30] != 0).any(-1).all()
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert all((t[30:] == 0).all() for t in grads)
    alone = pc.attention(q[:30], k[:30], v[:30], b[:30], b[:30])
    assert torch.equal(out[:30], alone)
    # garbage in the rows behind the last example does not matter
    k2, v2 = k.detach().clone(), v.detach().clone()
    k2[30:], v2[30:] = math.nan, math.inf
    assert torch.equal(pc.attention(q.detach(), k2, v2, b, b, batch_size=2), out)
    # empty sides
    e = torch.empty(0, 2, 64, device="cuda", dtype=dtype)
    assert pc.attention(e, k, v).shape == (0, 2, 64)
    out = pc.attention(q, e.requires_grad_(), e)
    assert (out == 0).all()
    out.sum().backward()
    assert (q.grad == 0).all()
    # keys that are infinitely far
    pos, far = torch.zeros(50, 1, device="cuda"), torch.full((50, 1), math.inf, device="cuda")
    out = pc.attention(q, k, v, pos_q=pos, pos_k=far, slope=torch.ones(2, device="cuda"))
    assert (out == 0).all()
    assert all((t == 0).all() for t in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_takes_strided_and_unaligned_inputs(dtype):
    import pytorch_cluster_b200 as pc

    g = gen(5)
    lens = [150, 40]
    n, b = sum(lens), ids(lens)
    joint = rand(g, n, 3, 4, 64, dtype=dtype)
    want = pc.attention(*(joint[:, i].contiguous() for i in range(3)), b, b)
    assert torch.equal(pc.attention(joint[:, 0], joint[:, 1], joint[:, 2], b, b), want)
    by_head = joint.permute(1, 2, 0, 3).contiguous()  # [3, heads, n, channels]
    assert torch.equal(pc.attention(*(by_head[i].transpose(0, 1) for i in range(3)), b, b), want)
    wide = torch.zeros(n, 3, 4, 65, device="cuda", dtype=dtype)  # rows that start anywhere
    wide[..., 1:] = joint
    odd = [wide[:, i, :, 1:] for i in range(3)]
    got = pc.attention(*odd, b, b)
    tol = attention_plain(*(joint[:, i] for i in range(3)), lens, lens)["out"][1]
    assert_close(got, want.double(), 2 * tol, "unaligned rows")
    assert torch.equal(pc.attention(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in odd), b, b), want)
    # a gradient that is broadcast, and keys shared by all rows of the batch's heads
    ts = [joint[:, i].clone().requires_grad_() for i in range(3)]
    out = pc.attention(*ts, b, b)
    one = torch.autograd.grad(out.sum(), ts, retain_graph=True)
    two = torch.autograd.grad(out, ts, torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    shared = joint[:, 1, :1].clone().requires_grad_()
    got, = torch.autograd.grad(pc.attention(ts[0], shared.expand(-1, 4, -1), ts[2], b, b).sum(), shared)
    each, = torch.autograd.grad(pc.attention(ts[0], k4 := shared.detach().expand(-1, 4, -1).clone().requires_grad_(),
                                             ts[2], b, b).sum(), k4)
    assert torch.allclose(got.float(), each.float().sum(1, keepdim=True), atol=4 * 4 * half_step(dtype) * each.abs().max().item())


def test_attention_gradient_against_differences():
    import pytorch_cluster_b200 as pc

    g = gen(6)
    lens = [23, 40, 1]
    n, b = sum(lens), ids(lens)
    ts = [rand(g, n, 2, 16, dtype=torch.float32) for _ in range(3)]
    pos, slope = rand(g, n, 2, dtype=torch.float32), torch.tensor([0.3, 1.1], device="cuda")
    do = rand(g, n, 2, 16, dtype=torch.float32)
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(pc.attention(*leaves, b, b, pos, pos, slope, cap=2.0), leaves, do)

    def value(ts):
        return (attention_plain(*ts, lens, lens, pos, pos, slope, cap=2.0)["out"][0] * do.double()).sum()

    h = 1e-5
    for i in range(3):
        step = torch.randn(ts[i].shape, generator=g, device="cuda").double()
        at = [t.double() for t in ts]
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * step, at[i] - h * step
        by_difference = (value(up) - value(down)) / (2 * h)
        by_gradient = (grads[i].double() * step).sum()
        # fp32 gradients: about a hundred roundings each; the difference's own error is below 1e-8
        assert abs(by_difference - by_gradient) <= 200 * U * (grads[i].double() * step).abs().sum() + 1e-6


def test_attention_same_bits_every_time_and_on_any_stream():
    import pytorch_cluster_b200 as pc

    g = gen(8)
    lens = [400, 100, 33]
    n, b = sum(lens), ids(lens)
    ts = [rand(g, n, 4, 64, dtype=torch.bfloat16).requires_grad_() for _ in range(3)]
    do = rand(g, n, 4, 64, dtype=torch.bfloat16)

    def run():
        out = pc.attention(*ts, b, b, batch_size=3)
        return [out, *torch.autograd.grad(out, ts, do)]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    third = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(first, second, third))


def test_attention_captured_and_replayed():
    import pytorch_cluster_b200 as pc

    g = gen(12)
    b, bq = ids([200, 300]), ids([1, 1])
    ts = [rand(g, 500, 4, 64, dtype=torch.bfloat16) for _ in range(3)]
    one = rand(g, 2, 4, 64, dtype=torch.bfloat16)

    def run():
        return (pc.attention(*ts, b, b, batch_size=2), pc.attention(one, *ts[1:], bq, b, batch_size=2),
                pc.attention(ts[0][..., :24], ts[1][..., :24], ts[2][..., :24], b, b, batch_size=2))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            outs = run()
        graphs.append((graph, outs))
    for seed in (1, 2):
        for t in [*ts, one]:
            t.copy_(rand(gen(20 + seed), *t.shape, dtype=t.dtype))
        for graph, outs in graphs:
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(outs, run()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens, channels", [([70, 200], 64), ([9, 30, 4], 32)])
def test_attention_gradients_of_some_inputs(dtype, lens, channels):
    import pytorch_cluster_b200 as pc

    g = gen(19)
    b, n = ids(lens), sum(lens)
    ts = [rand(g, n, 2, channels, dtype=dtype) for _ in range(3)]
    do = rand(g, n, 2, channels, dtype=dtype)

    def grads(wanted):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(ts)]
        out = pc.attention(*leaves, b, b, batch_size=len(lens))
        return dict(zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], do)))

    every = grads((0, 1, 2))
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        for i, got in grads(wanted).items():
            assert torch.equal(got, every[i]), (wanted, i)


def test_attention_training_step_captured():
    import pytorch_cluster_b200 as pc

    g = gen(13)
    lens = [130, 300]
    b, n = ids(lens), sum(lens)
    ts = [rand(g, n, 2, 64, dtype=torch.float16) for _ in range(3)]
    pos, slope = rand(g, n, 3, dtype=torch.float32), torch.tensor([1.0, 0.5], device="cuda")
    do = rand(g, n, 2, 64, dtype=torch.float16)

    def step():
        leaves = [t.detach().requires_grad_() for t in ts]
        out = pc.attention(*leaves, b, b, pos, pos, slope, batch_size=2)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in [*ts, do]:
        t.copy_(rand(g, *t.shape, dtype=t.dtype))
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, step()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [64, 128])
def test_attention_small_calls_split_over_the_keys(dtype, channels):
    check_attention(dtype, [1000], [1000], 2, 1, channels, 3, seed=31, train=False)
    check_attention(dtype, [200, 700, 77], [900, 300, 640], 2, 2, channels, 0, cap=20.0, seed=32, train=False)
    check_attention(dtype, [128, 128], [4000, 1], 1, 1, channels, 1, seed=33, train=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, groups, channels", [([1600, 0, 1900], 16, 16), ([300, 3000, 900], 4, 72)])
def test_attention_many_tiles_of_uneven_examples(dtype, lens, groups, channels):
    check_attention(dtype, lens, lens, 16, groups, channels, 3 if groups == 4 else 0, seed=41)


# ---- norm_rotate ---------------------------------------------------------------------------------------------

def rotate_plain(x, pos, freq, weight, eps, dy=None):
    u, dt = half_step(x.dtype), x.dtype
    x = x.double()
    c = x.size(-1)
    w = torch.ones(c, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    a = (pos.double() @ freq.double())[:, None]
    cos, sin = a.cos(), a.sin()
    # the angle is right to 64 bits, turned into 32 after its reduction to [-pi, pi]
    da = 4 * U + a.abs() * 2.0 ** -50

    def turn(z, way):
        l, h = z.chunk(2, -1)
        return torch.cat([l * cos - way * h * sin, h * cos + way * l * sin], -1)

    def turned(z):  # what the turn can be off by for a relative error of a few U in z
        l, h = z.abs().chunk(2, -1)
        s = (l + h) * (da + 12 * U)
        return torch.cat([s, s], -1)

    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    y = turn(n * w, 1)
    # the mean of squares: c roundings; then root, division, products
    rel = (c + 16) * U
    both = sum((n * w).abs().chunk(2, -1)).repeat(1, 1, 2)
    res = [y, u * y.abs() + turned(n * w) + rel * both + grid(dt)]
    if dy is not None:
        gy = turn(dy.double(), -1)
        eg = turned(dy.double())
        t = gy * w
        mean = (t * n).mean(-1, keepdim=True)
        dx = r * (t - n * mean)
        emean = (eg * w.abs() * n.abs()).mean(-1, keepdim=True) + 3 * rel * (t * n).abs().mean(-1, keepdim=True)
        edx = r * (eg * w.abs() + n.abs() * emean) + 6 * rel * r * (t.abs() + (n * mean).abs())
        dw = (gy * n).sum((0, 1))
        rows = x.size(0) * x.size(1)
        edw = (eg * n.abs() + (2 * rel + (rows / 64 + 64) * U) * (gy * n).abs()).sum((0, 1))
        res += [dx, edx + u * dx.abs() + grid(dt), dw, edw]
    return res


ROTATE = [
    # rows of q, rows of k (None: the same points), heads, key heads, channels, coordinates, weights, far
    (1, None, 1, 1, 2, 1, True, False),
    (7, None, 2, 1, 16, 3, True, False),
    (300, None, 8, 2, 64, 3, True, False),
    (257, 33, 3, 3, 32, 2, True, False),
    (5, 70, 4, 4, 128, 1, True, True),
    (1000, None, 4, 4, 6, 2, False, False),
    (33, None, 2, 2, 70, 8, True, False),
    (19, None, 5, 1, 256, 1, True, True),
    (64, 0, 2, 2, 48, 1, True, False),
    (129, None, 2, 2, 250, 3, True, False),
    (4099, None, 2, 1, 96, 1, False, True),
    (700, None, 1, 1, 256, 8, True, False),
    (600, 601, 1, 2, 256, 7, True, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(ROTATE)))
def test_norm_rotate_and_gradients(shape, dtype):
    import pytorch_cluster_b200 as pc

    m, n, heads, groups, c, dims, weights, far = ROTATE[shape]
    g = gen(shape)
    same = n is None
    n = m if same else n
    q = rand(g, m, heads, c, dtype=dtype, scale=3.0).requires_grad_()
    k = rand(g, n, groups, c, dtype=dtype).requires_grad_()
    if far:
        pos = [torch.randint(0, 3000000, (r, dims), generator=g, device="cuda").to(torch.float32) for r in (m, n)]
        freq = 10000.0 ** (-torch.arange(c // 2, device="cuda").float() / (c // 2)).expand(dims, -1)
    else:
        pos = [rand(g, r, dims, dtype=torch.float32) for r in (m, n)]
        freq = 5 * rand(g, dims, c // 2, dtype=torch.float32)
    if same:
        pos[1] = pos[0]
    w = [(1 + 0.2 * torch.randn(c, generator=g, device="cuda")).requires_grad_() if weights else None for _ in range(2)]
    out = pc.norm_rotate(q, k, *pos, freq, *w, eps=1e-5)
    dy = [rand(g, *t.shape, dtype=dtype) for t in (q, k)]
    leaves = [q, k] + [t for t in w if t is not None]
    grads = torch.autograd.grad(out, leaves, dy)
    for i, x in enumerate((q, k)):
        wi = None if w[i] is None else w[i].detach()
        y, ty, dx, tx, dw, tw = rotate_plain(x.detach(), pos[i], freq, wi, 1e-5, dy[i])
        assert_close(out[i].detach(), y, ty, "qk"[i])
        assert_close(grads[i], dx, tx, "d" + "qk"[i])
        if weights:
            assert_close(grads[2 + i], dw, tw, "dweight_" + "qk"[i])
    with torch.no_grad():
        again = pc.norm_rotate(q, k, pos[0].double(), pos[1].double(), freq.double(), *w, eps=1e-5)
    assert all(torch.equal(x, y) for x, y in zip(again, out))


def test_norm_rotate_strides_positions_and_special_rows():
    import pytorch_cluster_b200 as pc

    g = gen(1)
    joint = rand(g, 100, 3, 4, 64, dtype=torch.bfloat16)
    freq = rand(g, 1, 32, dtype=torch.float32)
    place = torch.arange(100, device="cuda")
    want = pc.norm_rotate(joint[:, 0].contiguous(), joint[:, 1].contiguous(), place, place, freq)
    for q, k in ((joint[:, 0], joint[:, 1]), (joint[:, 0].transpose(1, 2).contiguous().transpose(1, 2), joint[:, 1])):
        assert all(torch.equal(a, b) for a, b in zip(pc.norm_rotate(q, k, place, place.clone().float(), freq), want))
    wide = torch.zeros(100, 4, 65, device="cuda", dtype=torch.bfloat16)
    wide[..., 1:] = joint[:, 0]
    got = pc.norm_rotate(wide[..., 1:], joint[:, 1], place, place, freq)
    y, tol = rotate_plain(joint[:, 0], place[:, None], freq, None, 1e-6)
    assert_close(got[0], y, tol, "unaligned rows")
    # zeros stay zeros (eps), NaN and infinities stay in their head's row
    x = joint[:, 0].clone()
    x[3, 1], x[4, 2, 5], x[5, 0, 0] = 0, math.nan, math.inf
    a, _ = pc.norm_rotate(x, joint[:, 1], place, place, freq)
    assert (a[3, 1] == 0).all() and torch.isnan(a[4, 2]).all() and not torch.isfinite(a[5, 0]).all()
    keep = torch.ones(100, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = keep[4, 2] = keep[5, 0] = False
    assert torch.equal(a[keep], want[0][keep])
    # equal distances give equal products
    e = rand(g, 1, 1, 64, dtype=torch.float32).expand(100, 1, 64)
    f = rand(g, 1, 1, 64, dtype=torch.float32).expand(100, 1, 64)
    a, b = pc.norm_rotate(e, f, place + 1000000, place + 1000007, freq)
    dot = (a.double() * b.double()).sum(-1)
    assert (dot - dot[0]).abs().max() <= 64 * 64 * U


# ---- gather_rows ---------------------------------------------------------------------------------------------

GATHER = [
    # rows, edges, channels, index pattern
    (1, 1, 1, "any"), (5, 3, 8, "any"), (1000, 16384, 32, "any"), (3, 5000, 64, "any"), (1, 9000, 20, "any"),
    (100, 70001, 128, "skewed"), (70000, 5000, 7, "any"), (513, 4097, 130, "padded"), (40, 333, 3, "padded"),
    (300000, 20000, 4, "any"), (17, 0, 16, "any"), (0, 12, 16, "padded"), (4096, 4096, 64, "sorted"),
    (9, 64, 16, "all"), (1000000, 100, 16, "any"),
    # around the sizes at which the sort changes: one block, few blocks, many
    (700, 16383, 8, "all"), (700, 16385, 8, "padded"), (2000, 131073, 8, "any"), (2000, 131072, 8, "skewed"),
    (300000, 16384, 4, "any"), (300000, 140001, 4, "padded"), (40, 16385, 8, "all"),
    (4096, 4096, 8, "skewed"), (4097, 4096, 8, "padded"), (4096, 4097, 8, "any"), (3, 4096, 72, "all"),
    (4095, 7, 9, "padded"), (1, 1, 300, "all"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(GATHER)))
def test_gather_rows_and_gradient(shape, dtype):
    import pytorch_cluster_b200 as pc

    rows, edges, c, pattern = GATHER[shape]
    g = gen(shape)
    x = rand(g, rows, c, dtype=dtype).requires_grad_()
    index = torch.randint(0, max(rows, 1), (edges,), generator=g, device="cuda")
    if pattern == "skewed":
        index = (torch.rand(edges, generator=g, device="cuda") ** 4 * rows).long()
    if pattern == "sorted":
        index = index.sort().values
    if pattern == "all":
        index = torch.full_like(index, rows - 1)
    if pattern == "padded":
        index[::3] = -1
        index[1::7] = rows
        index[2::11] = 2 ** 40
    there = (index >= 0) & (index < rows)
    scale = 1.7
    out = pc.gather_rows(x, index, scale)
    dout = rand(g, edges, c, dtype=dtype)
    dx, = torch.autograd.grad(out, x, dout)
    u, s32 = half_step(dtype), torch.tensor(scale).float().double().item()
    want = torch.zeros(edges, c, dtype=torch.float64, device="cuda")
    want[there] = x.detach().double()[index[there]] * s32
    assert_close(out.detach(), want, (u + U) * want.abs() + grid(dtype), "out")
    sums = torch.zeros(rows, c, dtype=torch.float64, device="cuda").index_add_(0, index[there], dout[there].double())
    size = torch.zeros(rows, c, dtype=torch.float64, device="cuda").index_add_(0, index[there], dout[there].double().abs())
    count = torch.bincount(index[there], minlength=rows).double()[:, None] if rows else sums
    # pieces of 64, joined: fewer roundings than terms
    assert_close(dx, sums * s32, s32 * (size * U * (count + 2) + u * sums.abs()) + grid(dtype), "dx")
    assert torch.equal(torch.autograd.grad(pc.gather_rows(x, index, scale), x, dout)[0], dx)


def test_gather_rows_strided_other_stream_and_broadcast_gradient():
    import pytorch_cluster_b200 as pc

    g = gen(2)
    x = rand(g, 64, 200, dtype=torch.float32).t()  # [200, 64], column-major
    index = torch.randint(0, 200, (2, 3000), generator=g, device="cuda").t()[:, 1]  # strided
    x.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = pc.gather_rows(x, index)
        dx, = torch.autograd.grad(out.sum(), x)
    torch.cuda.synchronize()
    assert torch.equal(out, x.detach()[index])
    assert torch.equal(dx, torch.bincount(index, minlength=200).float()[:, None].expand(-1, 64))


# ---- together ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_on_the_graph(dtype):
    """Neighbour features along knn_graph's edges, then norm, rotation and attention inside each cloud."""
    import pytorch_cluster_b200 as pc

    g = gen(11)
    lens, heads, c = [200, 64, 1, 300], 2, 32
    n, b = sum(lens), ids(lens)
    pos = rand(g, n, 3, dtype=torch.float32)
    x = rand(g, n, heads * c, dtype=dtype).requires_grad_()
    edges = pc.knn_graph(pos, 8, b, loop=True)
    freq, slope = 2 * rand(g, 3, c // 2, dtype=torch.float32), torch.tensor([0.5, 0.25], device="cuda")
    w = torch.ones(c, device="cuda").requires_grad_()

    def layer(gather, rotate, attend, x):
        near = torch.zeros(n, heads * c, device="cuda", dtype=x.dtype).index_add(0, edges[1], gather(x, edges[0], 0.25))
        q, k = rotate(near.view(n, heads, c), x.view(n, heads, c), pos, pos, freq, w, w)
        return attend(q, k, x.view(n, heads, c))

    out = layer(pc.gather_rows, pc.norm_rotate, lambda q, k, v: pc.attention(q, k, v, b, b, pos, pos, slope), x)
    dout = rand(g, *out.shape, dtype=dtype)
    got = [out, *torch.autograd.grad(out, (x, w), dout)]

    def rotate(q, k, pq, pk, f, wq, wk):
        return [rotate_graph(t, pq, f, wt) for t, wt in ((q, wq), (k, wk))]

    def rotate_graph(t, p, f, wt):
        z = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wt.double()
        a = (p.double() @ f.double())[:, None]
        l, h = z.chunk(2, -1)
        return torch.cat([l * a.cos() - h * a.sin(), h * a.cos() + l * a.sin()], -1)

    def attend(q, k, v):
        same = b[:, None] == b[None]
        s = torch.einsum("ihc,jhc->hij", q, k) * c ** -0.5
        s = s - slope.double()[:, None, None] * torch.cdist(pos.double(), pos.double(),
                                                            compute_mode="donot_use_mm_for_euclid_dist")
        return torch.einsum("hij,jhc->ihc", s.masked_fill(~same, -math.inf).softmax(-1), v)

    x64 = x.detach().double().requires_grad_()
    ref = layer(lambda t, i, s: t[i] * s, rotate, attend, x64)
    want = [ref, *torch.autograd.grad(ref, (x64, w), dout.double())]
    # a chain of five roundings to the type, each of a value of the size of the result's rows: in the mean
    # well below 16 of them
    for a, z in zip(got, want):
        assert (a.double() - z.double()).norm() <= 16 * half_step(dtype) * z.double().norm()


def test_attention_long_examples_same_bits():
    """Every wait of the tensor-core kernels counts here: thousands of steps, slow and fast ones."""
    import pytorch_cluster_b200 as pc

    g = gen(30)
    lens = [2515, 1594, 2290, 1852]
    n, b = sum(lens), ids(lens)
    for channels, dims, cap in ((64, 3, None), (64, 0, None), (32, 8, 4.0), (128, 2, None), (128, 0, 4.0)):
        ts = [rand(g, n, 4, channels, dtype=torch.bfloat16).requires_grad_() for _ in range(3)]
        extra = {}
        if dims:
            pos = rand(g, n, dims, dtype=torch.float32)
            extra = dict(pos_q=pos, pos_k=pos, slope=torch.tensor([1.0, 0.5, 0.1, 0.0], device="cuda"))
        do = rand(g, n, 4, channels, dtype=torch.bfloat16)
        first = None
        for _ in range(6):
            out = pc.attention(*ts, b, b, cap=cap, batch_size=4, **extra)
            got = [out.detach(), *torch.autograd.grad(out, ts, do)]
            first = first or got
            assert all(torch.equal(x, y) for x, y in zip(first, got))
        assert all(torch.isfinite(x).all() for x in first)
