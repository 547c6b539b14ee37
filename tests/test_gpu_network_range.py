"""gather_rows, norm_rotate and attention where values lie far apart or rows belong to nothing: against their definitions
in 64 bits, with the tolerances of test_gpu_network."""
import math

import pytest
import torch
from test_gpu_network import DTYPES, assert_close, attention_plain, gen, ids, rand

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
