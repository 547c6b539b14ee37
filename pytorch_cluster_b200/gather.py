"""``gather_rows``: rows of node features along an edge list, differentiable, on top of
``torch.ops.torch_cluster.gather_rows``."""
import torch
from torch.autograd.function import once_differentiable


class _GatherRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, index, scale):
        ctx.save_for_backward(index)
        ctx.rows, ctx.scale = x.size(0), scale
        return torch.ops.torch_cluster.gather_rows(x, index, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        index, = ctx.saved_tensors
        return torch.ops.torch_cluster.gather_rows_backward(dout, index, ctx.rows, ctx.scale), None, None


def gather_rows(
    x: torch.Tensor,
    index: torch.Tensor,
    scale: float = 1.0,
) -> torch.Tensor:
    r"""Rows of :obj:`x` by :obj:`index`, times :obj:`scale`: ``out[e] = scale * x[index[e]]``.

    For the features of the neighbours along the edges of :func:`knn_graph` or :func:`radius_graph`
    (``gather_rows(x, edge_index[0])``), and for embeddings of node types.  The gradient adds the rows of
    every index in ascending order of ``e``, in fp32 and without atomics: the same bits every time.

    Args:
        x: ``[N, C]`` float, half or bfloat16 CUDA tensor.
        index: ``[E]`` int64.  An index outside ``[0, N)`` is padding: it gives a row of zeros and receives
            no gradient.
        scale: a number.

    Returns ``[E, C]`` of x's type.
    """
    if not x.is_cuda:
        raise RuntimeError("x must be CUDA tensor")
    scale = float(scale)
    if torch.is_grad_enabled() and x.requires_grad:
        return _GatherRows.apply(x, index, scale)
    return torch.ops.torch_cluster.gather_rows(x, index, scale)
