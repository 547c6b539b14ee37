"""``gather_rows``: rows of node features along an edge list, differentiable, on top of
``torch.ops.torch_cluster.gather_rows``."""
import torch


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
    return torch.ops.torch_cluster.gather_rows(x, index, float(scale))
