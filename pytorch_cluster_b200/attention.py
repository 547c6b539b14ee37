"""``attention``: softmax attention inside the examples of a ragged batch, differentiable, on top of
``torch.ops.torch_cluster.attention``."""
from typing import Optional, Tuple

import torch


def _segments(batch_q: Optional[torch.Tensor], batch_k: Optional[torch.Tensor], rows_q: int, rows_k: int,
              batch_size: Optional[int]) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    # Segment boundaries as for knn: B comes from the batch vectors (one host read each) unless it is given.
    if batch_q is None and batch_k is None:
        assert batch_size is None or batch_size == 1
        return None, None
    assert batch_q is not None and batch_k is not None
    assert batch_q.numel() == rows_q and batch_k.numel() == rows_k
    same = batch_q is batch_k
    examples = 1
    if batch_size is not None:
        examples = batch_size
    else:
        if batch_q.numel() > 0:
            examples = max(examples, torch.ops.torch_cluster.batch_info(batch_q)[0])
        if not same and batch_k.numel() > 0:
            examples = max(examples, torch.ops.torch_cluster.batch_info(batch_k)[0])
    assert examples > 0
    ptr_q = torch.ops.torch_cluster.segment_ptr(batch_q, examples)
    return ptr_q, ptr_q if same else torch.ops.torch_cluster.segment_ptr(batch_k, examples)


def _places(name: str, t: torch.Tensor) -> torch.Tensor:
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{name} receives no gradient here: pass {name}.detach()")
    t = t.float()
    return t.view(-1, 1) if t.dim() == 1 and name != "slope" else t


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    batch_q: Optional[torch.Tensor] = None,
    batch_k: Optional[torch.Tensor] = None,
    pos_q: Optional[torch.Tensor] = None,
    pos_k: Optional[torch.Tensor] = None,
    slope: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    cap: Optional[float] = None,
    batch_size: Optional[int] = None,
) -> torch.Tensor:
    r"""Softmax attention of every row of :obj:`q` over the rows of :obj:`k` and :obj:`v` of the same example.

    The score of query i and key j in head h is ``t - slope[h] * |pos_q[i] - pos_k[j]|`` with
    ``t = scale * (q_i . k_j)``, or ``t = cap * tanh(scale * (q_i . k_j) / cap)`` where a cap is given.

    Args:
        q: ``[M, H, C]``; k, v: ``[N, G, C]``; float, half or bfloat16 CUDA tensors of one type, C at most 128.
            H is a multiple of G: head h reads key head ``h // (H // G)``.  Channels are contiguous or the
            tensor is copied; other strides are free (slices of a joint projection are taken as they stand).
        batch_q, batch_k: sorted int64 example ids of the rows, as for :func:`knn`; None for one example.  The rows of
            one example see nothing of another, its NaNs included.
        pos_q, pos_k, slope: coordinates ``[M, D]`` and ``[N, D]`` (D at most 8, taken as fp32) and ``[H]``
            slopes of the bias by distance; all three or none.  They are constants: no gradient reaches them.
        scale: of the dot products, a finite number, ``C ** -0.5`` by default.
        cap: a positive number, or None; scale, cap and their quotient are numbers of 32 bits.
        batch_size: the number of examples; skips its inference and the host reads that takes (needed under stream
            capture).  Rows with ids at or above it belong to no example: zeros, without a gradient.

    Returns ``[M, H, C]``.  A query without keys gives zeros.  A few queries over many keys (pooling by a
    learned query, one new token) are split over the keys and joined.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be CUDA tensor")
        if t.dim() != 3:
            raise RuntimeError("Input mismatch")
    if scale is None:
        scale = float(q.size(-1)) ** -0.5 if q.size(-1) > 0 else 1.0
    if cap is not None and not (cap > 0.0 and cap < float("inf")):
        raise ValueError("`cap` needs to be positive and finite")
    if (pos_q is None) != (pos_k is None) or (pos_q is None) != (slope is None):
        raise ValueError("`pos_q`, `pos_k` and `slope` come together")
    if pos_q is not None and pos_k is not None and slope is not None:
        same = pos_q is pos_k
        pos_q = _places("pos_q", pos_q)
        pos_k = pos_q if same else _places("pos_k", pos_k)
        slope = _places("slope", slope)
    ptr_q, ptr_k = _segments(batch_q, batch_k, q.size(0), k.size(0), batch_size)
    return torch.ops.torch_cluster.attention(q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, float(scale),
                                             0.0 if cap is None else float(cap))
