"""``norm_rotate``: RMS norm of queries and keys for each head and rotation by the points' coordinates, in one
pass, differentiable, on top of ``torch.ops.torch_cluster.norm_rotate``."""
from typing import Optional, Tuple

import torch


def _constant(name: str, t: torch.Tensor) -> torch.Tensor:
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{name} receives no gradient here: pass {name}.detach()")
    return t


def _position(name: str, p: torch.Tensor) -> torch.Tensor:
    p = _constant(name, p)
    if not p.is_floating_point():
        p = p.double()
    elif p.dtype != torch.float32 and p.dtype != torch.float64:
        p = p.float()
    return p.view(-1, 1) if p.dim() == 1 else p


def norm_rotate(
    q: torch.Tensor,
    k: torch.Tensor,
    pos_q: torch.Tensor,
    pos_k: torch.Tensor,
    freq: torch.Tensor,
    weight_q: Optional[torch.Tensor] = None,
    weight_k: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""RMS norm of every head's query and key, then rotation by the coordinates of its point.

    For a row ``x`` of ``C`` channels at position ``p``: ``u = weight * x / sqrt(mean(x ** 2) + eps)``, and the
    pair ``(u[c], u[c + C / 2])`` is turned by the angle ``p @ freq[:, c]``.  Dot products of rotated queries and
    keys then depend on the difference of their positions only.  One coordinate with geometric
    frequencies is the rotation of sequence positions; several turn by points of space.

    Args:
        q, k: ``[M, H, C]`` and ``[N, G, C]`` float, half or bfloat16 CUDA tensors of one type; C even, at most
            256.  Their channels are contiguous or they are copied; other strides are free.
        pos_q, pos_k: ``[M, D]`` and ``[N, D]`` (or ``[M]``, ``[N]``), D at most 8, float or double; whole numbers
            are taken as double.  Pass the same tensor twice where queries and keys are the same points.
        freq: ``[D, C / 2]`` float or double, in radians per unit.  Angles are formed in 64 bits.
        weight_q, weight_k: ``[C]``, or None for ones.
        eps: added to the mean square.

    Returns the rotated q and k, contiguous, of the input type.  Gradients reach q, k and the weights;
    positions and frequencies are constants.
    """
    if not q.is_cuda:
        raise RuntimeError("q must be CUDA tensor")
    same = pos_q is pos_k
    pos_q = _position("pos_q", pos_q)
    pos_k = pos_q if same else _position("pos_k", pos_k)
    if pos_q.dtype != pos_k.dtype:
        pos_q, pos_k = pos_q.double(), pos_k.double()
    _constant("freq", freq)
    if weight_q is not None:
        weight_q = weight_q.float()
    if weight_k is not None:
        weight_k = weight_k.float()
    return torch.ops.torch_cluster.norm_rotate(q, k, pos_q, pos_k, freq, weight_q, weight_k, float(eps))
