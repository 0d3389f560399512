"""``norm_rope_func`` -- norm of queries and keys per head, and their rotation by position, in one pass.

What a layer runs between its projection and ``flash_bias_func`` where positions also enter as rotations, or where queries
and keys are normalised per head; it stands beside ``layout.prepare_bhsd`` (cast, cosine normalisation and scale, the form of
2_Vision_Transformer/swin_transformer_v2.py:194-199), and unlike it has a backward pass.  The host path is native code,
csrc/torch_paged.h.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .flash_bias import _op

__all__ = ["norm_rope_func"]


def norm_rope_func(q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor] = None,
                   inv_freq: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, axes: Optional[Sequence[int]] = None, interleaved: bool = False,
                   eps: float = 1e-6):
    """``(q', k')`` as new tensors; ``x' = rotate(x * rsqrt(mean(x^2) + eps) * weight)``, computed in fp32 and rounded once.

    q: (batch, seqlen, nheads, headdim), fp16 or bf16, headdim up to 128, any strides (slices of a fused projection are read
        where they lie; a last dimension that is not contiguous is copied).  k: the same with its own number of heads, or None.
    positions: int32 or int64, (seqlen) or (batch | 1, seqlen); with ``axes`` (A, seqlen) or (A, batch | 1, seqlen), A up to 4
        (time, height, width).  May be negative.
    inv_freq: fp32 or fp64, one angular frequency per rotated pair of columns: the first ``2 * len(inv_freq)`` columns of every
        head turn by ``position * inv_freq`` (an angle taken in 64 bits), the others pass.  None (with positions None): no
        rotation.
    q_weight, k_weight: headdim values, fp32, fp16 or bf16 (both of one type); None: that tensor is not normalised.
    axes: the position axis of every pair, e.g. ``[0] * 16 + [1] * 24 + [2] * 24``.
    interleaved: pair p is columns (2p, 2p + 1) instead of (p, p + len(inv_freq)).

    Gradients for q, k and the weights (fp32 sums over all rows, in a fixed order); inv_freq and positions are constants.
    They cannot be differentiated again.
    """
    return _op().norm_rope(q, k, positions, inv_freq, q_weight, k_weight, axes, interleaved, eps)
