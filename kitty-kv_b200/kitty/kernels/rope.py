"""RMS norm of queries and keys per head with the rotary embedding, in one pass.

What runs between a layer's projections and its KV cache: the caches of this package
store keys as they are given, so keys are normalised and rotated before they are
appended and queries before they are decoded.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _kv8


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0,
               inv_freq: Optional[torch.Tensor] = None, device: Optional[torch.device] = None) -> torch.Tensor:
    """Cosines and sines of the rotary embedding: (max_positions, rotary_dim) float32,
    row p holding cos(p f_i) for i < rotary_dim / 2 and then sin(p f_i), with
    f_i = base^(-2 i / rotary_dim) or ``inv_freq`` ((rotary_dim / 2,), for scaled
    variants).  The angles are formed in float64: in float32 those of far positions
    would be off by more than the table's rounding."""
    if rotary_dim <= 0 or rotary_dim % 2 or max_positions < 0:
        raise RuntimeError("rotary_dim must be positive and even, max_positions non-negative")
    if inv_freq is None:
        i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
        inv_freq = base ** (-2.0 * i / rotary_dim)
    elif inv_freq.numel() != rotary_dim // 2:
        raise RuntimeError(f"inv_freq must have {rotary_dim // 2} entries")
    f = inv_freq.to(device=device, dtype=torch.float64).reshape(1, -1)
    angle = torch.arange(max_positions, dtype=torch.float64, device=f.device).unsqueeze(1) * f
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.float32)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalise every head of q (N, Hq, D) and k (N, H, D) and rotate it to its token's
    position; float16 or bfloat16, float32 inside, rounded once.  Returns (q_out, k_out).

    positions: (N,) int32 or int64 rows of ``table`` (:func:`rope_table`); a negative
    position marks a padding row, whose output is left as it was (undefined where the
    output is made here); one past the table does the same and sets a sticky error bit
    (:func:`kv8_error_flags`).
    table: (max_positions, R) float32; channels from R on are normalised only.
    q_weight / k_weight: (D,) of q's dtype or float32, both or neither; without them
    there is no norm, only the rotation.
    interleaved: rotate channels (2i, 2i + 1) together instead of (i, i + R / 2).
    q_out / k_out: given tensors, also q and k themselves (same strides); any other overlap
    with an input or one another is refused.  q and k may be strided views, as of one fused
    projection.  D and R are multiples of 16, D <= 256.
    """
    return _kv8.ops().qk_norm_rope(q, k, positions, table, q_weight, k_weight, eps, interleaved, q_out, k_out)
