"""RMS norm of queries and keys per head with the rotary embedding, in one pass.

What runs between a layer's projections and its KV cache: the caches of this package
store keys as they are given, so keys are normalised and rotated before they are
appended and queries before they are decoded.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _kv8, _lib


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


def aligned_rows(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """t ((rows, heads, D)) with 16-byte aligned rows, copied if it has none, and its row
    and head strides in elements."""
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    s0, s1 = (s0 if n > 1 else 0), (s1 if h > 1 else 0)
    if s2 != 1 or s0 % 8 or s1 % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1 = h * d, d
    return t, s0, s1


def output_rows(t: torch.Tensor, like: torch.Tensor, name: str) -> Tuple[int, int]:
    """Row and head strides of a caller's output tensor; refused if its rows are not
    aligned or overlap."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise RuntimeError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    n, h, _ = t.shape
    s0, s1, s2 = t.stride()
    if (n > 1 and s0 == 0) or (h > 1 and s1 == 0):
        raise RuntimeError(f"{name} has rows that overlap")
    s0, s1 = (s0 if n > 1 else 0), (s1 if h > 1 else 0)
    if s2 != 1 or s0 % 8 or s1 % 8 or t.data_ptr() % 16:
        raise RuntimeError(f"{name} needs unit channel stride and 16-byte aligned rows")
    return s0, s1


def no_grad_inputs(*tensors: Optional[torch.Tensor]) -> None:
    """These operators have no backward pass: refuse inputs that ask for one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("this operator has no backward pass: call it under torch.no_grad() or on detached tensors")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalise every head of q (N, Hq, D) and k (N, H, D) and rotate it to its token's
    position; float16 or bfloat16, float32 inside, rounded once.  Returns (q_out, k_out).

    positions: (N,) int32 or int64 rows of ``table`` (:func:`rope_table`); a negative
    position marks a padding row, whose output is left as it was; one past the table
    does the same and sets a sticky error bit (:func:`kv8_error_flags`).
    table: (max_positions, R) float32; channels from R on are normalised only.
    q_weight / k_weight: (D,) of q's dtype or float32, both or neither; without them
    there is no norm, only the rotation.
    interleaved: rotate channels (2i, 2i + 1) together instead of (i, i + R / 2).
    q_out / k_out: given tensors, also q and k themselves (same strides); q and k may be
    strided views, as of one fused projection.  D and R are multiples of 16, D <= 256.
    """
    dev = _lib.require_cuda(q, k, positions, table, q_weight, k_weight, q_out, k_out)
    no_grad_inputs(q, k, q_weight, k_weight, table)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise RuntimeError("q must be (N, Hq, D) and k (N, H, D)")
    dt = _kv8.DTYPES.get(q.dtype)
    if dt is None or k.dtype != q.dtype:
        raise RuntimeError(f"q and k must both be float16 or both bfloat16, got {q.dtype} and {k.dtype}")
    n, hq, d = q.shape
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (n,):
        raise RuntimeError(f"positions must be ({n},) int32 or int64")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise RuntimeError("table must be (max_positions, R) float32, contiguous")
    if (q_weight is None) != (k_weight is None):
        raise RuntimeError("q_weight and k_weight must be given together")
    w32 = False
    if q_weight is not None:
        if q_weight.shape != (d,) or k_weight.shape != (d,):
            raise RuntimeError(f"q_weight and k_weight must be ({d},)")
        w32 = q_weight.dtype == torch.float32
        if k_weight.dtype != q_weight.dtype or not (w32 or q_weight.dtype == q.dtype):
            raise RuntimeError(f"q_weight and k_weight must both be {q.dtype} or both float32")
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    positions = positions.contiguous()
    a = _kv8.QkNormRopeArgs()
    if q_out is None:
        q_out = torch.empty((n, hq, d), dtype=q.dtype, device=dev)
    if k_out is None:
        k_out = torch.empty((n, k.shape[1], d), dtype=q.dtype, device=dev)
    a.qo_s_row, a.qo_s_head = output_rows(q_out, q, "q_out")
    a.ko_s_row, a.ko_s_head = output_rows(k_out, k, "k_out")
    q, a.q_s_row, a.q_s_head = aligned_rows(q)
    k, a.k_s_row, a.k_s_head = aligned_rows(k)
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.q_weight, a.k_weight = _lib.ptr(q_weight), _lib.ptr(k_weight)
    a.positions, a.table, a.table_rows = positions.data_ptr(), table.data_ptr(), table.shape[0]
    a.rows, a.num_q_heads, a.num_k_heads, a.head_dim, a.rot = n, hq, k.shape[1], d, table.shape[1]
    a.interleaved, a.positions64, a.weight_f32 = interleaved, positions.dtype == torch.int64, w32
    a.dtype, a.eps = dt, eps
    _kv8.launch(dev, "kitty_qk_norm_rope", a)
    return q_out, k_out
