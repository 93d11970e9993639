"""The paged KV cache of 8-bit codes with one scale per block of tokens and KV head.

For layers that do not stand 2 bits a value, and for keys and values that are to be
kept close to 16 bits at half their size.  The arrays are the caller's (or those of
``kitty.PagedKVCache8``), one set per layer:

* ``key_codes`` / ``value_codes``: (P, H, G, D) ``torch.float8_e4m3fn`` or ``torch.int8``,
  ``key_scale`` / ``value_scale``: (P, H) float32: a value is code * scale;
* ``tail_k`` / ``tail_v``: (slots, H, G, D) float16 or bfloat16: the tokens of each
  slot's last block while it is not full;
* ``block_table``: (slots, M) int32 pages, ``lengths``: (slots,) int32 tokens.

Token t of a slot with n tokens is in page ``block_table[slot, t // G]`` if that block
is full, ``(t // G + 1) * G <= n``, and otherwise in row ``t % G`` of the slot's tail.
G is a multiple of 32 up to 256, D a multiple of 16 up to 256.

Pools, tails, lengths and scales must be contiguous.  What only device data shows (a
page outside the pool, a slot given twice in one write, offsets that decrease) is
skipped without touching memory out of bounds and sets a sticky error bit
(:func:`kv8_error_flags`).  No host synchronisation: every call can be captured in a
CUDA graph.  No backward passes.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _kv8, _lib
from .rope import aligned_rows, no_grad_inputs, output_rows


def _fill_cache(c: _kv8.Cache, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k,
                tail_v) -> None:
    """Check the arrays of a cache against one another and describe them to the library."""
    if key_codes.dim() != 4 or value_codes.shape != key_codes.shape:
        raise RuntimeError("key_codes and value_codes must both be (P, H, G, D)")
    pages, h, g, d = key_codes.shape
    code = _kv8.CODES.get(key_codes.dtype)
    if code is None or value_codes.dtype != key_codes.dtype:
        raise RuntimeError("key_codes and value_codes must both be float8_e4m3fn or both int8")
    slots = lengths.shape[0] if lengths.dim() == 1 else -1
    if lengths.dtype != torch.int32 or slots < 0:
        raise RuntimeError("lengths must be (slots,) int32")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != slots:
        raise RuntimeError("block_table must be (slots, M) int32 with a row for each entry of lengths")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise RuntimeError("block_table rows need unit stride")
    dt = _kv8.DTYPES.get(tail_k.dtype)
    if dt is None or tail_v.dtype != tail_k.dtype:
        raise RuntimeError("tail_k and tail_v must both be float16 or both bfloat16")
    if tail_k.shape != (slots, h, g, d) or tail_v.shape != tail_k.shape:
        raise RuntimeError(f"tail_k and tail_v must be ({slots}, {h}, {g}, {d})")
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32 or key_scale.shape != (pages, h) or \
            value_scale.shape != (pages, h):
        raise RuntimeError(f"key_scale and value_scale must be ({pages}, {h}) float32")
    if not (key_codes.is_contiguous() and value_codes.is_contiguous() and key_scale.is_contiguous() and
            value_scale.is_contiguous() and tail_k.is_contiguous() and tail_v.is_contiguous() and
            lengths.is_contiguous()):
        raise RuntimeError("pools, scales, tails and lengths must be contiguous")
    c.key_codes, c.value_codes = key_codes.data_ptr(), value_codes.data_ptr()
    c.key_scale, c.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    c.tail_k, c.tail_v = tail_k.data_ptr(), tail_v.data_ptr()
    c.block_table, c.lengths = block_table.data_ptr(), lengths.data_ptr()
    c.bt_s_slot, c.pages, c.slots, c.max_pages = block_table.stride(0), pages, slots, block_table.shape[1]
    c.num_heads, c.head_dim, c.page_size, c.code, c.dtype = h, d, g, code, dt


def _index(t: Optional[torch.Tensor], name: str, n: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError(f"{name} must be ({n},) int32")
    return t.contiguous()


def write_kv8(key: torch.Tensor, value: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor,
              key_codes: torch.Tensor, value_codes: torch.Tensor, key_scale: torch.Tensor,
              value_scale: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor,
              row_offsets: Optional[torch.Tensor] = None, seq_map: Optional[torch.Tensor] = None) -> None:
    """Append rows of key / value ((N, H, D), the tails' dtype) to n slots, in one launch.

    Entry i's rows are ``row_offsets[i]`` .. ``row_offsets[i + 1] - 1`` ((n + 1,) int32;
    without it every entry has one row); they go behind the ``lengths[slot]`` tokens that
    slot ``seq_map[i]`` ((n,) int32, distinct; without it i) has.  Blocks that fill are quantised into
    the pages that ``block_table`` holds for them, the rest stays in the tail.  ``lengths``
    is not changed: add the new tokens before the next call on this cache.  Rows behind
    the last offset are ignored.
    """
    dev = _lib.require_cuda(key, value, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k,
                            tail_v, row_offsets, seq_map)
    no_grad_inputs(key, value)
    a = _kv8.WriteArgs()
    _fill_cache(a.cache, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v)
    if key.dim() != 3 or key.shape != value.shape or tuple(key.shape[1:]) != (a.cache.num_heads, a.cache.head_dim) or \
            key.dtype != tail_k.dtype or value.dtype != tail_k.dtype:
        raise RuntimeError(f"key and value must be (N, {a.cache.num_heads}, {a.cache.head_dim}) {tail_k.dtype}")
    rows = key.shape[0]
    n = seq_map.numel() if seq_map is not None else rows if row_offsets is None else row_offsets.numel() - 1
    if n < 0:
        raise RuntimeError("row_offsets must have n + 1 entries")
    if row_offsets is None and n != rows:
        raise RuntimeError("without row_offsets key and value must have one row for each slot")
    seq_map, row_offsets = _index(seq_map, "seq_map", n), _index(row_offsets, "row_offsets", n + 1)
    key, a.k_s_row, a.k_s_head = aligned_rows(key)
    value, a.v_s_row, a.v_s_head = aligned_rows(value)
    a.key, a.value, a.n, a.rows = key.data_ptr(), value.data_ptr(), n, rows
    a.row_offsets, a.seq_map = _lib.ptr(row_offsets), _lib.ptr(seq_map)
    _kv8.launch(dev, "kitty_kv8_write", a)


def read_kv8(lengths: torch.Tensor, block_table: torch.Tensor, key_codes: torch.Tensor, value_codes: torch.Tensor,
             key_scale: torch.Tensor, value_scale: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor,
             row_offsets: torch.Tensor, rows: int, first: Optional[torch.Tensor] = None,
             seq_map: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None,
             value_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read tokens back: (key, value), each (rows, H, D) of the tails' dtype.

    Output rows ``row_offsets[i]`` .. ``row_offsets[i + 1] - 1`` are the tokens of slot
    ``seq_map[i]`` (without it i) from ``first[i]`` (without it 0) on.  Rows behind the
    last offset, and rows of tokens that the slot does not have, are left as they were
    (``key_out`` / ``value_out``: the caller's tensors, contiguous).
    """
    dev = _lib.require_cuda(lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v,
                            row_offsets, first, seq_map, key_out, value_out)
    a = _kv8.ReadArgs()
    _fill_cache(a.cache, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v)
    n = row_offsets.numel() - 1
    if n < 0 or rows < 0:
        raise RuntimeError("row_offsets must have n + 1 entries and rows must not be negative")
    row_offsets, first, seq_map = _index(row_offsets, "row_offsets", n + 1), _index(first, "first", n), _index(
        seq_map, "seq_map", n)
    shape = (rows, a.cache.num_heads, a.cache.head_dim)
    if key_out is None:
        key_out = torch.empty(shape, dtype=tail_k.dtype, device=dev)
    if value_out is None:
        value_out = torch.empty(shape, dtype=tail_k.dtype, device=dev)
    for t, name in ((key_out, "key_out"), (value_out, "value_out")):
        if t.shape != shape or t.dtype != tail_k.dtype or not t.is_contiguous():
            raise RuntimeError(f"{name} must be {shape} {tail_k.dtype}, contiguous")
    a.key, a.value, a.n, a.rows = key_out.data_ptr(), value_out.data_ptr(), n, rows
    a.row_offsets, a.first, a.seq_map = row_offsets.data_ptr(), _lib.ptr(first), _lib.ptr(seq_map)
    _kv8.launch(dev, "kitty_kv8_read", a)
    return key_out, value_out


def paged_attention_kv8(q: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, key_codes: torch.Tensor,
                        value_codes: torch.Tensor, key_scale: torch.Tensor, value_scale: torch.Tensor,
                        tail_k: torch.Tensor, tail_v: torch.Tensor, sm_scale: Optional[float] = None,
                        seq_map: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention: q (B, Hq, D) -> (B, Hq, D), both of the tails' dtype.

    Row b attends to all ``lengths[slot]`` tokens of slot ``seq_map[b]`` ((B,) int32;
    without it b), query head qh to KV head ``qh // (Hq // H)``; softmax and sums in
    float32, scores scaled by ``sm_scale`` (default 1 / sqrt(D)).  An empty slot gives
    zeros.  Two launches; the scratch they share is allocated for each call, so calls on
    several streams or in several graphs do not meet.
    """
    dev = _lib.require_cuda(q, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v,
                            seq_map, out)
    no_grad_inputs(q)
    a = _kv8.AttentionArgs()
    _fill_cache(a.cache, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v)
    h, d = a.cache.num_heads, a.cache.head_dim
    if q.dim() != 3 or q.shape[2] != d or q.dtype != tail_k.dtype:
        raise RuntimeError(f"q must be (B, Hq, {d}) {tail_k.dtype}")
    b, hq, _ = q.shape
    if hq == 0 or hq % h:
        raise RuntimeError("num_q_heads must be a multiple of num_kv_heads")
    seq_map = _index(seq_map, "seq_map", b)
    if out is None:
        out = torch.empty((b, hq, d), dtype=q.dtype, device=dev)
    a.out_s_seq, a.out_s_head = output_rows(out, q, "out")
    q, a.q_s_seq, a.q_s_head = aligned_rows(q)
    a.q, a.out, a.seq_map, a.batch, a.num_q_heads = q.data_ptr(), out.data_ptr(), _lib.ptr(seq_map), b, hq
    a.sm_scale = 1.0 / math.sqrt(d) if sm_scale is None else float(sm_scale)
    nbytes = _lib.c_size(0)
    _kv8.check(_kv8.load().kitty_kv8_attention_workspace_size(a, nbytes), "kitty_kv8_attention_workspace_size")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes.value
    _kv8.launch(dev, "kitty_kv8_attention", a)
    return out


def kv8_error_flags(device: Optional[torch.device] = None, clear: bool = True) -> int:
    """Sticky error bits that the 8-bit cache operators and :func:`qk_norm_rope` have set on
    a device since they were last cleared (``_kv8.ERRORS`` names them); synchronises."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return _kv8.error_flags(dev, clear=clear)
