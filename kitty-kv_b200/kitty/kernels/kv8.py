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

from typing import Optional, Tuple

import torch

from . import _kv8


def write_kv8(key: torch.Tensor, value: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor,
              key_codes: torch.Tensor, value_codes: torch.Tensor, key_scale: torch.Tensor,
              value_scale: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor,
              row_offsets: Optional[torch.Tensor] = None, seq_map: Optional[torch.Tensor] = None) -> None:
    """Append rows of key / value ((N, H, D), the tails' dtype) to n slots, in one launch.

    Entry i's rows are ``row_offsets[i]`` .. ``row_offsets[i + 1] - 1`` ((n + 1,) int32;
    without it every entry has one row); they go behind the ``lengths[slot]`` tokens that
    slot ``seq_map[i]`` has ((n,) int32, distinct; without it i; negative: padding,
    skipped).  Blocks that fill are quantised into the pages that ``block_table`` holds for
    them, the rest stays in the tail.  ``lengths`` is not changed: add the new tokens
    before the next call on this cache (torch's indexing takes no negative slot; of single rows
    ``lengths.index_add_(0, seq_map.clamp(min=0), (seq_map >= 0).to(torch.int32))`` is safe with
    padding).  Rows behind the last offset are ignored.
    The offsets of all entries, padding too, must not decrease.
    """
    _kv8.ops().write(key, value, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v,
                     row_offsets, seq_map)


def read_kv8(lengths: torch.Tensor, block_table: torch.Tensor, key_codes: torch.Tensor, value_codes: torch.Tensor,
             key_scale: torch.Tensor, value_scale: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor,
             row_offsets: torch.Tensor, rows: int, first: Optional[torch.Tensor] = None,
             seq_map: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None,
             value_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read tokens back: (key, value), each (rows, H, D) of the tails' dtype.

    Output rows ``row_offsets[i]`` .. ``row_offsets[i + 1] - 1`` are the tokens of slot
    ``seq_map[i]`` (without it i) from ``first[i]`` (without it 0) on.  Rows behind the
    last offset, of a negative slot, and of tokens that the slot does not have are left as they
    were (``key_out`` / ``value_out``: the caller's tensors, contiguous, not overlapping; undefined
    in tensors made here).  The offsets of all entries, padding too, must not decrease or pass
    ``rows``.
    """
    return _kv8.ops().read(lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v,
                           row_offsets, rows, first, seq_map, key_out, value_out)


def paged_attention_kv8(q: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, key_codes: torch.Tensor,
                        value_codes: torch.Tensor, key_scale: torch.Tensor, value_scale: torch.Tensor,
                        tail_k: torch.Tensor, tail_v: torch.Tensor, sm_scale: Optional[float] = None,
                        seq_map: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention: q (B, Hq, D) -> (B, Hq, D), both of the tails' dtype.

    Row b attends to all ``lengths[slot]`` tokens of slot ``seq_map[b]`` ((B,) int32;
    without it b), query head qh to KV head ``qh // (Hq // H)``; softmax and sums in
    float32, scores scaled by ``sm_scale`` (default 1 / sqrt(D)).  The weights that multiply the
    values are off by at most 2^-22 of themselves, or 2^-31 of the largest.  An empty slot gives
    zeros, and so does a negative one (a padded batch).  The same call gives the same bits;
    which tokens are summed together depends on the whole batch's lengths.  ``out`` may be q
    itself (same strides); any other overlap of the two is refused.  Two launches; the scratch they share is allocated for each call, so calls on
    several streams or in several graphs do not meet.
    """
    return _kv8.ops().attention(q, lengths, block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v,
                                sm_scale, seq_map, out)


def kv8_error_flags(device: Optional[torch.device] = None, clear: bool = True) -> int:
    """Sticky error bits that the 8-bit cache operators and :func:`qk_norm_rope` have set on
    a device since they were last cleared (``_kv8.ERRORS`` names them); synchronises."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return _kv8.error_flags(dev, clear=clear)
