"""Kitty quantisation / decode kernels - B200 (sm_100a) CUDA implementations.

Same names as the reference's ``kitty/kernels/__init__.py:19-29`` plus the
batched forms, and the operators of the 8-bit paged cache (``kv8``) and of the
rotary embedding (``rope``).  All of them run the hand-written CUDA kernels of
``libkitty_b200.so`` / ``libkitty_kv8.so`` on CUDA tensors; there is no Triton and no
CPU fallback (CPU tensors raise ``RuntimeError``).  Each library is loaded on first use.
"""

from .quantize_key import quantize_key_page, quantize_key_page_torch, quantize_key_pages
from .dequantize_key import dequantize_key_page, dequantize_key_page_torch
from .quantize_value import (
    quantize_value_page,
    quantize_value_page_torch,
    quantize_value_pages,
    dequantize_value_page_torch,
)
from .attention import paged_attention, paged_attention_reference, paged_attention_batched
from .rope import qk_norm_rope, rope_table
from .kv8 import kv8_error_flags, paged_attention_kv8, read_kv8, write_kv8

__all__ = [
    "quantize_key_page",
    "quantize_key_page_torch",
    "dequantize_key_page",
    "dequantize_key_page_torch",
    "quantize_value_page",
    "quantize_value_page_torch",
    "dequantize_value_page_torch",
    "paged_attention",
    "paged_attention_reference",
    # batched extensions
    "quantize_key_pages",
    "quantize_value_pages",
    "paged_attention_batched",
    # norm and rotation of queries and keys, and the 8-bit paged cache
    "qk_norm_rope",
    "rope_table",
    "write_kv8",
    "read_kv8",
    "paged_attention_kv8",
    "kv8_error_flags",
]
