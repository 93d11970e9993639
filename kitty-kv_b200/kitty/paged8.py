"""PagedKVCache8 - the KV cache of many sequences in 8-bit codes.

For the layers of a model that do not stand the 2 bits of :class:`kitty.BatchedKVCache`
(about half the bytes of a 16-bit cache, 3.5 times those of a 2-bit one).  Keys and
values become e4m3 or int8 codes with one float32 scale for each block of ``page_size``
tokens and KV head; a block is quantised when its last token arrives and stays in
16 bits until then.  There are no sinks and no boosted channels.

Lengths and pages are kept on the host, which knows both without asking the device:
what does not fit raises ``RuntimeError`` before anything is changed.  Each call sends
its few integers in one copy and launches on the current stream; appending cannot be
captured in a CUDA graph, but the operators that it uses can
(``kitty.kernels.write_kv8``, ``paged_attention_kv8``), and so can :meth:`decode` with
``seq_ids`` in device memory.
"""

from __future__ import annotations

import heapq
from typing import List, Optional, Sequence, Tuple

import torch

from .config import KittyConfig
from .kernels import _kv8
from .kernels.kv8 import kv8_error_flags, paged_attention_kv8, read_kv8, write_kv8
from .layout import torch_dtype

CODE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class PagedKVCache8:
    """8-bit cache of ``max_seqs`` slots x ``config.num_layers`` layers.

    From ``config`` it takes num_layers, num_kv_heads, head_dim, dtype (the 16-bit type),
    max_seq_len and device.  page_size: tokens per block (a multiple of 32, at most 256).
    codes: "e4m3" or "int8".  num_pages: pool size shared by all layers (default: every
    slot can reach ``config.max_seq_len`` tokens in every layer).
    """

    def __init__(self, config: KittyConfig, max_seqs: int, num_pages: Optional[int] = None, page_size: int = 64,
                 codes: str = "e4m3", max_pages_per_seq: Optional[int] = None,
                 device: Optional[torch.device] = None) -> None:
        if codes not in CODE_DTYPES:
            raise RuntimeError(f"codes must be one of {sorted(CODE_DTYPES)}, got {codes!r}")
        if page_size <= 0 or page_size % 32 or page_size > 256:
            raise RuntimeError("page_size must be a multiple of 32 and at most 256")
        L, H, D = config.num_layers, config.num_kv_heads, config.head_dim
        if D % 16 or D > 256:
            raise RuntimeError("the 8-bit cache takes head_dim as a multiple of 16, at most 256")
        dev = torch.device(device if device is not None else config.device)
        if dev.type != "cuda":
            raise RuntimeError("PagedKVCache8 lives in CUDA memory (there is no CPU path)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.config, self.device, self.dtype = config, dev, torch_dtype(config.dtype)
        self.max_seqs, self.page_size = int(max_seqs), int(page_size)
        self.max_pages_per_seq = -(-config.max_seq_len // page_size) if max_pages_per_seq is None else int(
            max_pages_per_seq)
        self.num_pages = max_seqs * self.max_pages_per_seq * L if num_pages is None else int(num_pages)
        P, B, M, G = self.num_pages, self.max_seqs, self.max_pages_per_seq, self.page_size
        code = CODE_DTYPES[codes]
        self.key_codes = torch.zeros(P, H, G, D, dtype=torch.int8, device=dev).view(code)
        self.value_codes = torch.zeros(P, H, G, D, dtype=torch.int8, device=dev).view(code)
        self.key_scale = torch.zeros(P, H, dtype=torch.float32, device=dev)
        self.value_scale = torch.zeros(P, H, dtype=torch.float32, device=dev)
        self.tail_k = torch.zeros(L, B, H, G, D, dtype=self.dtype, device=dev)
        self.tail_v = torch.zeros(L, B, H, G, D, dtype=self.dtype, device=dev)
        self.block_table = torch.full((L, B, M), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(L, B, dtype=torch.int32, device=dev)
        self.reset()

    # ------------------------------------------------------------------ helpers

    def arrays(self, layer_id: int) -> Tuple[torch.Tensor, ...]:
        """The arrays of one layer in the order that ``kitty.kernels`` takes them behind the
        lengths: block_table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v."""
        return (self.block_table[layer_id], self.key_codes, self.value_codes, self.key_scale, self.value_scale,
                self.tail_k[layer_id], self.tail_v[layer_id])

    def _slots(self, seq_ids: Sequence[int], distinct: bool = True) -> List[int]:
        ids = [int(s) for s in (seq_ids.tolist() if isinstance(seq_ids, torch.Tensor) else seq_ids)]
        if any(s < 0 or s >= self.max_seqs for s in ids):
            raise RuntimeError(f"sequence ids must be in [0, {self.max_seqs})")
        if distinct and len(set(ids)) != len(ids):
            raise RuntimeError("a sequence id is given twice")
        return ids

    def _send(self, *lists: List[int]) -> List[torch.Tensor]:
        """int32 device tensors of host lists, by one copy."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("this call keeps host state and cannot be captured in a CUDA graph; "
                               "capture kitty.kernels.write_kv8 / paged_attention_kv8 instead")
        host = torch.tensor([x for part in lists for x in part], dtype=torch.int32)
        both = (host.pin_memory() if host.numel() else host).to(self.device, non_blocking=True)
        return list(both.split([len(part) for part in lists]))

    def _extend(self, layer_id: int, ids: List[int], counts: Optional[List[int]], key: torch.Tensor,
                value: torch.Tensor) -> None:
        rows = len(ids) if counts is None else sum(counts)
        H, D = self.config.num_kv_heads, self.config.head_dim
        for t, name in ((key, "key"), (value, "value")):
            if t.dtype != self.dtype or t.device != self.device or tuple(t.shape) != (rows, H, D):
                raise RuntimeError(f"{name} must be ({rows}, {H}, {D}) {self.dtype} on {self.device}")
        lens, G = self._lens[layer_id], self.page_size
        new = [1] * len(ids) if counts is None else counts
        need = [(lens[s] + n) // G - lens[s] // G for s, n in zip(ids, new)]
        for s, n in zip(ids, new):
            if (lens[s] + n) // G > self.max_pages_per_seq:
                raise RuntimeError(f"sequence {s} would pass its {self.max_pages_per_seq} pages of {G} tokens")
        if sum(need) > len(self._free):
            raise RuntimeError(f"KV cache page pool exhausted: {sum(need)} pages wanted, {len(self._free)} free")
        taken = [heapq.heappop(self._free) for _ in range(sum(need))]
        slots_of = [s for s, n in zip(ids, need) for _ in range(n)]
        blocks = [lens[s] // G + k for s, n in zip(ids, need) for k in range(n)]
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        try:
            d_ids, d_offsets, d_lens, d_slots, d_blocks, d_pages = self._send(
                ids, offsets, [lens[s] + n for s, n in zip(ids, new)], slots_of, blocks, taken)
            if taken:
                self.block_table[layer_id].index_put_((d_slots.long(), d_blocks.long()), d_pages)
            write_kv8(key, value, self.seq_lens[layer_id], *self.arrays(layer_id),
                      row_offsets=None if counts is None else d_offsets, seq_map=d_ids)
        except Exception:
            for p in taken:
                heapq.heappush(self._free, p)
            raise
        self.seq_lens[layer_id].index_copy_(0, d_ids.long(), d_lens)
        for s, n in zip(ids, new):
            lens[s] += n
        for s, p in zip(slots_of, taken):
            self._pages[layer_id][s].append(p)

    # ------------------------------------------------------------------ API

    def reset(self) -> None:
        """Empty every slot of every layer; all pages free."""
        L, B = self.config.num_layers, self.max_seqs
        self._lens = [[0] * B for _ in range(L)]
        self._pages: List[List[List[int]]] = [[[] for _ in range(B)] for _ in range(L)]
        self._free = list(range(self.num_pages))
        self.seq_lens.zero_()

    def append(self, layer_id: int, seq_ids, key: torch.Tensor, value: torch.Tensor) -> None:
        """Append token row i of key / value ((n, H, D), the cache's dtype) to slot seq_ids[i]
        (distinct) of ``layer_id``."""
        self._extend(layer_id, self._slots(seq_ids), None, key, value)

    def prefill(self, layer_id: int, seq_ids, key: torch.Tensor, value: torch.Tensor, lengths) -> None:
        """Append lengths[i] tokens to slot seq_ids[i] (distinct) of ``layer_id``: the next
        lengths[i] rows of key / value ((sum(lengths), H, D), sequences one after another).
        The same as appending them one at a time, and as any split into several calls."""
        ids = self._slots(seq_ids)
        counts = [int(x) for x in (lengths.tolist() if isinstance(lengths, torch.Tensor) else lengths)]
        if len(counts) != len(ids) or min(counts, default=0) < 0:
            raise RuntimeError("lengths must hold one non-negative count per sequence id")
        self._extend(layer_id, ids, counts, key, value)

    def decode(self, layer_id: int, q: torch.Tensor, seq_ids, out: Optional[torch.Tensor] = None,
               sm_scale: Optional[float] = None) -> torch.Tensor:
        """Decode attention of row i of q ((n, Hq, D), the cache's dtype) over slot seq_ids[i] (host
        integers, or an int32 tensor in device memory); output of q's dtype."""
        if isinstance(seq_ids, torch.Tensor) and seq_ids.is_cuda:
            ids = seq_ids
        else:
            ids, = self._send(self._slots(seq_ids, distinct=False))
        return paged_attention_kv8(q, self.seq_lens[layer_id], *self.arrays(layer_id), sm_scale=sm_scale, seq_map=ids,
                                   out=out)

    def read(self, layer_id: int, seq_ids) -> Tuple[torch.Tensor, torch.Tensor, List[int]]:
        """All tokens of the given slots as 16-bit rows, one sequence after another: key and
        value ((sum, H, D)) and the lengths."""
        ids = self._slots(seq_ids, distinct=False)
        lens = [self._lens[layer_id][s] for s in ids]
        offsets = [0]
        for n in lens:
            offsets.append(offsets[-1] + n)
        d_ids, d_offsets = self._send(ids, offsets)
        key, value = read_kv8(self.seq_lens[layer_id], *self.arrays(layer_id), d_offsets, offsets[-1], seq_map=d_ids)
        return key, value, lens

    def release(self, seq_ids) -> None:
        """Empty the given slots in every layer; their pages become free."""
        ids = self._slots(seq_ids)
        if not ids:
            return
        d_ids, = self._send(ids)
        self.seq_lens.index_fill_(1, d_ids.long(), 0)
        for l in range(self.config.num_layers):
            for s in ids:
                for p in self._pages[l][s]:
                    heapq.heappush(self._free, p)
                self._pages[l][s] = []
                self._lens[l][s] = 0

    # ------------------------------------------------------------------ inspection

    def free_page_count(self) -> int:
        return len(self._free)

    def lengths(self, layer_id: int) -> List[int]:
        """Tokens of each slot of one layer."""
        return list(self._lens[layer_id])

    def check_errors(self, clear: bool = True) -> None:
        """Raise if a call on this device has met bad device data since the last check
        (synchronises); the cache's own calls give none."""
        bits = kv8_error_flags(self.device, clear=clear)
        msgs = [m for b, m in _kv8.ERRORS.items() if bits & b]
        if msgs:
            raise RuntimeError("8-bit KV cache: " + "; ".join(msgs))
