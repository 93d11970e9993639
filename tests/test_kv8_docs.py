"""CPU test of what the documents tell a user of the 8-bit cache to run between its calls."""

from __future__ import annotations

import re
from pathlib import Path

import torch

from kitty import kernels as K

ROOT = Path(__file__).resolve().parent.parent


def test_documented_advance_of_lengths_takes_padding():
    """The lines of the integration document and of the docstring that add a step's tokens to the
    lengths, with padded slots."""
    texts = [p.read_text() for p in ROOT.glob("INTEGR*")] + [K.write_kv8.__doc__]
    lines = [x for t in texts for x in re.findall(r"lengths\.index_add_\(.*\)", t)]
    assert len(lines) >= 2
    for line in lines:
        slots = torch.tensor([2, -1, 0, -5], dtype=torch.int32)
        lengths = torch.tensor([7, 8, 9], dtype=torch.int32)
        exec(line, {"torch": torch, "lengths": lengths, "slots": slots, "seq_map": slots,
                    "ones": torch.ones(4, dtype=torch.int32)})
        assert lengths.tolist() == [8, 8, 10], line
