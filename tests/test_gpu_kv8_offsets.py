"""GPU tests of row offsets that are out of order or range, in reads and writes: always flagged,
padding entries included, and what the other entries ask for is done."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from kv8_model import CacheModel
from kv8_model import CacheModel
from test_gpu_kv8 import E4M3, FP16, INT8, check_cache, filled, i32

pytestmark = pytest.mark.gpu
ROWS = 1 << 2


def read(m, offsets, rows, slots=None):
    k = torch.full((rows, m.h, m.d), 9.0, dtype=m.dtype, device="cuda")
    K.read_kv8(m.lens(), *m.arrays(), i32(offsets), rows, seq_map=None if slots is None else i32(slots), key_out=k)
    return K.kv8_error_flags(), k.cpu()


def truth(m, slot, a, b):
    return m.truth(slot)[0][:, a:b].transpose(0, 1).float().to(m.dtype)


@pytest.mark.parametrize("heads", [1, 5])
def test_read_offsets(heads):
    m = filled([100, 70, 33], heads, 64, 32, INT8, FP16, seed=1)
    flags, k = read(m, [0, 40, 60], 45, [0, 1])           # the last entry's rows pass the call's
    assert flags == ROWS
    assert torch.equal(k, torch.cat([truth(m, 0, 0, 40), truth(m, 1, 0, 5)]))
    flags, k = read(m, [0, 45, 45, 46], 45)               # and one that begins behind them
    assert flags == ROWS and torch.equal(k, truth(m, 0, 0, 45))
    flags, k = read(m, [0, 30, 10, 10], 40)
    assert flags == ROWS
    flags, k = read(m, [-5, 30, 30, 30], 40)
    assert flags == ROWS and (k == 9).all()
    flags, k = read(m, [0, 33, 0, 0], 33, [2, -1, -1])    # padding has offsets too
    assert flags == ROWS
    flags, k = read(m, [0, 33, 33, 33], 33, [2, -1, -1])
    assert flags == 0 and torch.equal(k, truth(m, 2, 0, 33))
    flags, k = read(m, [0, 33, 33, 40], 41, [2, -1, -1])
    assert flags == 0 and torch.equal(k[:33], truth(m, 2, 0, 33)) and (k[33:] == 9).all()


@pytest.mark.parametrize("n", [31, 32, 33, 64, 700])
def test_read_offsets_of_many_entries(n):
    """One fault in many entries, before, at and behind a warp's window of them."""
    m = filled([100, 70], 1, 64, 32, E4M3, FP16, seed=n)
    good = [3 * i for i in range(n + 1)]
    slots = [i % 2 for i in range(n)]
    want = torch.cat([truth(m, i % 2, 0, 3) for i in range(n)])
    flags, k = read(m, good, 3 * n, slots)
    assert flags == 0 and torch.equal(k, want)
    for at in {0, 1, n // 2, n - 2, n - 1}:
        bad = list(good)
        bad[at + 1] = bad[at] - 1                         # entry `at` ends before it begins
        flags, k = read(m, bad, 3 * n, slots)
        assert flags & ROWS, at
        bad = list(good)
        bad[-1] = 3 * n + 1
        flags, k = read(m, bad, 3 * n, slots)
        assert flags == ROWS and torch.equal(k, want)


def test_write_offsets_of_padding_entries():
    """A write looks rows up by all entries' offsets, so those of padding have to follow one another
    too: flagged where they do not, and padding that keeps the order is skipped silently."""
    def fresh():
        m = CacheModel(3, 2, 64, 32, E4M3, FP16, pages=8, table_width=4, seed=2)
        return m, m.new_rows(69), m.new_rows(69)

    for offsets, slots in (([0, 5, 69, 0, 0], [0, 2, -1, -1]), ([0, 5, 69, 69, 70], [0, 2, -1, -1]),
                           ([-1, 0, 5, 69, 69], [-1, 0, 2, -1])):
        m, k, v = fresh()
        table = torch.arange(12, dtype=torch.int32).view(3, 4) % 8
        K.write_kv8(k.cuda(), v.cuda(), m.lens(), *m.arrays(table), row_offsets=i32(offsets), seq_map=i32(slots))
        assert K.kv8_error_flags() == ROWS, offsets
    m, k, v = fresh()
    before = m.lens()
    m.append(0, k[:5], v[:5])
    m.append(2, k[5:65], v[5:65])
    K.write_kv8(k.cuda(), v.cuda(), before, *m.arrays(), row_offsets=i32([0, 5, 65, 69, 69]), seq_map=i32([0, 2, -1, -9]))
    assert K.kv8_error_flags() == 0
    check_cache(m)
