"""GPU tests of the 8-bit cache's attention at the limits of its inputs: pages that are none
beside pages of NaN, NaN in one tile of many, the largest values, and how exactly the weights
are held."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from kv8_model import CacheModel, attention
from test_gpu_kv8 import BF16, E4M3, FP16, INT8, filled, i32

pytestmark = pytest.mark.gpu


def bound(out, absum, mass, dtype):
    """Bound of |kernel - exact| with weights held in 22 bits or more: a score is off by at most 64
    roundings of 2^-23 of its sum of magnitudes, a weight by that, the exponential's 2^-20 and the
    2^-22 that two fp16 parts leave of it; that counts in numerator and denominator; the output is
    rounded once, half a step or half the smallest subnormal."""
    w = 64 * 2.0 ** -23 * mass + 2.0 ** -20 + 2.0 ** -22
    return torch.finfo(dtype).eps / 2 * out.abs() + 2 * w * absum * (1 + torch.finfo(dtype).eps) + 2.0 ** -25


def check(m, q, got, slot, i, keep=None):
    k, v = m.truth(slot)
    if keep is not None:
        k, v = k[:, keep], v[:, keep]
    want, absum, mass = attention(q[i].cpu(), k, v)
    err = (got[i].cpu().double() - want).abs()
    assert (err <= bound(want, absum, mass, m.dtype)).all(), f"row {i}: {(err / bound(want, absum, mass, m.dtype)).max():.2f}"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 128), (1, 256)])
@pytest.mark.parametrize("lens", [[96, 200], [4000, 5000]])
def test_a_missing_page_does_not_let_page_0_in(dtype, heads, dim, lens):
    """Page 0 is another sequence's, and holds NaN codes and scales; a block whose table entry is no
    page is left out and flagged, and the rest of its sequence comes out."""
    m = CacheModel(3, heads, dim, 32, E4M3, dtype, pages=2 + sum(n // 32 for n in lens), table_width=200, seed=dim)
    m.free.remove(0)
    m.free.append(0)                                      # slot 2's block
    bad = m.new_rows(32)
    bad[5, :, 3], bad[6, :, 9] = float("nan"), float("inf")
    m.append(2, bad, bad)
    for s, n in enumerate(lens):
        m.append(s, m.new_rows(n), m.new_rows(n))
    m.fill_arrays()
    q = torch.randn(3, 4 * heads, dim, generator=m.g).to(dtype).cuda()
    table = m.table.clone()
    table[0, 1], table[1, 0], table[1, 4] = -1, 10 ** 6, m.key_scale.shape[0]
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays(table))
    assert K.kv8_error_flags() == 1 << 1
    assert got[2].isnan().all()
    check(m, q, got, 0, 0, [t for t in range(lens[0]) if t // 32 != 1])
    check(m, q, got, 1, 1, [t for t in range(lens[1]) if t // 32 not in (0, 4)])


@pytest.mark.parametrize("code,dtype", [(E4M3, BF16), (E4M3, FP16), (INT8, BF16)])
@pytest.mark.parametrize("group", [4, 16])
def test_nan_in_one_key_tile_or_tail_row(code, dtype, group):
    """NaN scores reach the output of their own sequence and head group, and no other."""
    lens = [3000, 3000, 3010, 1]
    m = filled(lens, 2, 128, 64, code, dtype, seed=group)
    table = m.table
    m.key_scale[int(table[0, 20]), 1] = float("nan")       # one page in the middle, KV head 1
    m.tail_k[2, 0, 1, 7] = float("nan")                  # the second of the tail's two rows, KV head 0
    q = torch.randn(4, 2 * group, 128, generator=m.g).to(dtype).cuda()
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays())
    bad = torch.zeros(4, 2 * group, 128, dtype=torch.bool)
    bad[0, group:], bad[2, :group] = True, True
    assert torch.equal(got.isnan().cpu(), bad)
    for i in (1, 3):
        check(m, q, got, i, i)
    assert K.kv8_error_flags() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("lens", [[5, 32, 61], [300, 96, 40], [9000, 3, 64]])
def test_the_largest_values(code, lens):
    """bf16 values up to 2^128 / tokens: every partial sum of weights of at most one fits float32, so
    the outputs are finite, and right."""
    m = CacheModel(3, 1, 64, 32, code, BF16, pages=sum(lens) // 32 + 3, table_width=300, seed=sum(lens))
    for s, n in enumerate(lens):
        top = 2.0 ** 127 / n
        v = (torch.rand(n, 1, 64, generator=m.g) * 2 - 1) * 0.99 * top
        v[n // 2, 0, 0] = top * 0.99
        m.append(s, (m.new_rows(n) * torch.linspace(0.2, 1, n)[:, None, None]).to(BF16), v.to(BF16))
    m.fill_arrays()
    q = torch.randn(3, 4, 64, generator=m.g).to(BF16).cuda()
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays())
    assert torch.isfinite(got).all()
    for i in range(3):
        check(m, q, got, i, i)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (1, 16, 128), (2, 8, 64), (1, 3, 256), (1, 5, 80)])
def test_weights_are_held_in_22_bits(code, dtype, heads, group, dim):
    """Values of both signs nearly cancel, small queries make the weights alike: what is left shows
    how far the weights are off, in pages and in the tail."""
    lens = [32, 31, 64, 40, 2000]
    m = CacheModel(len(lens), heads, dim, 32, code, dtype, pages=100, table_width=64, seed=dim + group)
    for s, n in enumerate(lens):
        v = m.new_rows(n)
        v[1::2] = -v[:n // 2 * 2:2]
        m.append(s, m.new_rows(n, 0.1), v)
    m.fill_arrays()
    q = (0.05 * torch.randn(len(lens), heads * group, dim, generator=m.g)).to(dtype).cuda()
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays())
    for i in range(len(lens)):
        check(m, q, got, i, i)
