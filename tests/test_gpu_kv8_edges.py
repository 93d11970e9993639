"""GPU tests of the 8-bit cache operators where callers go past the ordinary: padded
batches, caches without pages, tables with strided rows, scores far outside the usual,
overlapping streams, a first call inside a capture."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kitty import kernels as K
from kv8_model import CacheModel
from test_gpu_kv8 import BF16, E4M3, FP16, INT8, check_attention, check_cache, filled, i32, write

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def test_padded_batches():
    """Negative slots: nothing written, read rows left, zeros attended, no error."""
    m = CacheModel(3, 2, 64, 32, E4M3, BF16, pages=12, table_width=4, seed=1)
    write(m, range(3), [31, 40, 5])
    k, v = m.new_rows(5), m.new_rows(5)
    before = m.lens()
    slots = [2, -1, 0, -1, -5]
    for i in (0, 2):
        m.append(slots[i], k[i:i + 1], v[i:i + 1])
    K.write_kv8(k.cuda(), v.cuda(), before, *m.arrays(), seq_map=i32(slots))
    check_cache(m)
    before = m.lens()
    for s, a, b in ((1, 0, 2), (0, 3, 5)):
        m.append(s, k[a:b], v[a:b])
    K.write_kv8(k.cuda(), v.cuda(), before, *m.arrays(), row_offsets=i32([0, 2, 3, 5]), seq_map=i32([1, -1, 0]))
    check_cache(m)
    ko = torch.full((9, 2, 64), 3.0, dtype=BF16, device="cuda")
    K.read_kv8(m.lens(), *m.arrays(), i32([0, 4, 9]), 9, seq_map=i32([-1, 2]), key_out=ko)
    assert (ko[:4] == 3).all() and torch.equal(ko[4:].cpu(), m.truth(2)[0][:, :5].transpose(0, 1).to(BF16))
    q = torch.randn(4, 4, 64, generator=m.g).to(BF16).cuda()
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays(), seq_map=i32([1, -1, 0, -7]))
    assert not got[[1, 3]].any()
    check_attention(m, 4, rows=[1, 0], q=q[[0, 2]], got=got[[0, 2]])
    assert K.kv8_error_flags() == 0


def test_cache_without_pages_and_table_with_strided_rows():
    m = CacheModel(2, 1, 64, 64, INT8, FP16, pages=0, table_width=0, seed=2)
    write(m, range(2), [63, 7])
    check_cache(m)
    check_attention(m, 3)
    k, _ = K.read_kv8(m.lens(), *m.arrays(), i32([0, 63, 70]), 70)
    assert torch.equal(k[:63].cpu(), m.truth(0)[0].transpose(0, 1).to(FP16))
    assert K.kv8_error_flags() == 0
    m = filled([100, 70], 1, 64, 32, INT8, FP16, seed=3)
    wide = torch.full((2, 3 * m.table.shape[1]), -9, dtype=torch.int32, device="cuda")
    wide[:, :m.table.shape[1]] = m.table.cuda()
    q = torch.randn(2, 3, 64, generator=m.g).to(FP16).cuda()
    got = K.paged_attention_kv8(q, m.lens(), wide[:, :m.table.shape[1]], *m.arrays()[1:])
    check_attention(m, 3, q=q, got=got)


def test_an_empty_pool_has_tails_only():
    """Lengths that ask for pages of a pool that has none: flagged, no tokens, no page touched."""
    m = CacheModel(3, 1, 64, 32, E4M3, BF16, pages=0, table_width=2, seed=12)
    m.append(0, m.new_rows(9), m.new_rows(9))
    m.fill_arrays()
    lens = m.lens()
    lens[1], lens[2] = 40, 64
    q = torch.randn(3, 2, 64, generator=m.g).to(BF16).cuda()
    got = K.paged_attention_kv8(q, lens, *m.arrays())
    assert K.kv8_error_flags() == 1 << 4 and not got[1:].any()
    check_attention(m, 2, rows=[0], q=q[:1], got=got[:1])
    k = torch.full((40, 1, 64), 3.0, dtype=BF16, device="cuda")
    K.read_kv8(lens, *m.arrays(), i32([0, 0, 40, 40]), 40, key_out=k)
    assert K.kv8_error_flags() == 1 << 1 and (k[:32] == 3).all() and not (k[32:] == 3).any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scores_far_from_zero(code, dtype):
    """Scores of 10^4 to 10^9, where only the largest counts: its value comes out, whatever the
    rounding of the products, and no overflow makes a NaN."""
    m = filled([70, 200, 33], 1, 64, 32, code, dtype, seed=4, scale=50.0)
    for scale in (1e3, 1e6, 1e8, -1e6):
        q = torch.randn(3, 4, 64, generator=m.g).to(dtype).cuda()
        got = K.paged_attention_kv8(q, m.lens(), *m.arrays(), sm_scale=scale)
        for s in range(3):
            k, v = m.truth(s)
            scores = q[s].cpu().double() @ k[0].T * scale
            two = scores.topk(2, -1)
            for h in range(4):
                gap = two.values[h, 0] - two.values[h, 1]
                # float32 sums are off by 2^-17 of the magnitudes; below that and 30 the winner is open
                if gap > 30 + 2.0 ** -16 * (q[s, h].cpu().double().abs() @ k[0].T.abs()).max() * abs(scale):
                    want = v[0, two.indices[h, 0]]
                    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -11 * want.abs() + 1e-12 * v.abs().max() + 2.0 ** -25
                    assert ((got[s, h].cpu().double() - want).abs() <= tol).all(), (scale, s, h)
        assert torch.isfinite(got).all()


def test_rising_and_falling_scores():
    """Keys ordered so that the reference moves again and again, or only once."""
    m = CacheModel(2, 1, 64, 32, E4M3, FP16, pages=64, table_width=40, seed=5)
    n = 900
    d = torch.randn(64, generator=m.g)
    d /= d.norm()
    ramp = torch.linspace(-60, 60, n)
    for s, r in ((0, ramp), (1, ramp.flip(0))):
        m.append(s, (r[:, None, None] * d + 0.1 * torch.randn(n, 1, 64, generator=m.g)).to(FP16), m.new_rows(n))
    m.fill_arrays()
    q = (8 * d + 0.05 * torch.randn(2, 5, 64, generator=m.g)).to(FP16).cuda()
    check_attention(m, 5, q=q, sm_scale=0.5)
    check_attention(m, 5, q=q, sm_scale=0.02)


@pytest.mark.parametrize("batch", [1, 31, 32, 33, 128, 129, 600])
def test_batches_around_the_scan_sizes(batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 80, (batch,), generator=g).tolist()
    lens[batch // 2] = 300
    m = filled(lens, 1, 64, 32, INT8, BF16, seed=batch)
    check_attention(m, 2)
    assert K.kv8_error_flags() == 0


@pytest.mark.parametrize("batch", [64, 65, 255, 256, 257])
def test_batches_around_the_scan_sizes_mapped_and_with_faults(batch):
    """Slots in another order, some twice, some empty, padded, out of range or of a wrong length."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 200, (90,), generator=g).tolist()
    lens[7], lens[8], lens[9] = 1500, 0, 70
    m = filled(lens, 2, 64, 96, E4M3, FP16, seed=batch)
    rows = torch.randint(0, 90, (batch,), generator=g).tolist()
    rows[3], rows[5], rows[-1], rows[batch // 2], rows[batch // 2 + 1] = 7, 8, 7, -3, 90
    n = m.lens()
    n[9], n[10] = -4, 2 ** 31 - 1
    q = torch.randn(batch, 6, 64, generator=m.g).to(FP16).cuda()
    got = K.paged_attention_kv8(q, n, *m.arrays(), seq_map=i32(rows))
    none = torch.tensor([s < 0 or s in (8, 9, 10, 90) for s in rows])
    assert not got[none.cuda()].any()
    some = [i for i in range(batch) if not none[i]]
    check_attention(m, 6, rows=[rows[i] for i in some], q=q[some], got=got[some])
    flags = (1 << 3) | ((1 << 4) if 9 in rows or 10 in rows else 0)
    assert K.kv8_error_flags() == flags


@pytest.mark.parametrize("code,dtype", [(E4M3, FP16), (INT8, BF16)])
@pytest.mark.parametrize("heads,dim,page,rows", [(8, 64, 32, 6000), (5, 64, 32, 6000), (3, 64, 64, 13000), (2, 64, 32, 10000),
                                                 (8, 128, 32, 4000), (3, 128, 32, 7000), (16, 16, 32, 6000),
                                                 (7, 80, 32, 4000), (9, 48, 64, 5000), (1, 64, 32, 20000)])
def test_large_writes_of_small_blocks(code, dtype, heads, dim, page, rows):
    """Enough rows that a CTA quantises several heads: rows of a fused projection, slots that have
    begun a block, NaN and infinities in some heads' blocks, and pages that are none."""
    n = 20
    m = CacheModel(n, heads, dim, page, code, dtype, pages=rows // page + 3 * n, table_width=rows // page, seed=dim + rows)
    write(m, range(n), [i * 7 % page for i in range(n)])
    g = torch.Generator().manual_seed(rows)
    counts = torch.distributions.Multinomial(rows, torch.rand(n, generator=g)).sample().int().tolist()
    counts[4] = 0
    both = torch.cat([m.new_rows(sum(counts)), m.new_rows(sum(counts))], 1)
    both[40, 0, 3], both[900, heads - 1, 2], both[1700, heads, 5] = float("nan"), float("inf"), float("nan")
    both[2000:2200] = 0
    before, offsets = m.lens(), [0]
    for s, c in enumerate(counts):
        m.append(s, *both[offsets[-1]:offsets[-1] + c].split(heads, 1))
        offsets.append(offsets[-1] + c)
    table = m.table.clone()
    lost = [s for s in range(n) if m.lengths[s] // page > 3][:2]
    for s in lost:
        table[s, 2] = 10 ** 6 if s == lost[0] else -1
    key, value = both.cuda().split(heads, 1)
    tails = m.tail_k.clone(), m.tail_v.clone()               # a write takes the rows of a begun block from them
    K.write_kv8(key, value, before, *m.arrays(table), row_offsets=i32(offsets))
    assert K.kv8_error_flags() == (1 << 1 if lost else 0)
    spare = m.table[lost, 2].long().cuda()
    for t in (m.key_codes, m.value_codes):
        assert not t.view(torch.uint8)[spare].any()          # nothing went to the pages that were not named
    m.tail_k.copy_(tails[0]), m.tail_v.copy_(tails[1])
    K.write_kv8(key, value, before, *m.arrays(), row_offsets=i32(offsets))
    assert K.kv8_error_flags() == 0
    check_cache(m)


def test_all_slots_empty():
    m = CacheModel(40, 2, 128, 64, E4M3, BF16, pages=1, table_width=1, seed=6, fill=float("nan"))
    for b in (1, 40):
        q = torch.randn(b, 8, 128, device="cuda").to(BF16)
        assert not K.paged_attention_kv8(q, m.lens(), *m.arrays(), seq_map=i32(list(range(b)))).any()


def test_the_same_call_gives_the_same_bits():
    m = filled([3000, 0, 77, 640], 2, 128, 64, E4M3, FP16, seed=7)
    q = torch.randn(4, 8, 128, generator=m.g).to(FP16).cuda()
    outs = [K.paged_attention_kv8(q, m.lens(), *m.arrays()) for _ in range(5)]
    assert all(torch.equal(outs[0], o) for o in outs)


def test_overlapping_calls_on_several_streams():
    """Calls in flight on four streams at once, each with its own scratch."""
    caches = [filled([2000 + 100 * i, 50, 700], 2, 128, 64, E4M3, BF16, seed=30 + i) for i in range(4)]
    qs = [torch.randn(3, 8, 128, generator=m.g).to(BF16).cuda() for m in caches]
    args = [(q, m.lens(), *m.arrays()) for q, m in zip(qs, caches)]
    want = [K.paged_attention_kv8(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[] for _ in caches]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.paged_attention_kv8(*args[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_output_in_the_place_of_the_queries():
    """Rows whose segments are stored by one warp, and rows joined from many parts."""
    for lens, hq in (([9000, 5, 0], 8), ([9000, 5, 0], 40), ([40 + i for i in range(200)], 4)):
        m = filled(lens, 2, 64, 32, E4M3, BF16, seed=len(lens) + hq)
        q = torch.randn(len(lens), hq, 64, generator=m.g).to(BF16).cuda()
        want = K.paged_attention_kv8(q, m.lens(), *m.arrays())
        assert K.paged_attention_kv8(q, m.lens(), *m.arrays(), out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("n", [1, 30, 31, 32, 33, 63, 64, 65, 500])
@pytest.mark.parametrize("heads", [1, 8])
def test_read_of_many_entries_most_of_them_empty(n, heads):
    """Runs of entries without rows, longer than a warp, between and behind entries with some."""
    m = filled([70, 33, 64], heads, 64, 32, INT8, FP16, seed=n)
    g = torch.Generator().manual_seed(n)
    counts = torch.where(torch.rand(n, generator=g) < 0.1, torch.randint(1, 30, (n,), generator=g), 0)
    counts[-1] = 3
    slots, first = torch.randint(0, 3, (n,), generator=g), torch.randint(0, 4, (n,), generator=g)
    offsets = [2] + (counts.cumsum(0) + 2).tolist()
    rows = offsets[-1] + 2
    ko = torch.full((rows, heads, 64), 9.0, dtype=FP16, device="cuda")
    k, v = K.read_kv8(m.lens(), *m.arrays(), i32(offsets), rows, first=i32(first.tolist()), seq_map=i32(slots.tolist()),
                      key_out=ko)
    want = [[torch.full((2, heads, 64), 9.0, dtype=FP16)], []]
    for x in range(2):
        for c, s, f in zip(counts.tolist(), slots.tolist(), first.tolist()):
            want[x].append(m.truth(s)[x][:, f:f + c].transpose(0, 1).float().to(FP16))
    want[0].append(want[0][0])
    assert torch.equal(k.cpu(), torch.cat(want[0])) and torch.equal(v[2:-2].cpu(), torch.cat(want[1]))
    assert K.kv8_error_flags() == 0


def test_in_a_graph_behind_copies_fills_and_other_streams():
    """Each operator captured behind what is not a kernel (a copy, a fill), as the first of its
    graph, and behind two streams that meet."""
    m = filled([300, 31, 0, 95], 2, 128, 32, E4M3, BF16, seed=50)
    m.table[1, 0], m.table[3, 2] = m.free.pop(), m.free.pop()          # of the blocks that a token completes
    n, arrays = m.lens(), m.arrays()
    q0, k0 = (torch.randn(4, h, 128, generator=m.g).to(BF16).cuda() for h in (8, 2))
    table, pos, off = K.rope_table(512, 128, device="cuda"), i32([300, 31, 0, 95]), i32([0, 300, 331, 331, 426])
    lens, q, k = n.clone(), q0.clone(), k0.clone()
    mutable = arrays[1:]
    start = [t.clone() for t in mutable]

    def call(what):
        if what == "rope":
            return K.qk_norm_rope(q, k, pos, table)
        if what == "write":
            K.write_kv8(k, k, lens, *arrays)
            return mutable
        if what == "read":
            return K.read_kv8(lens, *arrays, off, 426)
        return (K.paged_attention_kv8(q, lens, *arrays),)

    def before(how):
        if how == "copies":
            lens.copy_(n), q.copy_(q0), k.copy_(k0)
        elif how == "fills":
            lens.zero_(), q.zero_(), k.zero_()
        elif how == "streams":
            main, side = torch.cuda.current_stream(), torch.cuda.Stream()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                k.mul_(2)
                lens.copy_(n)
            q.mul_(2)
            main.wait_stream(side)

    def same(a, b):
        return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))

    for how in ("first", "copies", "fills", "streams"):
        for what in ("rope", "write", "read", "attention"):
            def set_up():
                for t, s in zip(mutable, start):
                    t.copy_(s)
                lens.copy_(n), q.copy_(q0), k.copy_(k0)
                torch.cuda.synchronize()
            set_up()
            before(how)
            torch.cuda.synchronize()
            want = [t.clone() for t in call(what)]
            flags = K.kv8_error_flags()                # (rows of emptied slots are none that can be read)
            graph = torch.cuda.CUDAGraph()
            set_up()
            with torch.cuda.graph(graph):
                before(how)
                got = call(what)
            for _ in range(3):
                if what == "read":
                    for t, w in zip(got, want):
                        t.copy_(w)                     # rows that are not read are left as they were
                set_up()
                graph.replay()
                torch.cuda.synchronize()
                assert same(got, want), (how, what)
            assert K.kv8_error_flags() == flags == (1 << 4 if how == "fills" and what == "read" else 0)


FIRST = """
import sys
sys.path[:0] = [{root!r}, {root!r} + "/kitty-kv_b200"]
import torch
from kitty import kernels as K
g = dict(device="cuda")
c = [torch.zeros(2, 1, 32, 64, dtype=torch.int8, **g) for _ in range(2)]
a = (torch.zeros(1, 2, dtype=torch.int32, **g), *c, torch.zeros(2, 1, **g), torch.zeros(2, 1, **g),
     torch.zeros(1, 1, 32, 64, dtype=torch.float16, **g), torch.zeros(1, 1, 32, 64, dtype=torch.float16, **g))
n = torch.zeros(1, dtype=torch.int32, **g)
row = torch.full((1, 1, 64), 2.0, dtype=torch.float16, **g)
table, pos = K.rope_table(8, 64, device="cuda"), torch.zeros(1, dtype=torch.int64, **g)
off = torch.tensor([0, 1], dtype=torch.int32, **g)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, k = K.qk_norm_rope(row, row, pos, table)
    K.write_kv8(k, row, n, *a)
    n += 1
    out = K.paged_attention_kv8(q, n, *a)
    kk, vv = K.read_kv8(n, *a, off, 1)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, row) and torch.equal(kk, row) and torch.equal(vv, row) and int(n) == 1
assert K.kv8_error_flags() == 0
print("captured")
"""


def test_first_calls_of_a_process_inside_a_capture():
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
