"""GPU tests of the 8-bit paged cache operators against the plain model (codes and
scales bit for bit, attention in float64 within a derived bound)."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from kv8_model import CacheModel, attention, attention_tolerance

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same_bits(a, b):
    """Equal bit for bit, any NaN equal to any NaN."""
    a, b = a.cpu(), b.cpu()
    if a.dtype == INT8:
        return torch.equal(a, b)
    x, y = a.float(), b.float()
    return bool(((x == y) | (x.isnan() & y.isnan())).all())


def expect_arrays(m):
    """The arrays that the model's tokens lead to, on fresh zeros."""
    e = CacheModel(m.slots, m.h, m.d, m.page, m.code, m.dtype, m.key_scale.shape[0], m.table.shape[1])
    e.rows, e.table, e.lengths = m.rows, m.table, m.lengths
    e.fill_arrays()
    return e


def check_cache(m):
    """Codes and scales of every page in use, and the live tail rows."""
    e = expect_arrays(m)
    for s in range(m.slots):
        n = int(m.lengths[s])
        pages = m.table[s, :n // m.page].long()
        for name in ("key_codes", "value_codes", "key_scale", "value_scale"):
            a, b = getattr(m, name), getattr(e, name)
            a, b = (a.view(torch.uint8)[pages.cuda()].view(a.dtype), b.view(torch.uint8)[pages.cuda()].view(b.dtype)) \
                if "codes" in name else (a[pages.cuda()], b[pages.cuda()])
            assert same_bits(a, b), f"slot {s}: {name}"
        for name in ("tail_k", "tail_v"):
            assert same_bits(getattr(m, name)[s, :, :n % m.page], getattr(e, name)[s, :, :n % m.page]), f"slot {s}: {name}"


def write(m, slots, counts, seq_map=None, with_offsets=True, padding=0, scale=1.0, edit=None):
    """Append counts[i] new rows to slots[i] by one call and note them in the model."""
    before = m.lens()
    n = sum(counts)
    k, v = m.new_rows(n + padding, scale), m.new_rows(n + padding, scale)
    if edit is not None:
        edit(k, v)
    at = [0]
    for s, c in zip(slots, counts):
        m.append(s, k[at[-1]:at[-1] + c], v[at[-1]:at[-1] + c])
        at.append(at[-1] + c)
    K.write_kv8(k.cuda(), v.cuda(), before, *m.arrays(), row_offsets=i32(at) if with_offsets else None,
                seq_map=seq_map)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,dim,page", [(2, 128, 64), (1, 64, 32), (3, 80, 96), (2, 256, 256), (1, 16, 32)])
def test_write_prefill_then_chunks_then_tokens(code, dtype, heads, dim, page):
    m = CacheModel(5, heads, dim, page, code, dtype, pages=40, table_width=16, seed=dim + page)
    write(m, range(5), [0, 1, page - 1, page, 2 * page + 5])
    check_cache(m)
    write(m, range(5), [page, page - 1, 1, 3, 3 * page - 5])             # blocks that began in the tail
    check_cache(m)
    write(m, range(5), [page + 1, 2 * page, 7, 0, page // 2], padding=page + 3)
    check_cache(m)
    for _ in range(3):
        write(m, range(5), [1] * 5, with_offsets=False)
        check_cache(m)
    assert K.kv8_error_flags() == 0


def test_write_single_tokens_through_a_block_boundary():
    m = CacheModel(3, 2, 128, 32, E4M3, BF16, pages=9, table_width=3, seed=3)
    write(m, range(3), [30, 31, 0])
    for _ in range(35):
        write(m, range(3), [1] * 3, with_offsets=False)
    check_cache(m)
    assert m.lengths.tolist() == [65, 66, 35] and K.kv8_error_flags() == 0


def test_write_to_mapped_slots_leaves_the_others():
    m = CacheModel(6, 2, 64, 32, INT8, FP16, pages=30, table_width=8, seed=5)
    write(m, range(6), [40, 3, 64, 0, 17, 31])
    tails = m.tail_k.clone()
    write(m, [4, 0, 5], [20, 30, 1], seq_map=i32([4, 0, 5]))
    check_cache(m)
    for s in (1, 2, 3):
        assert torch.equal(m.tail_k[s], tails[s])
    assert K.kv8_error_flags() == 0


def test_write_many_ragged_entries():
    """More entries than a warp looks at in one step of its search, many of them empty."""
    g = torch.Generator().manual_seed(1)
    n = 1100
    m = CacheModel(n, 1, 64, 32, E4M3, FP16, pages=4000, table_width=8, seed=6)
    counts = torch.randint(0, 90, (n,), generator=g)
    counts[torch.rand(n, generator=g) < 0.4] = 0
    counts[:5] = 0
    write(m, range(n), counts.tolist(), padding=40)
    check_cache(m)
    assert K.kv8_error_flags() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_write_extreme_blocks(code, dtype):
    """All zeros, the smallest and the largest magnitudes, ties, an infinity and a NaN."""
    m = CacheModel(7, 1, 64, 32, code, dtype, pages=7, table_width=1, seed=8)
    small, large = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max

    def edit(k, v):
        for x in (k, v):
            b = x.view(7, 32, 64)
            b[0] = 0
            b[1] *= small
            b[2] = b[2].sign() * large
            b[3] = torch.arange(-64, 64, dtype=torch.float32).repeat(16).view(32, 64).to(dtype) / 2
            b[4, 3, 5] = float("inf")
            b[5, 7, 9] = float("nan")
            b[6] *= torch.tensor(1e-3, dtype=dtype)

    write(m, range(7), [32] * 7, edit=edit)
    check_cache(m)
    k, v = K.read_kv8(m.lens(), *m.arrays(), i32(list(range(0, 225, 32))), 224)
    assert k.view(7, -1)[0].eq(0).all()
    assert not k.view(7, -1)[[0, 1, 2, 3, 6]].isnan().any()
    assert k.view(7, -1)[4:6].isnan().all() and v.view(7, -1)[4:6].isnan().all()
    assert K.kv8_error_flags() == 0


def test_write_strided_and_unaligned_rows():
    m = CacheModel(2, 2, 64, 32, E4M3, BF16, pages=8, table_width=4, seed=9)
    n = 70
    for pad in (0, 3):                                   # 3: rows that are not 16-byte aligned
        k, v = m.new_rows(n), m.new_rows(n)
        big = torch.zeros(n, 4 * 64 + 16 + pad, dtype=BF16)
        big[:, 8 + pad:8 + pad + 128] = k.view(n, -1)
        big[:, 136 + pad:136 + pad + 128] = v.view(n, -1)
        big = big.cuda()
        before = m.lens()
        m.append(0, k[:37], v[:37])
        m.append(1, k[37:], v[37:])
        K.write_kv8(big[:, 8 + pad:136 + pad].view(n, 2, 64), big[:, 136 + pad:264 + pad].view(n, 2, 64), before,
                    *m.arrays(), row_offsets=i32([0, 37, 70]))
        check_cache(m)
    assert K.kv8_error_flags() == 0


def test_write_flags_bad_device_data():
    """Repeated or missing slots, bad pages, bad offsets: skipped, flagged, nothing else touched."""
    def fresh():
        m = CacheModel(4, 1, 64, 32, E4M3, BF16, pages=4, table_width=1, seed=11)
        return m, m.new_rows(32).cuda(), m.new_rows(32).cuda()

    def call(m, k, v, table=None, **kw):
        K.write_kv8(k, v, m.lens(), *m.arrays(table), **kw)
        return K.kv8_error_flags()

    m, k, v = fresh()
    assert call(m, k[:3], v[:3], seq_map=i32([2, 1, 2])) == 1 << 3
    assert torch.equal(m.tail_k[2, 0, 0], k[0, 0]) and torch.equal(m.tail_k[1, 0, 0], k[1, 0])
    m, k, v = fresh()
    assert call(m, k[:2], v[:2], seq_map=i32([4, -1])) == 1 << 3
    assert not m.tail_k.any()
    for page in (-7, 4, 1 << 30):
        m, k, v = fresh()
        assert call(m, k, v, table=torch.full((4, 1), page, dtype=torch.int32),
                    row_offsets=i32([0, 32, 32, 32, 32])) == 1 << 1
        assert not m.key_scale.any() and not m.tail_k.any()
    for offsets in ([0, 40, 40, 40, 40], [0, 5, 3, 4, 4], [-3, 2, 2, 2, 2], [0, 1 << 30, -5, 9, 9]):
        m, k, v = fresh()
        assert call(m, k, v, row_offsets=i32(offsets)) & (1 << 2)
    m, k, v = fresh()
    m.lengths[1] = -1
    assert call(m, k[:4], v[:4]) == 1 << 4
    m, k, v = fresh()
    m.lengths[0] = 63                                     # its next block has no entry in the table
    assert call(m, k[:1], v[:1], row_offsets=i32([0, 1, 1, 1, 1])) == 1 << 1


# ------------------------------------------------------------------------------------------------ read

@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,dim,page", [(2, 128, 64), (1, 64, 32), (3, 80, 96), (2, 256, 256)])
def test_read_back(code, dtype, heads, dim, page):
    m = CacheModel(5, heads, dim, page, code, dtype, pages=40, table_width=10, seed=dim, fill=float("nan"))
    lens = [0, 1, page, 2 * page + 9, 3 * page - 1]
    for s, n in enumerate(lens):
        m.append(s, m.new_rows(n), m.new_rows(n))
    m.fill_arrays()
    slots = [3, 0, 4, 3, 1, 2]
    first = [0, 0, page + 3, page - 1, 0, 5]
    counts = [lens[3], 0, lens[4] - first[2], 7, 1, page - 5]
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    rows = at[-1] + 4                                     # four rows behind the last entry
    ko = torch.full((rows, heads, dim), 9.0, dtype=dtype, device="cuda")
    vo = torch.full_like(ko, 7.0)
    k, v = K.read_kv8(m.lens(), *m.arrays(), i32(at), rows, first=i32(first), seq_map=i32(slots), key_out=ko,
                      value_out=vo)
    assert k is ko and v is vo
    for i, s in enumerate(slots):
        want = m.truth(s)
        for got, w in ((k, want[0]), (v, want[1])):
            w = w[:, first[i]:first[i] + counts[i]].transpose(0, 1).float().to(dtype)
            assert torch.equal(got[at[i]:at[i + 1]].cpu(), w)
    assert (k[at[-1]:] == 9).all() and (v[at[-1]:] == 7).all()
    assert K.kv8_error_flags() == 0


def test_read_flags_what_is_not_there():
    m = CacheModel(2, 1, 64, 32, INT8, FP16, pages=4, table_width=2, seed=2)
    m.append(0, m.new_rows(40), m.new_rows(40))
    m.fill_arrays()

    def call(offsets, rows, table=None, **kw):
        ko = torch.full((rows, 1, 64), 9.0, dtype=FP16, device="cuda")
        k, _ = K.read_kv8(m.lens(), *m.arrays(table), i32(offsets), rows, key_out=ko, **kw)
        return K.kv8_error_flags(), k

    f, k = call([0, 45, 45], 45)                          # five tokens more than there are
    assert f == 1 << 4 and (k[40:] == 9).all() and not (k[:40] == 9).all()
    f, k = call([0, 4], 4, seq_map=i32([2]))
    assert f == 1 << 3 and (k == 9).all()
    f, k = call([0, 4, 4], 4, first=i32([-2, 0]))
    assert f == 1 << 4 and (k[:2] == 9).all() and not (k[2:] == 9).any()
    f, k = call([0, 40, 40], 40, table=torch.full((2, 2), 99, dtype=torch.int32))
    assert f == 1 << 1 and (k[:32] == 9).all()


# ------------------------------------------------------------------------------------------------ attention

def check_attention(m, hq, rows=None, sm_scale=None, q=None, out=None, got=None):
    """Run (or take) the decode of batch rows ``rows`` (slots) and compare with float64."""
    rows = list(range(m.slots)) if rows is None else rows
    if q is None:
        q = torch.randn(len(rows), hq, m.d, generator=m.g).to(m.dtype).cuda()
    if got is None:
        seq_map = i32(rows) if rows != list(range(m.slots)) else None
        got = K.paged_attention_kv8(q, m.lens(), *m.arrays(), sm_scale=sm_scale, seq_map=seq_map, out=out)
    for i, s in enumerate(rows):
        want, absum, mass = attention(q[i].cpu(), *m.truth(s), sm_scale=sm_scale)
        err = (got[i].cpu().double() - want).abs()
        tol = attention_tolerance(want, absum, mass, m.dtype)
        assert (err <= tol).all(), f"row {i}, length {int(m.lengths[s])}: error / bound {(err / tol).max():.2f}"
    return got


def filled(lens, heads, dim, page, code, dtype, seed=0, scale=1.0, fill=float("nan")):
    pages = sum(n // page for n in lens) + 3
    m = CacheModel(len(lens), heads, dim, page, code, dtype, pages, max(n // page for n in lens) + 2, seed, fill=fill)
    for s, n in enumerate(lens):
        m.append(s, m.new_rows(n, scale), m.new_rows(n))
    m.fill_arrays()
    return m


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,group,dim,page", [(2, 4, 128, 64), (1, 8, 128, 128), (2, 1, 64, 32), (1, 16, 64, 96),
                                                  (1, 9, 128, 32), (2, 5, 80, 64), (1, 40, 96, 32), (1, 3, 256, 256),
                                                  (1, 17, 256, 32), (1, 2, 16, 32), (2, 7, 48, 32), (1, 12, 160, 64)])
def test_attention_lengths(code, dtype, heads, group, dim, page):
    lens = [0, 1, 15, 16, 17, page - 1, page, page + 1, 2 * page + 33, 5 * page, 700]
    m = filled(lens, heads, dim, page, code, dtype, seed=dim + page + group)
    got = check_attention(m, heads * group)
    assert not got[0].any()                               # the empty slot
    assert K.kv8_error_flags() == 0


@pytest.mark.parametrize("code,dtype", [(E4M3, BF16), (INT8, FP16)])
def test_attention_long_sequences(code, dtype):
    """Sequences that many warps share, beside short and empty ones."""
    m = filled([9000, 0, 3, 4097], 1, 128, 64, code, dtype, seed=4)
    check_attention(m, 4)
    assert K.kv8_error_flags() == 0


def test_attention_mapped_rows_any_order_and_twice():
    m = filled([100, 0, 64, 333, 12], 2, 64, 32, E4M3, FP16, seed=7)
    check_attention(m, 8, rows=[3, 3, 1, 0, 4])


def test_attention_many_short_sequences():
    """More sequences than a warp scans at once, about as many segments as warps."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 130, (300,), generator=g).tolist()
    m = filled(lens, 4, 64, 32, INT8, BF16, seed=10)
    check_attention(m, 8)
    assert K.kv8_error_flags() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_strided_q_and_out(dtype):
    m = filled([90, 257], 2, 128, 64, E4M3, dtype, seed=12)
    big = torch.randn(2, 3 * 8 * 128, generator=m.g).to(dtype).cuda()
    q = big[:, 1024:2048].view(2, 8, 128)
    out = torch.full((8, 2, 128), 5.0, dtype=dtype, device="cuda").transpose(0, 1)      # head-major
    got = check_attention(m, 8, q=q, out=out)
    assert got is out
    odd = torch.randn(2 * 8 * 128 + 1, generator=m.g).to(dtype).cuda()[1:].view(2, 8, 128)  # not 16-byte aligned
    check_attention(m, 8, q=odd)
    inplace = torch.randn(2, 8, 128, generator=m.g).to(dtype).cuda()
    q = inplace.clone()
    check_attention(m, 8, q=q, got=K.paged_attention_kv8(inplace, m.lens(), *m.arrays(), out=inplace))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sm_scale", [1.0, 0.01, -0.3, 0.0])
def test_attention_scales(dtype, sm_scale):
    m = filled([200, 40], 1, 64, 32, E4M3, dtype, seed=13)
    check_attention(m, 4, sm_scale=sm_scale)


def test_attention_wide_range_of_queries_and_scales():
    """bf16 queries far outside fp16's range, and pages whose scales differ by 2^60."""
    m = CacheModel(1, 1, 64, 32, E4M3, BF16, pages=8, table_width=8, seed=14)
    for e in (-20, 0, 20, -40, 10, -20):
        m.append(0, m.new_rows(32, 2.0 ** -30), m.new_rows(32, 2.0 ** e))
    m.append(0, m.new_rows(5, 2.0 ** -30), m.new_rows(5))
    m.fill_arrays()
    check_attention(m, 4, q=(torch.randn(1, 4, 64, generator=m.g) * 2.0 ** 30).to(BF16).cuda())
    q = torch.randn(1, 4, 64, generator=m.g) * 2.0 ** 30
    q[..., 3] *= 2.0 ** 20
    q[..., 9] *= 2.0 ** -12
    check_attention(m, 4, q=q.to(BF16).cuda(), sm_scale=2.0 ** -20)


def test_attention_zero_blocks_and_nan_blocks():
    m = CacheModel(2, 1, 64, 32, INT8, FP16, pages=8, table_width=4, seed=15)
    z = torch.zeros(32, 1, 64, dtype=FP16)
    m.append(0, z, z)
    m.append(0, m.new_rows(40), m.new_rows(40))
    bad = m.new_rows(32)
    bad[3, 0, 5] = float("nan")
    m.append(1, m.new_rows(64), m.new_rows(64))
    m.fill_arrays()
    check_attention(m, 2)
    m.append(1, m.new_rows(32), bad)
    m.fill_arrays()
    got = K.paged_attention_kv8(torch.ones(2, 2, 64, dtype=FP16, device="cuda"), m.lens(), *m.arrays())
    assert got[1].isnan().all() and not got[0].isnan().any()


def test_attention_skips_and_flags_bad_device_data():
    m = filled([96, 50, 200], 1, 64, 32, E4M3, BF16, seed=16)
    q = torch.randn(3, 2, 64, generator=m.g).to(BF16).cuda()
    table = m.table.clone()
    table[0, 1] = 1 << 29                                 # one block of slot 0 is gone
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays(table))
    assert K.kv8_error_flags() == 1 << 1
    check_attention(m, 2, rows=[1, 2], q=q[1:], got=got[1:])
    k, v = m.truth(0)
    keep = [t for t in range(96) if not 32 <= t < 64]
    want, absum, mass = attention(q[0].cpu(), k[:, keep], v[:, keep])
    assert ((got[0].cpu().double() - want).abs() <= attention_tolerance(want, absum, mass, BF16)).all()
    got = K.paged_attention_kv8(q, m.lens(), *m.arrays(), seq_map=i32([0, 3, -1]))
    assert K.kv8_error_flags() == 1 << 3 and not got[1:].any()
    lens = m.lens()
    lens[1], lens[2] = -4, 32 * (m.table.shape[1] + 1)
    got = K.paged_attention_kv8(q, lens, *m.arrays())
    assert K.kv8_error_flags() == 1 << 4 and not got[1:].any()
    check_attention(m, 2, rows=[0], q=q[:1], got=got[:1])


def test_offsets_past_32_bits():
    """Pages whose byte offsets pass 2^32, written, read and attended to."""
    pages, h, page, d = 70000, 8, 64, 128                 # 4.6 GB of codes each
    m = CacheModel(1, h, d, page, E4M3, BF16, pages=pages, table_width=6, seed=17)
    m.free = [69999, 12, 69000, 65537, 65535, 3]
    write(m, [0], [5 * page + 9])
    k, v = K.read_kv8(m.lens(), *m.arrays(), i32([0, 5 * page + 9]), 5 * page + 9)
    want = m.truth(0)
    assert torch.equal(k.cpu(), want[0].transpose(0, 1).float().to(BF16))
    assert torch.equal(v.cpu(), want[1].transpose(0, 1).float().to(BF16))
    check_attention(m, 32)
    assert K.kv8_error_flags() == 0


def test_on_other_streams_and_in_graphs():
    """A decode step captured once and replayed with new rows, lengths and queries, beside
    a second graph of another cache on another stream."""
    caches = [filled([70, 5, 300], 2, 64, 32, E4M3, BF16, seed=20 + i) for i in range(2)]
    for m in caches:
        m.table[m.table < 0] = 0                          # entries for the blocks to come
        for s in range(3):
            for b in range(int(m.lengths[s]) // 32, min(int(m.lengths[s]) // 32 + 2, m.table.shape[1])):
                m.table[s, b] = -7
        # pages of the next block, given beforehand
    steps, graphs = 40, []
    for m in caches:
        extra = torch.zeros(6, 2, 32, 64, dtype=torch.int8, device="cuda")
        m.key_codes = torch.cat([m.key_codes.view(torch.int8), extra]).view(E4M3)
        m.value_codes = torch.cat([m.value_codes.view(torch.int8), extra]).view(E4M3)
        m.key_scale = torch.cat([m.key_scale, torch.zeros(6, 2, device="cuda")])
        m.value_scale = torch.cat([m.value_scale, torch.zeros(6, 2, device="cuda")])
        m.free = list(range(m.key_scale.shape[0] - 6, m.key_scale.shape[0]))
        s = {"m": m, "k": torch.zeros(3, 2, 64, dtype=BF16, device="cuda"), "lens": m.lens(),
             "table": m.table.cuda(), "q": torch.zeros(3, 8, 64, dtype=BF16, device="cuda"),
             "stream": torch.cuda.Stream()}
        s["v"] = torch.zeros_like(s["k"])

        def step(s=s, arrays=(s["table"], *m.arrays()[1:])):
            K.write_kv8(s["k"], s["v"], s["lens"], *arrays)
            s["lens"] += 1
            return K.paged_attention_kv8(s["q"], s["lens"], *arrays)

        tails = m.tail_k.clone(), m.tail_v.clone()
        with torch.cuda.stream(s["stream"]):
            step()                                        # a first call outside the capture
            s["stream"].synchronize()
            s["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(s["graph"], stream=s["stream"]):
                s["out"] = step()
            s["stream"].synchronize()
        m.tail_k.copy_(tails[0])
        m.tail_v.copy_(tails[1])
        s["lens"].copy_(m.lens())
        graphs.append(s)
    torch.cuda.synchronize()
    for t in range(steps):
        for s in graphs:
            m = s["m"]
            k, v = m.new_rows(3), m.new_rows(3)
            q = torch.randn(3, 8, 64, generator=m.g).to(BF16)
            for slot in range(3):
                m.append(slot, k[slot:slot + 1], v[slot:slot + 1])
            with torch.cuda.stream(s["stream"]):
                s["k"].copy_(k)
                s["v"].copy_(v)
                s["q"].copy_(q)
                s["table"].copy_(m.table)
        for s in graphs:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        if t % 13 == 0 or t == steps - 1:
            for s in graphs:
                check_attention(s["m"], 8, q=s["q"], got=s["out"])
    for s in graphs:
        check_cache(s["m"])
    assert K.kv8_error_flags() == 0
