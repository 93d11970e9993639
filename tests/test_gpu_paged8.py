"""GPU tests of ``kitty.PagedKVCache8`` and of the operators around it as a decode loop
uses them: norm and rotation, append, attention, over layers and changing batches,
against a float64 model of the whole run."""

from __future__ import annotations

import random

import pytest
import torch

import kitty
from kitty import KittyConfig, PagedKVCache8
from kitty import kernels as K
from kv8_model import CacheModel, attention, attention_tolerance

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def config(**kw):
    d = dict(num_layers=2, num_kv_heads=2, head_dim=64, max_seq_len=512, device="cuda:0", dtype="bfloat16")
    d.update(kw)
    return KittyConfig(**d)


class Run:
    """A cache and the rows that went into it."""

    def __init__(self, seed=0, codes="e4m3", max_seqs=5, page_size=32, num_pages=None, **kw):
        self.cfg = config(**kw)
        self.cache = PagedKVCache8(self.cfg, max_seqs, page_size=page_size, codes=codes, num_pages=num_pages)
        self.models = [CacheModel(max_seqs, self.cfg.num_kv_heads, self.cfg.head_dim, page_size,
                                  self.cache.key_codes.dtype, self.cache.dtype, 1, 1, seed=seed + l)
                       for l in range(self.cfg.num_layers)]

    def note(self, l, slot, k, v):
        m = self.models[l]
        m.rows[slot][0].extend(k.cpu().unbind(0))
        m.rows[slot][1].extend(v.cpu().unbind(0))
        m.lengths[slot] += len(k)

    def drop(self, slots):
        for m in self.models:
            for s in slots:
                m.rows[s] = ([], [])
                m.lengths[s] = 0

    def check(self, l, slots, hq):
        m = self.models[l]
        q = torch.randn(len(slots), hq, m.d, generator=m.g).to(m.dtype).cuda()
        got = self.cache.decode(l, q, slots)
        for i, s in enumerate(slots):
            want, absum, mass = attention(q[i].cpu(), *m.truth(s))
            err = (got[i].cpu().double() - want).abs()
            assert (err <= attention_tolerance(want, absum, mass, m.dtype)).all(), (l, s, int(m.lengths[s]))

    def check_read(self, l, slots):
        key, value, lens = self.cache.read(l, slots)
        at = 0
        for s, n in zip(slots, lens):
            want = self.models[l].truth(s)
            assert n == want[0].shape[1]
            for got, w in ((key, want[0]), (value, want[1])):
                assert torch.equal(got[at:at + n].cpu(), w.transpose(0, 1).float().to(got.dtype))
            at += n
        assert key.shape[0] == at


@pytest.mark.parametrize("codes,dtype", [("e4m3", "bfloat16"), ("int8", "float16")])
def test_a_serving_loop(codes, dtype):
    """Prompts of several lengths, then decode steps of changing batches with norm, rotation,
    append and attention in every layer, a release and a new prompt in between."""
    run = Run(seed=1, codes=codes, dtype=dtype, max_seqs=4)
    cfg, cache, rng = run.cfg, run.cache, random.Random(3)
    h, d, hq = cfg.num_kv_heads, cfg.head_dim, 8
    t16 = cache.dtype
    table = K.rope_table(cfg.max_seq_len, d, device="cuda")
    wq, wk = (torch.rand(d, generator=run.models[0].g).add(0.5).to(t16).cuda() for _ in range(2))

    def rows(l, counts, slots):
        """Projections of new tokens -> rotated keys (checked against the operator's own values by
        its tests) and values, appended."""
        n = sum(counts)
        qkv = torch.randn(n, (hq + 2 * h) * d, generator=run.models[l].g).to(t16).cuda()
        pos = torch.cat([torch.arange(c) + cache.lengths(l)[s] for c, s in zip(counts, slots)]).cuda()
        q, k = K.qk_norm_rope(qkv[:, :hq * d].view(n, hq, d), qkv[:, hq * d:(hq + h) * d].view(n, h, d), pos, table, wq, wk)
        v = qkv[:, (hq + h) * d:].view(n, h, d)
        at = 0
        for c, s in zip(counts, slots):
            run.note(l, s, k[at:at + c], v[at:at + c])
            at += c
        return q, k, v

    def prompt(slots, counts):
        for l in range(cfg.num_layers):
            _, k, v = rows(l, counts, slots)
            cache.prefill(l, slots, k, v, counts)

    prompt([0, 1, 2], [70, 1, 33])
    for step in range(40):
        slots = rng.sample([0, 1, 2] if step < 20 else [0, 2, 3], rng.randint(1, 3))
        for l in range(cfg.num_layers):
            q, k, v = rows(l, [1] * len(slots), slots)
            cache.append(l, slots, k, v)
            got = cache.decode(l, q, slots)
            if step % 13 == 0 or step == 39:
                m = run.models[l]
                for i, s in enumerate(slots):
                    want, absum, mass = attention(q[i].cpu(), *m.truth(s))
                    assert ((got[i].cpu().double() - want).abs() <= attention_tolerance(want, absum, mass, m.dtype)).all()
        if step == 19:
            cache.release([1])
            run.drop([1])
            prompt([3, 1], [64, 31])
    for l in range(cfg.num_layers):
        run.check(l, [3, 0, 1, 2], hq)
        run.check_read(l, [2, 0, 3, 1])
    assert cache.lengths(0) == run.models[0].lengths.tolist()
    cache.check_errors()


def test_prefill_in_pieces_is_the_same_as_at_once():
    whole, pieces = Run(seed=5), Run(seed=5)
    m = whole.models[0]
    k, v = m.new_rows(200).cuda(), m.new_rows(200).cuda()
    whole.cache.prefill(0, [1, 3], k, v, [150, 50])
    for a, b in ((0, 1), (1, 31), (31, 33), (33, 97), (97, 150)):
        pieces.cache.prefill(0, [1], k[a:b], v[a:b], [b - a])
    for t in range(150, 200):
        pieces.cache.append(0, [3], k[t:t + 1], v[t:t + 1])
    for x, y in zip(whole.cache.read(0, [1, 3]), pieces.cache.read(0, [1, 3])):
        assert x == y if isinstance(x, list) else torch.equal(x, y)
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    assert torch.equal(whole.cache.decode(0, q, [1, 3]), pieces.cache.decode(0, q, [1, 3]))


def test_what_does_not_fit_changes_nothing():
    run = Run(num_pages=5, num_layers=1)
    m, cache = run.models[0], run.cache
    k, v = m.new_rows(120).cuda(), m.new_rows(120).cuda()
    cache.prefill(0, [0, 1], k, v, [70, 50])
    run.note(0, 0, k[:70], v[:70])
    run.note(0, 1, k[70:], v[70:])
    assert cache.free_page_count() == 2
    big, one = m.new_rows(130).cuda(), m.new_rows(1).cuda()
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.prefill(0, [2], big, big, [130])
    with pytest.raises(RuntimeError, match="twice"):
        cache.append(0, [1, 1], big[:2], big[:2])
    with pytest.raises(RuntimeError, match="sequence ids"):
        cache.append(0, [5], one, one)
    with pytest.raises(RuntimeError, match="key must be"):
        cache.append(0, [0], one.half(), one)
    with pytest.raises(RuntimeError, match="value must be"):
        cache.append(0, [0], one, big[:2])
    with pytest.raises(RuntimeError, match="lengths"):
        cache.prefill(0, [0, 1], one, one, [1])
    small = Run(num_layers=1, max_seq_len=64)
    with pytest.raises(RuntimeError, match="pages of 32"):
        small.cache.prefill(0, [0], k[:96], v[:96], [96])
    assert cache.free_page_count() == 2 and cache.lengths(0) == [70, 50, 0, 0, 0]
    run.check(0, [0, 1, 2], 4)
    run.check_read(0, [0, 1, 2])
    cache.release([0, 2])
    run.drop([0, 2])
    assert cache.free_page_count() == 4
    cache.prefill(0, [2], big, big, [130])
    run.note(0, 2, big, big)
    run.check(0, [2, 1, 0], 4)
    cache.check_errors()


def test_empty_calls_and_reset():
    run = Run()
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    run.cache.append(0, [], none, none)
    run.cache.prefill(0, [2], none, none, [0])
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    assert not run.cache.decode(0, q, [0, 2]).any()
    k, v, lens = run.cache.read(0, [0, 2])
    assert k.shape == v.shape == (0, 2, 64) and lens == [0, 0]
    assert run.cache.decode(0, q[:0], []).shape == (0, 4, 64)
    rows = run.models[0].new_rows(40).cuda()
    run.cache.prefill(0, [2], rows, rows, [40])
    run.cache.reset()
    assert run.cache.lengths(0) == [0] * 5 and run.cache.free_page_count() == run.cache.num_pages
    assert not run.cache.decode(0, q, [0, 2]).any()
    run.cache.check_errors()


def test_capture_is_refused_for_appends_and_taken_for_decodes():
    run = Run(num_layers=1)
    m = run.models[0]
    k, v = m.new_rows(100).cuda(), m.new_rows(100).cuda()
    run.cache.prefill(0, [0, 1], k, v, [64, 36])
    run.note(0, 0, k[:64], v[:64])
    run.note(0, 1, k[64:], v[64:])
    ids = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    want = run.cache.decode(0, q, ids)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run.cache.decode(0, q, ids)
        with pytest.raises(RuntimeError, match="captured"):
            run.cache.append(0, [0], k[:1], v[:1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and run.cache.lengths(0)[:2] == [64, 36]


# ------------------------------------------------------------------------------------------------ refusals

def arrays(slots=2, h=2, g=32, d=64, p=3, m=2, code=torch.int8, dtype=BF16):
    kw = dict(device="cuda")
    c = lambda: torch.zeros(p, h, g, d, dtype=torch.int8, **kw).view(code)
    return dict(lengths=torch.zeros(slots, dtype=torch.int32, **kw), block_table=torch.zeros(slots, m, dtype=torch.int32, **kw),
                key_codes=c(), value_codes=c(), key_scale=torch.zeros(p, h, **kw), value_scale=torch.zeros(p, h, **kw),
                tail_k=torch.zeros(slots, h, g, d, dtype=dtype, **kw), tail_v=torch.zeros(slots, h, g, d, dtype=dtype, **kw))


BAD_ARRAYS = [("lengths", lambda t: t.long()), ("lengths", lambda t: t[:1]), ("lengths", lambda t: t.view(1, -1)),
              ("block_table", lambda t: t.long()), ("block_table", lambda t: t[:1]), ("block_table", lambda t: t.t()),
              ("key_codes", lambda t: t.view(torch.uint8)), ("key_codes", lambda t: t[:2]),
              ("value_codes", lambda t: t.view(torch.float8_e4m3fn)), ("key_codes", lambda t: t.transpose(1, 2)),
              ("key_scale", lambda t: t.half()), ("key_scale", lambda t: t[:2]), ("value_scale", lambda t: t.t()),
              ("tail_k", lambda t: t.float()), ("tail_v", lambda t: t.half()), ("tail_v", lambda t: t[:1]),
              ("tail_k", lambda t: t[..., :32]), ("tail_k", lambda t: t.cpu()), ("lengths", lambda t: t.cpu()),
              ("key_scale", lambda t: None)]


@pytest.mark.parametrize("i", range(len(BAD_ARRAYS)))
def test_bad_cache_arrays_are_refused(i):
    name, change = BAD_ARRAYS[i]
    a = arrays()
    a[name] = change(a[name])
    row = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    for call in (lambda: K.write_kv8(row, row, **a), lambda: K.read_kv8(**a, row_offsets=off, rows=0),
                 lambda: K.paged_attention_kv8(row, **a)):
        with pytest.raises(RuntimeError):
            call()


def test_bad_calls_are_refused():
    a = arrays()
    row = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bad = [lambda: K.write_kv8(row.half(), row, **a), lambda: K.write_kv8(row, row.half(), **a),
           lambda: K.write_kv8(row[:, :1], row[:, :1], **a), lambda: K.write_kv8(row, row[:1], **a),
           lambda: K.write_kv8(row[0], row[0], **a), lambda: K.write_kv8(row, row, **a, seq_map=i(1)),
           lambda: K.write_kv8(row, row, **a, row_offsets=i(0, 1, 2, 2)),        # more entries than slots
           lambda: K.write_kv8(row, row, **a, row_offsets=i(0, 2), seq_map=i(0, 1)),
           lambda: K.write_kv8(row, row, **a, row_offsets=i(0, 1, 2).long()),
           lambda: K.write_kv8(row, row, **a, row_offsets=i(), seq_map=None),
           lambda: K.write_kv8(row, row, **a, seq_map=i(0, 1).cpu()),
           lambda: K.write_kv8(row.clone().requires_grad_(), row, **a),
           lambda: K.read_kv8(**a, row_offsets=i(0, 1, 2), rows=-1), lambda: K.read_kv8(**a, row_offsets=i(), rows=0),
           lambda: K.read_kv8(**a, row_offsets=i(0, 1), rows=1, first=i(0, 0)),
           lambda: K.read_kv8(**a, row_offsets=i(0, 2), rows=2, key_out=row.half()),
           lambda: K.read_kv8(**a, row_offsets=i(0, 2), rows=2, value_out=row.transpose(0, 1)),
           lambda: K.read_kv8(**a, row_offsets=i(0, 2), rows=1, value_out=row),
           lambda: K.paged_attention_kv8(row.half(), **a), lambda: K.paged_attention_kv8(row[..., :32], **a),
           lambda: K.paged_attention_kv8(row[:, :1], **a), lambda: K.paged_attention_kv8(row[:, :0], **a),
           lambda: K.paged_attention_kv8(row[0], **a), lambda: K.paged_attention_kv8(torch.cat([row, row]), **a),
           lambda: K.paged_attention_kv8(row, **a, seq_map=i(0)), lambda: K.paged_attention_kv8(row, **a, out=row.half()),
           lambda: K.paged_attention_kv8(row, **a, out=row[:1].expand(2, 2, 64)),
           lambda: K.paged_attention_kv8(row, **a, out=torch.zeros(2, 2, 65, dtype=BF16, device="cuda")[..., 1:]),
           lambda: K.paged_attention_kv8(row, **a, sm_scale="x"),
           lambda: K.paged_attention_kv8(row.clone().requires_grad_(), **a)]
    for n, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            raise AssertionError(f"call {n} was taken")
    for kw in (dict(d=72), dict(g=48), dict(g=512), dict(d=272)):
        b = arrays(**kw)
        with pytest.raises(RuntimeError):
            K.paged_attention_kv8(torch.zeros(2, 2, kw.get("d", 64), dtype=BF16, device="cuda"), **b)


def test_bad_rope_calls_are_refused():
    q = torch.zeros(3, 4, 64, dtype=BF16, device="cuda")
    pos, table = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(5, 64, device="cuda")
    w = torch.ones(64, dtype=BF16, device="cuda")
    bad = [lambda: K.qk_norm_rope(q, q.half(), pos, table), lambda: K.qk_norm_rope(q.float(), q.float(), pos, table),
           lambda: K.qk_norm_rope(q, q[:2], pos, table), lambda: K.qk_norm_rope(q, q[..., :32], pos, table),
           lambda: K.qk_norm_rope(q, q, pos[:2], table), lambda: K.qk_norm_rope(q, q, pos.short(), table),
           lambda: K.qk_norm_rope(q, q, pos, table.half()), lambda: K.qk_norm_rope(q, q, pos, table.t()),
           lambda: K.qk_norm_rope(q, q, pos, table[:, :24].contiguous()),
           lambda: K.qk_norm_rope(q, q, pos, torch.zeros(5, 80, device="cuda")),
           lambda: K.qk_norm_rope(q, q, pos, table, w), lambda: K.qk_norm_rope(q, q, pos, table, w, w.float()),
           lambda: K.qk_norm_rope(q, q, pos, table, w.half(), w.half()), lambda: K.qk_norm_rope(q, q, pos, table, w[:32], w[:32]),
           lambda: K.qk_norm_rope(q, q, pos, table, q_out=q.half()), lambda: K.qk_norm_rope(q, q, pos, table, q_out=q[:, :2]),
           lambda: K.qk_norm_rope(q, q, pos, table, k_out=q[:1].expand(3, 4, 64)),
           lambda: K.qk_norm_rope(q, q, pos.cpu(), table), lambda: K.qk_norm_rope(q.clone().requires_grad_(), q, pos, table),
           lambda: K.qk_norm_rope(q, q, pos, table, w.clone().requires_grad_(), w)]
    for n, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            raise AssertionError(f"call {n} was taken")
    with torch.no_grad():
        K.qk_norm_rope(q.clone().requires_grad_(), q, pos, table)
