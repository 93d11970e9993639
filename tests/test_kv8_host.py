"""CPU tests of the 8-bit cache's library and bindings: exports, struct layouts, and
everything that is refused before a kernel is launched."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from kitty import kernels as K
from kitty.kernels import _kv8

HEADER = Path(__file__).resolve().parent.parent / "include" / "kitty_kv8.h"


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\*?\s+\**(kitty_\w+)\s*\(", text, flags=re.M)))


def test_exports_are_what_the_header_declares():
    names = declared()
    assert set(names) == set(_kv8.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", str(_kv8.library_path())], capture_output=True, text=True)
    if out.returncode == 0:
        assert set(re.findall(r"\sT\s(\w+)$", out.stdout, flags=re.M)) == set(names)


def test_version_and_struct_layouts():
    lib = _kv8.load()
    assert lib.kitty_kv8_abi_version() == _kv8.ABI_VERSION
    for kind, st in _kv8.STRUCTS.items():
        assert lib.kitty_kv8_args_size(kind) == ctypes.sizeof(st), st.__name__
    assert lib.kitty_kv8_args_size(99) == 0


def test_header_compiles_as_c(tmp_path):
    import shutil
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    src = tmp_path / "a.c"
    src.write_text('#include "kitty_b200.h"\n#include "kitty_kv8.h"\n'
                   "int main(void) { KittyKv8WriteArgs a = {0}; return kitty_kv8_write(&a, 0) == "
                   "KITTY_ERR_INVALID_ARGUMENT && kitty_kv8_args_size(0) == sizeof(KittyKv8Cache) ? 0 : 1; }\n")
    lib = _kv8.library_path()
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(HEADER.parent), str(src), "-o",
                        str(tmp_path / "a"), str(lib), f"-Wl,-rpath,{lib.parent}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(tmp_path / "a")]).returncode == 0


def cache(**kw):
    c = _kv8.Cache()
    for f in ("key_codes", "value_codes", "key_scale", "value_scale", "tail_k", "tail_v", "block_table", "lengths"):
        setattr(c, f, 0x1000)
    c.bt_s_slot, c.pages, c.slots, c.max_pages, c.num_heads, c.head_dim, c.page_size = 4, 8, 2, 4, 2, 64, 32
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(head_dim=72), dict(head_dim=272), dict(head_dim=0), dict(page_size=16), dict(page_size=33),
              dict(page_size=288), dict(num_heads=0), dict(num_heads=70000), dict(code=2), dict(dtype=2),
              dict(pages=1 << 31), dict(pages=-1), dict(slots=-1), dict(max_pages=-1), dict(lengths=0),
              dict(tail_k=0), dict(tail_v=0x1008), dict(key_codes=0x1001), dict(value_scale=0), dict(block_table=0)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_c_entry_points_refuse_bad_caches(bad):
    lib = _kv8.load()
    w, r, a = _kv8.WriteArgs(), _kv8.ReadArgs(), _kv8.AttentionArgs()
    n = _kv8.c_size(0)
    for s in (w, r, a):
        s.cache = cache(**bad)
    a.batch, a.num_q_heads = 1, 4
    for rc in (lib.kitty_kv8_write(w, None), lib.kitty_kv8_read(r, None), lib.kitty_kv8_attention(a, None),
               lib.kitty_kv8_attention_workspace_size(a, n)):
        assert rc in (1, 2) and lib.kitty_kv8_last_error()


def test_c_entry_points_refuse_bad_calls():
    lib = _kv8.load()

    def write(**kw):
        w = _kv8.WriteArgs()
        w.cache, w.key, w.value, w.n, w.rows = cache(), 0x1000, 0x1000, 2, 2
        w.k_s_row = w.v_s_row = 128
        w.k_s_head = w.v_s_head = 64
        for k, v in kw.items():
            setattr(w, k, v)
        return lib.kitty_kv8_write(w, None)

    for kw in (dict(n=1), dict(n=-1, rows=-1), dict(n=3, rows=3), dict(key=0), dict(value=0x1008), dict(k_s_row=4),
               dict(v_s_head=63)):
        assert write(**kw) == 1, kw
    assert write(n=0, rows=0) == 0

    def read(**kw):
        r = _kv8.ReadArgs()
        r.cache, r.key, r.value, r.row_offsets, r.n, r.rows = cache(), 0x1000, 0x1000, 0x1000, 2, 2
        for k, v in kw.items():
            setattr(r, k, v)
        return lib.kitty_kv8_read(r, None)

    for kw in (dict(n=-1), dict(rows=-1), dict(n=3), dict(key=0), dict(value=0x1008), dict(row_offsets=0)):
        assert read(**kw) == 1, kw
    assert read(rows=0) == 0

    def attend(**kw):
        a = _kv8.AttentionArgs()
        a.cache, a.q, a.out, a.batch, a.num_q_heads, a.workspace = cache(), 0x1000, 0x1000, 2, 4, 0x1000
        a.q_s_seq = a.out_s_seq = 256
        a.q_s_head = a.out_s_head = 64
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.kitty_kv8_attention(a, None)

    for kw in (dict(batch=-1), dict(num_q_heads=3), dict(num_q_heads=0), dict(batch=3), dict(q=0), dict(out=0),
               dict(q=0x1008), dict(q_s_head=4), dict(out_s_head=2)):
        assert attend(**kw) == 1, kw
    assert attend(workspace=0) == 4 and attend(workspace=0x1004) == 4
    assert attend(batch=1 << 30, seq_map=0x1000, num_q_heads=1 << 12) == 2
    assert attend(batch=0) == 0

    def rope(**kw):
        a = _kv8.QkNormRopeArgs()
        a.q = a.k = a.q_out = a.k_out = a.positions = a.table = 0x1000
        a.rows, a.num_q_heads, a.num_k_heads, a.head_dim, a.rot, a.table_rows = 2, 4, 2, 64, 32, 10
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.kitty_qk_norm_rope(a, None)

    for kw in (dict(rows=-1), dict(head_dim=0), dict(rot=-16), dict(dtype=2), dict(q_weight=0x1000), dict(positions=0),
               dict(table=0), dict(q=0), dict(k_out=0), dict(q_s_row=4), dict(ko_s_head=1), dict(k=0x1008),
               dict(table=0x1004)):
        assert rope(**kw) == 1, kw
    for kw in (dict(head_dim=72), dict(head_dim=512), dict(rot=24), dict(rot=80)):
        assert rope(**kw) == 2, kw
    assert rope(rows=0) == 0
    for fn in ("kitty_kv8_write", "kitty_kv8_read", "kitty_kv8_attention", "kitty_qk_norm_rope"):
        assert getattr(lib, fn)(None, None) == 1


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.qk_norm_rope(z, z, torch.zeros(1, dtype=torch.int64), torch.zeros(4, 64))
    p = torch.zeros(1, 1, 32, 64, dtype=torch.int8)
    arrays = (torch.zeros(1, 1, dtype=torch.int32), p, p, torch.zeros(1, 1), torch.zeros(1, 1), p.half(), p.half())
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.write_kv8(z, z, n, *arrays)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.read_kv8(n, *arrays, n, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.paged_attention_kv8(z, n, *arrays)


def test_rope_table_is_exact_far_out():
    t = K.rope_table(131072, 64)
    assert t.shape == (131072, 64) and t.dtype == torch.float32
    p = torch.tensor([0, 1, 4097, 131071])
    f = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    a = p.double()[:, None] * f
    assert (t[p].double() - torch.cat([a.cos(), a.sin()], 1)).abs().max() <= 2.0 ** -24
    assert torch.equal(K.rope_table(9, 64, inv_freq=f), t[:9])
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(max_positions=-1),
                dict(inv_freq=torch.ones(5))):
        with pytest.raises(RuntimeError):
            K.rope_table(**{**dict(max_positions=4, rotary_dim=64), **bad})


def test_cache_class_is_refused_on_the_cpu_and_for_bad_shapes():
    import kitty
    ok = dict(num_layers=1, num_kv_heads=2, head_dim=64, max_seq_len=128, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        kitty.PagedKVCache8(kitty.KittyConfig(**ok), 2)
    for cfg, kw in ((dict(head_dim=72), {}), (dict(head_dim=288), {}), ({}, dict(page_size=48)), ({}, dict(page_size=0)),
                    ({}, dict(page_size=512)), ({}, dict(codes="int4"))):
        with pytest.raises(RuntimeError):
            kitty.PagedKVCache8(kitty.KittyConfig(**{**ok, **cfg, "device": "cuda:0"}), 2, **kw)
