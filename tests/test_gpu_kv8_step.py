"""GPU test of a layer's decode step as a user puts it together: norm and rotation, write,
lengths, attention, captured once and replayed with padded batches."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from kv8_model import CacheModel
from test_gpu_kv8 import BF16, E4M3, FP16, INT8, check_attention, check_cache, write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,dtype", [(E4M3, BF16), (INT8, FP16)])
def test_captured_step_of_padded_batches(code, dtype):
    heads, group, dim, page, batch = 2, 3, 64, 32, 5
    m = CacheModel(6, heads, dim, page, code, dtype, pages=20, table_width=4, seed=3)
    write(m, range(6), [30, 0, 31, 64, 5, 95])
    g = dict(device="cuda")
    lengths, table = m.lens(), m.table.cuda()
    arrays = (table, *m.arrays()[1:])
    slots = torch.full((batch,), -1, dtype=torch.int32, **g)
    positions = torch.full((batch,), -1, dtype=torch.int32, **g)
    q_in = torch.zeros(batch, heads * group, dim, dtype=dtype, **g)
    k_in, v = torch.zeros(batch, heads, dim, dtype=dtype, **g), torch.zeros(batch, heads, dim, dtype=dtype, **g)
    rope = K.rope_table(256, dim, device="cuda")
    w = [(1 + 0.1 * torch.randn(dim, generator=m.g)).cuda() for _ in range(2)]
    # made once: outputs of padding rows are left as they were
    q, k = torch.zeros_like(q_in), torch.zeros_like(k_in)

    def step():
        K.qk_norm_rope(q_in, k_in, positions, rope, *w, q_out=q, k_out=k)
        K.write_kv8(k, v, lengths, *arrays, seq_map=slots)
        lengths.index_add_(0, slots.clamp(min=0), (slots >= 0).to(torch.int32))
        return K.paged_attention_kv8(q, lengths, *arrays, seq_map=slots)

    step()                                                # all padding: nothing changes
    check_cache(m)
    assert torch.equal(lengths, m.lens())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(40):
        now = torch.randperm(6, generator=m.g)[:batch]
        now[torch.rand(batch, generator=m.g) < 0.4] = -1
        if t == 7:
            now[:] = -1
        for s in now.tolist():
            if s >= 0 and int(m.lengths[s]) >= 126:
                now[now == s] = -1
        q_in.copy_(torch.randn(batch, heads * group, dim, generator=m.g).to(dtype))
        k_in.copy_(m.new_rows(batch))
        v.copy_(m.new_rows(batch))
        slots.copy_(now.int())
        positions.copy_(torch.tensor([int(m.lengths[s]) if s >= 0 else -1 for s in now], dtype=torch.int32))
        # pages of the blocks that this step fills
        rows_of = [i for i, s in enumerate(now.tolist()) if s >= 0]
        for i in rows_of:
            s = int(now[i])
            if int(m.lengths[s]) % page == page - 1:
                m.table[s, int(m.lengths[s]) // page] = m.free[-1]
                table[s, int(m.lengths[s]) // page] = m.free[-1]
            m.append(s, torch.zeros(1, heads, dim, dtype=dtype), v[i:i + 1].cpu())
        graph.replay()
        torch.cuda.synchronize()
        for i in rows_of:                                 # the key row as it was rotated
            m.rows[int(now[i])][0][-1] = k[i].cpu()
        assert torch.equal(lengths, m.lens())
        pad = [i for i in range(batch) if i not in rows_of]
        assert not out[pad].any()
        check_attention(m, heads * group, rows=[int(now[i]) for i in rows_of], q=q[rows_of], got=out[rows_of])
    check_cache(m)
    assert K.kv8_error_flags() == 0
