"""GPU tests of the per-head norm with rotary embedding against float64."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from kv8_model import norm_rope

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def close(got, x, w, pos, table, eps, inter):
    """Rounded once: half a step.  Before it, float32: the mean of squares is off by at most
    24 roundings (halved by the root), the root's reciprocal by 2 units, the products and
    the rotation by 6 more: under 2^-19 of the magnitudes that meet."""
    want, mag = norm_rope(x.cpu(), None if w is None else w.cpu(), pos.cpu(), table.cpu(), eps, inter)
    err = (got.cpu().double() - want).abs()
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0 ** -19 * mag * (1 + torch.finfo(x.dtype).eps) + 2.0 ** -25
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n,hq,h,d,rot", [(1, 32, 8, 128, 128), (7, 5, 1, 64, 32), (33, 4, 2, 80, 80), (3, 9, 3, 96, 48),
                                          (5, 2, 2, 256, 64), (2, 17, 1, 256, 256), (9, 1, 1, 16, 16),
                                          (1000, 40, 8, 128, 64), (4, 3, 1, 160, 16), (6, 64, 64, 48, 32)])
def test_norm_and_rotation(dtype, inter, n, hq, h, d, rot):
    g = torch.Generator().manual_seed(n + d)
    q, k = (torch.randn(n, x, d, generator=g).mul(3).to(dtype).cuda() for x in (hq, h))
    table = K.rope_table(5000, rot, device="cuda")
    pos = torch.randint(0, 5000, (n,), generator=g).cuda()
    pos[-1] = 4999
    for w32 in (False, True):
        wq, wk = (torch.randn(d, generator=g).to(torch.float32 if w32 else dtype).cuda() for _ in range(2))
        qo, ko = K.qk_norm_rope(q, k, pos if w32 else pos.int(), table, wq, wk, eps=1e-5, interleaved=inter)
        close(qo, q, wq, pos, table, 1e-5, inter)
        close(ko, k, wk, pos, table, 1e-5, inter)
    qo, ko = K.qk_norm_rope(q, k, pos, table, interleaved=inter)
    close(qo, q, None, pos, table, 0, inter)
    close(ko, k, None, pos, table, 0, inter)
    assert K.kv8_error_flags() == 0


def test_in_place_on_a_fused_projection_leaves_the_values():
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(50, (8 + 2 + 2) * 64, generator=g).to(BF16).cuda()
    before = rows.clone()
    q, k = rows[:, :512].view(50, 8, 64), rows[:, 512:640].view(50, 2, 64)
    q0, k0 = q.clone(), k.clone()
    table, pos = K.rope_table(64, 64, device="cuda"), torch.arange(50, device="cuda")
    w = torch.ones(64, dtype=BF16, device="cuda")
    qo, ko = K.qk_norm_rope(q, k, pos, table, w, w, q_out=q, k_out=k)
    assert qo is q and ko is k
    close(q, q0, w, pos, table, 1e-6, False)
    close(k, k0, w, pos, table, 1e-6, False)
    assert torch.equal(rows[:, 640:], before[:, 640:])


def test_unaligned_inputs_and_strided_outputs():
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(4 * 3 * 64 + 1, generator=g).to(FP16).cuda()
    q = flat[1:].view(4, 3, 64)
    k = torch.randn(3, 4, 64, generator=g).to(FP16).cuda().transpose(0, 1)
    out = torch.zeros(3, 4, 64, dtype=FP16, device="cuda").transpose(0, 1)
    table, pos = K.rope_table(9, 32, device="cuda"), torch.tensor([8, 0, 3, 3], device="cuda")
    qo, ko = K.qk_norm_rope(q, k, pos, table, q_out=out)
    close(qo, q, None, pos, table, 0, False)
    close(ko, k, None, pos, table, 0, False)


def test_padding_rows_and_positions_past_the_table():
    q = torch.ones(4, 2, 64, dtype=BF16, device="cuda")
    qo, ko = torch.full_like(q, 9), torch.full_like(q, 9)
    table = K.rope_table(10, 64, device="cuda")
    K.qk_norm_rope(q, q, torch.tensor([-1, 3, -(1 << 40), 2], device="cuda"), table, q_out=qo, k_out=ko)
    assert (qo[[0, 2]] == 9).all() and (ko[[0, 2]] == 9).all() and not (qo[[1, 3]] == 9).any()
    assert K.kv8_error_flags() == 0
    qo.fill_(9)
    K.qk_norm_rope(q, q, torch.tensor([1, 10, 1 << 40, 2], device="cuda"), table, q_out=qo, k_out=ko)
    assert (qo[[1, 2]] == 9).all() and not (qo[[0, 3]] == 9).any()
    assert K.kv8_error_flags() == 1 << 5


def test_special_values():
    """A zero row stays zero, NaN and infinity stay in their row; channels that are not
    rotated do not meet the others."""
    q = torch.randn(5, 1, 64, generator=torch.Generator().manual_seed(4)).to(FP16).cuda()
    q[0] = 0
    q[1, 0, 3] = float("nan")
    q[2, 0, 60] = float("inf")
    q[3] = -0.0
    table, pos = K.rope_table(9, 32, device="cuda"), torch.arange(5, device="cuda")
    w = torch.ones(64, device="cuda")
    qo, _ = K.qk_norm_rope(q, q, pos, table, w, w)
    assert (qo[0] == 0).all() and qo[1].isnan().all() and not qo[[0, 3, 4]].isnan().any()
    qo, _ = K.qk_norm_rope(q, q, pos, table)
    assert qo[1].isnan().sum() == 2 and torch.isfinite(qo[2, 0, :60]).all() and qo[2, 0, 60] == float("inf")


def test_empty_calls():
    table = K.rope_table(9, 32, device="cuda")
    q = torch.zeros(0, 4, 64, dtype=FP16, device="cuda")
    qo, ko = K.qk_norm_rope(q, q, torch.zeros(0, dtype=torch.int64, device="cuda"), table)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 4, 64)


def test_norm_without_rotation_and_staged_sizes_in_place():
    """A table of no columns only normalises; many rows go through the staged form, also in place
    and with padding rows between."""
    g = torch.Generator().manual_seed(6)
    q = torch.randn(5, 3, 64, generator=g).to(BF16).cuda()
    w = torch.rand(64, generator=g).add(0.5).cuda()
    pos = torch.arange(5, device="cuda")
    none = torch.zeros(9, 0, device="cuda")
    qo, _ = K.qk_norm_rope(q, q, pos, none, w, w)
    close(qo, q, w, pos, none, 1e-6, False)
    n = 9000
    rows = torch.randn(n, 10 * 128, generator=g).to(FP16).cuda()
    x, y = rows[:, :1024].view(n, 8, 128), rows[:, 1024:].view(n, 2, 128)
    x0, y0 = x.clone(), y.clone()
    table = K.rope_table(n, 128, device="cuda")
    pos = torch.randint(0, n, (n,), generator=g)
    pos[torch.rand(n, generator=g) < 0.1] = -1
    pos = pos.cuda()
    w = torch.rand(128, generator=g).add(0.5).cuda()
    K.qk_norm_rope(x, y, pos, table, w, w, q_out=x, k_out=y)
    live = pos >= 0
    assert torch.equal(x[~live], x0[~live]) and torch.equal(y[~live], y0[~live])
    close(x[live], x0[live], w, pos[live], table, 1e-6, False)
    close(y[live], y0[live], w, pos[live], table, 1e-6, False)


def test_padding_between_staged_rows_again_and_again():
    """A row that is skipped leaves its copy in flight: the next copy to that place has to wait
    for it.  Half of the rows are padding, in runs of every length, and each call is checked."""
    g = torch.Generator().manual_seed(7)
    n = 12000
    x = torch.randn(n, 16, 128, generator=g).to(BF16).cuda()
    y = torch.randn(n, 4, 128, generator=g).to(BF16).cuda()
    table = K.rope_table(n, 128, device="cuda")
    pos = torch.randint(0, n, (n,), generator=g)
    want = K.qk_norm_rope(x, y, pos.cuda(), table)
    for i in range(20):
        some = pos.clone()
        some[torch.rand(n, generator=g) < 0.5] = -1
        some[i * 100:i * 100 + 5000] = -1
        live = (some >= 0).cuda()
        got = K.qk_norm_rope(x, y, some.cuda(), table)
        assert torch.equal(got[0][live], want[0][live]) and torch.equal(got[1][live], want[1][live])
