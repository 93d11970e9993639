"""GPU tests of what the 8-bit cache operators refuse of tensors on the device, before
anything is launched, and of the neighbouring calls that they take."""

from __future__ import annotations

import pytest
import torch

from kitty import kernels as K
from test_gpu_kv8 import BF16, E4M3, FP16, filled, i32

pytestmark = pytest.mark.gpu


def rope(q, k, **kw):
    n, d = q.shape[0], q.shape[2]
    return K.qk_norm_rope(q, k, torch.arange(n, device="cuda"), K.rope_table(n, d, device="cuda"), **kw)


@pytest.mark.parametrize("n", [1, 5, 3000])
def test_rope_outputs_that_overlap_are_refused(n):
    hq, h, d = 6, 2, 64
    flat = torch.randn((n + 2) * (hq + 2 * h) * d, device="cuda").to(BF16)
    rows = flat[:n * (hq + 2 * h) * d].view(n, -1)
    q, k = rows[:, :hq * d].view(n, hq, d), rows[:, hq * d:(hq + h) * d].view(n, h, d)
    v = rows[:, (hq + h) * d:].view(n, h, d)
    before = flat.clone()
    shifted = rows[:, d:(hq + 1) * d].view(n, hq, d)                       # a head further on: over q and k
    later = flat[(hq + 2 * h) * d:][:n * (hq + 2 * h) * d].view(n, -1)[:, :hq * d].view(n, hq, d)   # a token further on
    other = flat[:n * hq * d].view(n, hq, d)                               # q's memory with other strides
    bad = [dict(q_out=shifted), dict(k_out=q[:, :h]), dict(k_out=q[:, hq - h:]), dict(q_out=rows[:, 2 * h * d:].view(n, hq, d)),
           dict(q_out=torch.empty_like(q), k_out=shifted[:, -h:]), dict(k_out=rows[:, (hq - 1) * d + 8:(hq + h - 1) * d + 8].view(n, h, d))]
    both = torch.empty(n, hq + 1, d, dtype=BF16, device="cuda")
    bad.append(dict(q_out=both[:, :hq], k_out=both[:, hq - 1:]))
    if n > 1:
        bad += [dict(q_out=later), dict(q_out=other)]
    for kw in bad:
        with pytest.raises(RuntimeError, match="overlap"):
            rope(q, k, **kw)
    assert torch.equal(flat, before)
    want = rope(q, k)
    # the fused rows themselves, k's output in the place of v, outputs between one another
    got = rope(q, k, k_out=v)
    assert torch.equal(got[0], want[0]) and torch.equal(v, want[1])
    pair = torch.empty(n, h, 2, d, dtype=BF16, device="cuda")
    got = rope(k, k.clone(), q_out=pair[:, :, 0], k_out=pair[:, :, 1])
    assert torch.equal(pair[:, :, 0], want[1]) and torch.equal(pair[:, :, 1], want[1])
    got = rope(q, k, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v, want[1])


def test_rope_into_a_head_major_buffer_of_its_own_and_of_the_queries():
    n, h, d = 7, 4, 64
    q, k = (torch.randn(n, h, d, device="cuda").to(FP16) for _ in range(2))
    want = rope(q, k)
    out = torch.empty(2 * h, n, d, dtype=FP16, device="cuda")
    got = rope(q, k, q_out=out[:h].transpose(0, 1), k_out=out[h:].transpose(0, 1))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError, match="overlap"):
        rope(q, k, q_out=q.view(h, n, d).transpose(0, 1))


def test_read_and_attention_outputs_that_overlap_are_refused():
    m = filled([70, 33], 2, 64, 32, E4M3, BF16, seed=1)
    off = i32([0, 70, 103])
    buf = torch.zeros(2 * 103 - 1, 2, 64, dtype=BF16, device="cuda")
    for a, b in ((buf[:103], buf[:103]), (buf[:103], buf[102:]), (buf[102:], buf[:103])):
        with pytest.raises(RuntimeError, match="overlap"):
            K.read_kv8(m.lens(), *m.arrays(), off, 103, key_out=a, value_out=b)
    assert not buf.any()
    k, v = K.read_kv8(m.lens(), *m.arrays(), off, 103)
    buf = torch.zeros(206, 2, 64, dtype=BF16, device="cuda")
    K.read_kv8(m.lens(), *m.arrays(), off, 103, key_out=buf[:103], value_out=buf[103:])
    assert torch.equal(buf, torch.cat([k, v]))
    big = torch.randn(3, 8, 64, device="cuda").to(BF16)
    for q, out in ((big[:2], big[1:]), (big[:2, :6], big[:2, 2:]), (big[:2], big.view(-1)[:1024].view(8, 2, 64).transpose(0, 1)),
                   (big[:2, :4], big.view(-1)[:512].view(2, 4, 64))):
        with pytest.raises(RuntimeError, match="overlap"):
            K.paged_attention_kv8(q, m.lens(), *m.arrays(), out=out)
    want = K.paged_attention_kv8(big[:2, :4], m.lens(), *m.arrays())
    out = big[:2, 4:]
    assert K.paged_attention_kv8(big[:2, :4], m.lens(), *m.arrays(), out=out) is out and torch.equal(out, want)
    assert K.kv8_error_flags() == 0


def grad_cases():
    """(name, call of the tensors by name) of every operator; the tensors may be replaced."""
    m = filled([70, 33], 1, 64, 32, E4M3, FP16, seed=2)
    names = ("block_table", "key_codes", "value_codes", "key_scale", "value_scale", "tail_k", "tail_v")
    t = dict(zip(names, (x.clone() for x in m.arrays())), lengths=m.lens(), q=torch.randn(2, 2, 64).half().cuda(),
             k=torch.randn(2, 1, 64).half().cuda(), v=torch.randn(2, 1, 64).half().cuda(), wq=torch.ones(64).cuda(),
             wk=torch.ones(64).cuda(), table=K.rope_table(4, 64, device="cuda"), q_out=torch.empty(2, 2, 64).half().cuda(),
             k_out=torch.empty(2, 1, 64).half().cuda(), key_out=torch.empty(103, 1, 64).half().cuda(),
             value_out=torch.empty(103, 1, 64).half().cuda(), off=i32([0, 70, 103]), pos=i32([0, 1]))

    def cache(t):
        return (t["lengths"], *(t[n] for n in names))

    calls = {
        "rope": (lambda t: K.qk_norm_rope(t["q"], t["k"], t["pos"], t["table"], t["wq"], t["wk"], q_out=t["q_out"], k_out=t["k_out"]),
                 ("q", "k", "wq", "wk", "table", "q_out", "k_out"), ("q_out", "k_out")),
        "write": (lambda t: K.write_kv8(t["k"], t["v"], *cache(t)), ("k", "v", "key_scale", "value_scale", "tail_k", "tail_v"),
                  ("key_codes", "value_codes", "key_scale", "value_scale", "tail_k", "tail_v")),
        "read": (lambda t: K.read_kv8(*cache(t), t["off"], 103, key_out=t["key_out"], value_out=t["value_out"]),
                 ("key_scale", "value_scale", "tail_k", "tail_v", "key_out", "value_out"), ("key_out", "value_out")),
        "attention": (lambda t: K.paged_attention_kv8(t["q"], *cache(t), out=t["q_out"]),
                      ("q", "key_scale", "value_scale", "tail_k", "tail_v", "q_out"), ("q_out",))}
    return t, calls


@pytest.mark.parametrize("what", ["rope", "write", "read", "attention"])
def test_tensors_that_ask_for_derivatives_are_refused(what):
    import torch.autograd.forward_ad as fw
    t, calls = grad_cases()
    call, asks, written = calls[what]
    before = {n: x.view(torch.uint8).clone() for n, x in t.items()}
    for name in asks:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call({**t, name: t[name].detach().requires_grad_()})
        with fw.dual_level():
            dual = fw.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(RuntimeError, match="no forward derivative"):
                call({**t, name: dual})
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward derivative"):
                call({**t, name: dual})
    assert all(torch.equal(x.view(torch.uint8), before[n]) for n, x in t.items())
    with torch.no_grad():                                  # as with torch's own operators, in place too
        for name in asks:
            call({**t, name: t[name].detach().requires_grad_()})


@pytest.mark.parametrize("what", ["rope", "write", "read", "attention"])
def test_what_is_written_counts_as_changed(what):
    """A backward pass that saved what a call has since written raises; inference tensors are taken."""
    t, calls = grad_cases()
    call, _, written = calls[what]
    for name in written:
        if t[name].dtype == E4M3:
            v = t[name]._version
            call(t)
            assert t[name]._version > v
            continue
        x = torch.ones_like(t[name], requires_grad=True)
        y = (x * t[name]).sum()
        call(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    reads = {n: x._version for n, x in t.items() if n not in written}
    call(t)
    assert all(t[n]._version == v for n, v in reads.items())
    with torch.inference_mode():
        own = {n: x.clone() for n, x in t.items()}
        call(own)
    call(own)
    assert K.kv8_error_flags() == 0
