"""Plain model of the 8-bit paged cache for the tests: the quantisation formula in
float32 (what the codes are defined by) and attention, norm and rotation in float64."""

from __future__ import annotations

import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def quantise(block: torch.Tensor, code: torch.dtype):
    """Codes and scale of one head's block (G, D), 16-bit input."""
    x = block.float()
    top = x.abs().max()                       # NaN propagates
    top = torch.where(top < 2.0 ** -100, torch.tensor(2.0 ** -100, device=x.device), top)
    one, q = torch.ones_like(top), torch.full_like(top, QMAX[code])
    y = x * (one / top * q)
    if code == torch.int8:
        y = torch.nan_to_num(y.round(), nan=0.0).clamp(-127, 127)
    else:
        y = y.clamp(-448, 448)
    return y.to(code), top * (one / q)


class CacheModel:
    """A cache of ``slots`` slots whose pages are handed out in a shuffled order; the rows
    of every token are kept, so that what stands in the arrays can be worked out anew."""

    def __init__(self, slots, heads, dim, page, code, dtype, pages, table_width, seed=0, device="cuda", fill=None):
        self.g = torch.Generator().manual_seed(seed)
        self.slots, self.h, self.d, self.page, self.code, self.dtype = slots, heads, dim, page, code, dtype
        self.device = device
        kw = dict(device=device)
        self.key_codes = torch.zeros(pages, heads, page, dim, dtype=torch.int8, **kw).view(code)
        self.value_codes = torch.zeros(pages, heads, page, dim, dtype=torch.int8, **kw).view(code)
        self.key_scale = torch.zeros(pages, heads, **kw)
        self.value_scale = torch.zeros(pages, heads, **kw)
        self.tail_k = torch.zeros(slots, heads, page, dim, dtype=dtype, **kw)
        self.tail_v = torch.zeros(slots, heads, page, dim, dtype=dtype, **kw)
        if fill is not None:                  # what nobody may read
            self.tail_k.fill_(fill)
            self.tail_v.fill_(fill)
            self.key_scale.fill_(fill)
            self.value_scale.fill_(fill)
        self.table = torch.full((slots, table_width), -7, dtype=torch.int32)
        self.free = torch.randperm(pages, generator=self.g).tolist()
        self.rows = [([], []) for _ in range(slots)]          # per slot: lists of (H, D) key rows, value rows
        self.lengths = torch.zeros(slots, dtype=torch.int32)

    def new_rows(self, n, scale=1.0):
        """Random rows (n, H, D) with a few large channels, on the device."""
        x = torch.randn(n, self.h, self.d, generator=self.g)
        x[..., ::7] *= 5.0
        return (x * scale).to(self.dtype)

    def append(self, slot, k, v):
        """Note rows (n, H, D) (host) as the slot's next tokens and give their blocks pages."""
        have = int(self.lengths[slot])
        for b in range(have // self.page, (have + len(k)) // self.page):
            self.table[slot, b] = self.free.pop()
        self.rows[slot][0].extend(k.unbind(0))
        self.rows[slot][1].extend(v.unbind(0))
        self.lengths[slot] = have + len(k)

    def truth(self, slot):
        """(keys, values) of a slot as the cache stands for them: (H, T, D) float64."""
        out = []
        n, full = int(self.lengths[slot]), int(self.lengths[slot]) // self.page * self.page
        for x in self.rows[slot]:
            t = torch.stack(x, 1) if n else torch.zeros(self.h, 0, self.d, dtype=self.dtype)
            y = t.double()
            for b in range(0, full, self.page):
                for h in range(self.h):
                    c, s = quantise(t[h, b:b + self.page], self.code)
                    y[h, b:b + self.page] = c.double() * s.double()
            out.append(y)
        return out

    def fill_arrays(self):
        """Put every slot's tokens into the arrays directly (without the framework)."""
        for s in range(self.slots):
            n = int(self.lengths[s])
            for x, codes, scale, tail in ((self.rows[s][0], self.key_codes, self.key_scale, self.tail_k),
                                          (self.rows[s][1], self.value_codes, self.value_scale, self.tail_v)):
                if not n:
                    continue
                t = torch.stack(x, 1)
                full = n // self.page * self.page
                for b in range(n // self.page):
                    p = int(self.table[s, b])
                    for h in range(self.h):
                        c, sc = quantise(t[h, b * self.page:(b + 1) * self.page], self.code)
                        codes[p, h] = c.to(codes.device)
                        scale[p, h] = sc
                if n > full:
                    tail[s, :, :n - full] = t[:, full:].to(tail.device)

    def arrays(self, table=None):
        t = (self.table if table is None else table).to(self.device)
        return (t, self.key_codes, self.value_codes, self.key_scale, self.value_scale, self.tail_k, self.tail_v)

    def lens(self):
        return self.lengths.to(self.device)


def attention(q, keys, values, sm_scale=None):
    """q (Hq, D), keys / values (H, T, D) float64 -> out (Hq, D) and, for the error bound,
    sum p |v| (Hq, D) and the largest sum |q_i k_i| * sm_scale over the tokens (Hq, 1)."""
    hq, d = q.shape
    h, t, _ = keys.shape
    sc = 1 / math.sqrt(d) if sm_scale is None else sm_scale
    if t == 0:
        z = torch.zeros(hq, d, dtype=torch.float64)
        return z, z, torch.zeros(hq, 1, dtype=torch.float64)
    qq = q.double().view(h, hq // h, d)
    s = qq @ keys.transpose(1, 2) * sc
    p = torch.softmax(s, -1)
    mass = (qq.abs() @ keys.abs().transpose(1, 2)).amax(-1) * abs(sc)
    return (p @ values).reshape(hq, d), (p @ values.abs()).reshape(hq, d), mass.reshape(hq, 1)


def attention_tolerance(out, absum, mass, dtype):
    """Bound of |kernel - exact|.  A score is a sum of D <= 256 exact products in float32,
    off by at most 64 roundings (16 in an instruction's sum, up to 16 instructions and the
    factors, doubled) of 2^-23 of the sum of magnitudes; a weight by that, by the
    exponential's 2^-20, and for bf16 caches by its rounding to fp16, 2^-11.  The output
    moves by at most twice that of sum p |v| (numerator and denominator), and is rounded
    once: half a step, or half the smallest subnormal."""
    w = 64 * 2.0 ** -23 * mass + 2.0 ** -20 + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -21)
    return torch.finfo(dtype).eps / 2 * out.abs() + 2 * w * absum * (1 + torch.finfo(dtype).eps) + 2.0 ** -25


def norm_rope(x, weight, positions, table, eps, interleaved):
    """(rows, heads, D) -> float64 result and the magnitude its float32 error scales with."""
    y = x.double()
    if weight is not None:
        y = y / ((y ** 2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    r = table.shape[1] // 2
    c, s = table.double()[positions.long()][:, None, :r], table.double()[positions.long()][:, None, r:]
    z, mag = y.clone(), y.abs().clone()
    ia = torch.arange(r) * 2 if interleaved else torch.arange(r)
    ib = ia + (1 if interleaved else r)
    a, b = y[..., ia], y[..., ib]
    z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return z, mag
