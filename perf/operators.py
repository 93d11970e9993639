"""What the operators around the 8-bit cache are measured on.

Four operators: the per-head norm of queries and keys with the rotary embedding (``qk_norm_rope``), and the paged
cache of 8-bit codes with one scale per block of tokens and KV head: writing it (``write_kv8``), reading it back
(``read_kv8``) and decode attention over it (``paged_attention_kv8``).  The sizes are the framework's own: 32 or 64
query heads on 8 KV heads of 128 channels, 4096 tokens for the latency case, batches of 32 x 32768 and
16 x 131072 tokens, a batch of 256 mixed lengths; keys and values are N(0, 1) with 16 outlier channels per head
scaled by U(4, 10).
"""

import math
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
SMALLEST = 2.0 ** -100          # floor of a block's largest magnitude


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one sequence decodes one token: only the latency of the call counts
        dict(name="rope one token", op="rope", n=1, hq=32, h=8, d=128, rot=128, dtype="bf16", inter=False, norm=True,
             fused=True, max_pos=32768),
        # a decode step of a few hundred sequences, rotary on half of the channels, adjacent pairs
        dict(name="rope step 301", op="rope", n=301, hq=64, h=8, d=128, rot=64, dtype="fp16", inter=True, norm=True,
             fused=False, max_pos=131072),
        # a prefill of 32768 tokens straight from the rows of a fused projection
        dict(name="rope prefill 32768", op="rope", n=32768, hq=32, h=8, d=128, rot=128, dtype="bf16", inter=False,
             norm=True, fused=True, max_pos=32768),
        # a decode step of 256 sequences: one token each, a few blocks fill up and are quantised
        dict(name="write step 256", op="write", mode="step", n=256, new=1, ctx=1000, h=8, d=128, page=64, code="e4m3",
             dtype="bf16"),
        # prefill of 32 prompts of mixed lengths into empty slots
        dict(name="write prefill ragged", op="write", mode="prefill", n=32, new=4096, ctx=0, h=8, d=128, page=64,
             code="e4m3", dtype="bf16"),
        # chunked prefill: ragged chunks behind what is cached, written and read back for the prefill's attention
        dict(name="write and read chunk", op="write", mode="chunk", n=24, new=701, ctx=999, h=4, d=64, page=32,
             code="int8", dtype="fp16"),
        # one prefix of 4096 tokens and a bit, handed to another worker
        dict(name="read one prefix", op="read", n=1, tokens=4137, h=8, d=128, page=64, code="e4m3", dtype="bf16"),
        # a batch of 16 x 32K tokens read back
        dict(name="read 16 x 32K", op="read", n=16, tokens=32768, h=8, d=128, page=64, code="int8", dtype="fp16"),
        # one sequence of 4096 tokens and a bit: the latency case
        dict(name="attention one 4K", op="attention", n=1, tokens=4133, mixed=False, hq=32, h=8, d=128, page=64,
             code="e4m3", dtype="bf16"),
        # the throughput case: 32 sequences of 32K tokens
        dict(name="attention 32 x 32K", op="attention", n=32, tokens=32768, mixed=False, hq=32, h=8, d=128, page=64,
             code="e4m3", dtype="bf16"),
        # long contexts with 8 query heads on each KV head
        dict(name="attention 16 x 131K", op="attention", n=16, tokens=131071, mixed=False, hq=64, h=8, d=128, page=128,
             code="int8", dtype="fp16"),
        # continuous batching: 256 sequences from empty to 8192 tokens, small heads, small pages
        dict(name="attention 256 mixed", op="attention", n=256, tokens=8192, mixed=True, hq=40, h=8, d=64, page=32,
             code="e4m3", dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attention", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128, 128, 256, 96, 80])
    h = rng.choice([1, 2, 4, 8, 8])
    if op == "rope":
        hq = h * rng.choice([1, 3, 4, 5, 8])
        rot = rng.choice([d, d, d // 2 if d % 32 == 0 else d])
        n = _log(rng, 1, max(2, min(32768, 160_000_000 // ((hq + h) * d))))
        return dict(op="rope", n=n, hq=hq, h=h, d=d, rot=rot, dtype=dtype, inter=rng.random() < 0.4,
                    norm=rng.random() < 0.8, fused=rng.random() < 0.5, max_pos=_log(rng, 1000, 131072))
    page, code = rng.choice([32, 64, 64, 128, 256]), rng.choice(["e4m3", "int8"])
    if op == "write":
        mode = rng.choice(["step", "prefill", "chunk"])
        n = _log(rng, 1, 256 if mode == "step" else 32)
        new = 1 if mode == "step" else _log(rng, 2, max(4, min(4096, 60_000_000 // (n * h * d))))
        return dict(op="write", mode=mode, n=n, new=new, ctx=0 if mode == "prefill" else _log(rng, 10, 1000), h=h, d=d,
                    page=page, code=code, dtype=dtype)
    if op == "read":
        n = _log(rng, 1, 32)
        return dict(op="read", n=n, tokens=_log(rng, 1, max(4, min(32768, 250_000_000 // (n * h * d)))), h=h, d=d,
                    page=page, code=code, dtype=dtype)
    n = _log(rng, 1, 256)
    return dict(op="attention", n=n, tokens=_log(rng, 16, max(32, min(131072, 800_000_000 // (n * h * d)))),
                mixed=rng.random() < 0.5, hq=h * rng.choice([1, 2, 4, 4, 5, 7, 8, 16]), h=h, d=d, page=page, code=code,
                dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _outliers(g, h, d):
    """(h, d) factors: 16 of the channels of each head scaled by U(4, 10)."""
    f = torch.ones(h, d, device="cuda")
    at = torch.rand(h, d, generator=g, device="cuda").argsort(dim=1)[:, :16]
    return f.scatter_(1, at, 4 + 6 * torch.rand(h, 16, generator=g, device="cuda"))


def _rows(g, n, h, d, factors, dtype):
    return (torch.randn(n, h, d, generator=g, device="cuda") * factors).to(dtype)


def _quantise(x, code):
    """Codes and scales of blocks x (blocks, H, G, D) float32."""
    top = x.abs().amax((2, 3)).clamp(min=SMALLEST)
    y = x * (QMAX[code] / top)[:, :, None, None]
    y = y.round().clamp(-127, 127) if code == "int8" else y.clamp(-448, 448)
    return y.to(CODES[code]), top / QMAX[code]


def _spread(case):
    """Tokens of each sequence, in no order: of a mixed batch from none to the most, evenly in the logarithm; of
    chunks and prompts evenly from an eighth of the most."""
    n = case["n"]
    if case["op"] == "write":
        if case["mode"] == "step":
            return [1] * n
        return [max(1, case["new"] * (n + 7 * i) // (8 * n)) for i in range(1, n)] + [case["new"]]
    if not case.get("mixed"):
        return [case["tokens"]] * n
    return [int((case["tokens"] + 1.0) ** (i / n)) if i else 0 for i in range(n - 1)] + [case["tokens"]]


def _shuffled(g, values):
    x = torch.tensor(values, dtype=torch.int64)
    return x[torch.randperm(len(values), generator=g, device="cuda").cpu()]


def _cache(g, lengths, room, p, case, filled=True):
    """Pools of p pages, tails and a shuffled block table for sequences of ``lengths`` tokens with ``room`` more to
    come."""
    n, h, d, page, code, dtype = (case[k] for k in ("n", "h", "d", "page", "code", "dtype"))
    pages = (lengths + room) // page
    table = torch.full((n, max(1, int(pages.max()))), -1, dtype=torch.int32)
    order = torch.randperm(p, generator=g, device="cuda").to(torch.int32).cpu()
    table[torch.arange(table.shape[1])[None, :] < pages[:, None]] = order[:int(pages.sum())]
    s = {"table": table.cuda(), "lengths": lengths.to(torch.int32).cuda()}
    for x in ("key", "value"):
        factors = _outliers(g, h, d)
        codes = torch.zeros(p, h, page, d, dtype=torch.int8, device="cuda").view(CODES[code])
        scale = torch.zeros(p, h, device="cuda")
        step = max(1, (1 << 27) // (h * page * d))
        for a in range(0, p if filled else 0, step):
            b = min(p, a + step)
            codes[a:b], scale[a:b] = _quantise(
                torch.randn(b - a, h, page, d, generator=g, device="cuda") * factors[:, None, :], code)
        s[x + "_codes"], s[x + "_scale"] = codes, scale
        s["tail_" + x[0]] = (torch.randn(n, h, page, d, generator=g, device="cuda") * factors[:, None, :]).to(
            DTYPES[dtype])
        s[x + "_factors"] = factors
    return s


def prepare(case, seed):
    g = _gen(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    h, d, n = case["h"], case["d"], case["n"]
    if op == "rope":
        hq, rot = case["hq"], case["rot"]
        rows = torch.randn(n, (hq + 2 * h) * d, generator=g, device="cuda").to(dtype)
        q, k = rows[:, :hq * d].view(n, hq, d), rows[:, hq * d:(hq + h) * d].view(n, h, d)
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        angle = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        first = int(torch.randint(0, max(1, case["max_pos"] - n), (1,), generator=g, device="cuda"))
        # a prefill's positions follow one another, a step's are anywhere
        pos = first + torch.arange(n, device="cuda") if first + n <= case["max_pos"] and n > 4096 else torch.randint(
            0, case["max_pos"], (n,), generator=g, device="cuda")
        w = [1 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2)] if case["norm"] else [None, None]
        return {"op": op, "q": q, "k": k, "positions": pos.to(torch.int64), "table": torch.cat(
            [angle.cos(), angle.sin()], 1).float(), "wq": w[0] if w[0] is None else w[0].to(dtype),
            "wk": w[1] if w[1] is None else w[1].to(dtype), "inter": case["inter"], "eps": 1e-6}
    if op == "write":
        new = _shuffled(g, _spread(case))
        cached = torch.zeros(n, dtype=torch.int64)
        if case["mode"] != "prefill":
            cached = torch.randint(0, case["ctx"] + 1, (n,), generator=g, device="cuda").cpu()
        s = _cache(g, cached, new, max(1, sum((case["ctx"] + x) // case["page"] for x in _spread(case))), case, False)
        offsets = torch.zeros(n + 1, dtype=torch.int32)
        offsets[1:] = new.cumsum(0)
        total = int(offsets[-1])
        s.update(op=op, mode=case["mode"], key=_rows(g, total, h, d, s["key_factors"], dtype),
                 value=_rows(g, total, h, d, s["value_factors"], dtype), offsets=offsets.cuda(), most=int(new.max()),
                 rows=total, code=case["code"], after=(cached + new).to(torch.int32).cuda(),
                 first=cached.to(torch.int32).cuda())
        return s
    lengths = _shuffled(g, _spread(case))
    s = _cache(g, lengths, 0, max(1, sum(x // case["page"] for x in _spread(case))), case)
    s.update(op=op, code=case["code"])
    if op == "read":
        offsets = torch.zeros(n + 1, dtype=torch.int32)
        offsets[1:] = lengths.cumsum(0)
        s.update(offsets=offsets.cuda(), rows=int(offsets[-1]))
    else:
        s["q"] = torch.randn(n, case["hq"], d, generator=g, device="cuda").to(dtype)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _rotate(x, cos, sin, inter):
    r = cos.shape[-1]
    a, b, rest = (x[..., 0:2 * r:2], x[..., 1:2 * r:2], x[..., 2 * r:]) if inter else (
        x[..., :r], x[..., r:2 * r], x[..., 2 * r:])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1), rest], -1)


def _plain_rope(s):
    cos, sin = s["table"][s["positions"]][:, None, :].chunk(2, -1)

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w.float()
        return _rotate(y, cos, sin, s["inter"]).to(x.dtype)

    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _plain_write(s):
    """Every block that the new rows touch, gathered from the tails and the new rows for all sequences at once."""
    n, h, page, d = s["tail_k"].shape
    cached, offsets = s["lengths"].long(), s["offsets"].long()
    end = cached + offsets[1:] - offsets[:-1]
    block = cached[:, None] // page + torch.arange((s["most"] + page - 1) // page + 1, device="cuda")
    pos = block[:, :, None] * page + torch.arange(page, device="cuda")
    seq = torch.arange(n, device="cuda")[:, None, None].expand_as(pos)
    row = (offsets[:-1, None, None] + pos - cached[:, None, None]).clamp(0, s["rows"] - 1)
    full = (block + 1) * page <= end[:, None]
    fresh = (pos >= cached[:, None, None]) & (pos < end[:, None, None])
    left = fresh & ~full[:, :, None]
    to = s["table"].long()[seq[:, :, 0], block.clamp(max=s["table"].shape[1] - 1)][full]
    for x in ("key", "value"):
        tail = s["tail_" + x[0]]
        old = tail[seq[full], :, pos[full] % page]
        rows = torch.where(fresh[full][..., None, None], s[x][row[full]], old).float().transpose(1, 2)
        codes, scale = _quantise(rows, s["code"])
        s[x + "_codes"].view(torch.uint8)[to] = codes.view(torch.uint8)
        s[x + "_scale"][to] = scale
        tail[seq[left], :, pos[left] % page] = s[x][row[left]]


def _plain_read(s, lengths, first=None):
    n, _, page, _ = s["tail_k"].shape
    offsets = s["offsets"].long()
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), offsets[1:] - offsets[:-1], output_size=s["rows"])
    pos = torch.arange(s["rows"], device="cuda") - offsets[seq] + (0 if first is None else first.long()[seq])
    block = pos // page
    paged = ((block + 1) * page <= lengths.long()[seq])[:, None, None]
    at = s["table"].long()[seq, block.clamp(max=s["table"].shape[1] - 1)].clamp(min=0)

    def one(x):
        codes = s[x + "_codes"].view(torch.uint8)[at, :, pos % page].view(CODES[s["code"]]).float()
        tail = s["tail_" + x[0]]
        return torch.where(paged, (codes * s[x + "_scale"][at][..., None]).to(tail.dtype), tail[seq, :, pos % page])

    return one("key"), one("value")


def _plain_attention(s):
    q, table, lengths = s["q"], s["table"].long().clamp(min=0), s["lengths"].long()
    n, hq, d = q.shape
    _, h, page, _ = s["tail_k"].shape
    most = table.shape[1]

    def pages(x):    # (n, h, tokens, d) of all pages, in float32
        codes = s[x + "_codes"].view(torch.uint8)[table.flatten()].view(CODES[s["code"]]).float()
        codes *= s[x + "_scale"][table.flatten()][..., None, None]
        return codes.view(n, most, h, page, d).transpose(1, 2).reshape(n, h, most * page, d)

    qf = q.float().view(n, h, hq // h, d) / math.sqrt(d)
    scores = torch.cat([qf @ pages("key").transpose(2, 3), qf @ s["tail_k"].float().transpose(2, 3)], -1)
    t = torch.arange(most * page + page, device="cuda")
    full = (lengths // page * page)[:, None]
    there = torch.where(t < most * page, t < full, t - most * page < lengths[:, None] - full)[:, None, None]
    scores = torch.where(there, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = p[..., :most * page] @ pages("value") + p[..., most * page:] @ s["tail_v"].float()
    return torch.where(total > 0, out / total, 0.0).view(n, hq, d).to(q.dtype)


# ------------------------------------------------------------------------------------------------ one pass

def _kernels():
    if "kitty-kv_b200" not in sys.path:
        sys.path.insert(0, "kitty-kv_b200")
    from kitty import kernels
    return kernels


def _written(s):
    return {k: s[k] for k in ("key_codes", "value_codes", "key_scale", "value_scale", "tail_k", "tail_v")}


def run(s):
    op = s["op"]
    if own:
        K = _kernels()
        if op == "rope":
            return K.qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], s["wq"], s["wk"], eps=s["eps"],
                                  interleaved=s["inter"])
        pools = (s["table"], s["key_codes"], s["value_codes"], s["key_scale"], s["value_scale"], s["tail_k"],
                 s["tail_v"])
        if op == "write":
            K.write_kv8(s["key"], s["value"], s["lengths"], *pools,
                        row_offsets=None if s["mode"] == "step" else s["offsets"])
            if s["mode"] != "chunk":
                return _written(s)
            return K.read_kv8(s["after"], *pools, s["offsets"], s["rows"], first=s["first"])
        if op == "read":
            return K.read_kv8(s["lengths"], *pools, s["offsets"], s["rows"])
        return K.paged_attention_kv8(s["q"], s["lengths"], *pools)
    if op == "rope":
        return _plain_rope(s)
    if op == "write":
        _plain_write(s)
        return _written(s) if s["mode"] != "chunk" else _plain_read(s, s["after"], s["first"])
    if op == "read":
        return _plain_read(s, s["lengths"])
    return _plain_attention(s)


def work(case):
    h, d, n = case["h"], case["d"], case["n"]
    if case["op"] == "rope":
        x = n * (case["hq"] + h) * d
        return {"bytes": 4 * x + 4 * min(n, case["max_pos"]) * case["rot"], "flops": 7 * x}
    if case["op"] == "write":
        rows = sum(_spread(case)) * h * d * 2
        if case["mode"] == "chunk":      # read 2, write 1; the read back: 1 and 2
            return {"bytes": 6 * rows, "flops": 4 * rows}
        return {"bytes": (4 if case["mode"] == "step" else 3) * rows, "flops": 3 * rows}
    tokens = sum(_spread(case))
    if case["op"] == "read":
        return {"bytes": 6 * tokens * h * d, "flops": 2 * tokens * h * d}
    return {"bytes": 2 * tokens * h * d + 4 * n * case["hq"] * d, "flops": 4 * tokens * case["hq"] * d}


# ------------------------------------------------------------------------------------------------ in 64 bits

def _e4m3(x):
    """Nearest e4m3 value of float64 x (ties to even), saturating."""
    m, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_block(x, code):
    """Values that stand in the codes of one block (H, G, D) in float64, and the scales."""
    top = x.abs().flatten(1).max(1).values.clamp(min=SMALLEST)
    scale = top / QMAX[code]
    y = x / scale[:, None, None]
    return (torch.round(y).clamp(-127, 127) if code == "int8" else _e4m3(y)), scale


def _exact_rope(s):
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.double()
        if w is not None:
            y = y / ((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + s["eps"]).sqrt() * w.double()
        t = s["table"].double()[s["positions"]]
        half = t.shape[1] // 2
        z = y.clone()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if s["inter"] else (i, i + half)
            c, sn = t[:, i, None], t[:, half + i, None]
            z[..., a] = y[..., a] * c - y[..., b] * sn
            z[..., b] = y[..., b] * c + y[..., a] * sn
        out.append(z)
    return tuple(out)


def _exact_write(s):
    page = s["tail_k"].shape[2]
    r = {k: v.double() for k, v in _written(s).items()}
    back = {"key": [], "value": []}
    table, offsets, cached = s["table"].cpu(), s["offsets"].cpu().tolist(), s["lengths"].cpu().tolist()
    for i, c in enumerate(cached):
        have = c % page
        for x in ("key", "value"):
            t = "tail_" + x[0]
            rows = torch.cat([s[t][i, :, :have].double(), s[x][offsets[i]:offsets[i + 1]].double().transpose(0, 1)], 1)
            stored = rows.clone()
            blocks = rows.shape[1] // page
            for b in range(blocks):
                to = int(table[i, c // page + b])
                v, scale = _exact_block(rows[:, b * page:(b + 1) * page], s["code"])
                r[x + "_codes"][to], r[x + "_scale"][to] = v, scale
                stored[:, b * page:(b + 1) * page] = v * scale[:, None, None]
            keep = rows[:, blocks * page:]
            if keep.shape[1]:
                r[t][i, :, :keep.shape[1]] = keep
            back[x].append(stored[:, have:].transpose(0, 1))
    return r if s["mode"] != "chunk" else (torch.cat(back["key"]), torch.cat(back["value"]))


def _sequence(s, i, x):
    """(H, T, D) float64 keys or values of sequence i."""
    h, page, d = s["tail_k"].shape[1:]
    length = int(s["lengths"][i])
    pages = s["table"][i, :length // page].long()
    y = s[x + "_codes"].view(torch.uint8)[pages].view(CODES[s["code"]]).double()
    y = (y * s[x + "_scale"][pages].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(h, -1, d)
    return torch.cat([y, s["tail_" + x[0]][i, :, :length % page].double()], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rope":
        return _exact_rope(s)
    if s["op"] == "write":
        return _exact_write(s)
    n = case["n"]
    if s["op"] == "read":
        return tuple(torch.cat([_sequence(s, i, x).transpose(0, 1) for i in range(n)]) for x in ("key", "value"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(n):
        if int(s["lengths"][i]):
            q = s["q"][i].double().view(case["h"], -1, case["d"])
            z = q @ _sequence(s, i, "key").transpose(1, 2) * case["d"] ** -0.5
            w = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            out[i] = (w @ _sequence(s, i, "value")).reshape(out[i].shape)
    return out
