"""Performance cases of the operators that serve many utterances at once over
a key/value cache held in 4 bits: block tables and slot maps from request
lengths, the norms and rotation of queries and keys (with the new positions
stored into the cache in the same pass), and the attention that reads it.

A serving step is: tables for the step's rows, q|k|v of every layer's linear
map normed, rotated and stored, attention over the pages.  The cache of one
layer is pages of 64 positions; a page holds for each kv head a block of
72 D bytes (D the head's width, 32 values to a scale):

    K codes   [p % 4][p / 4][D / 2 bytes]     low nibble first
    V codes   [p / 4][D / 4][p % 4] 16 bits   four codes each, lowest first
    K scales  [D / 32][64] f16
    V scales  [D / 32][64] f16

and a value is (code - 8) * scale.  A scale has 8 significant bits, so a
value is exact in f16.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 64
EPS = 1e-6
MOST = 65280.0               # the largest magnitude that the format holds

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a streaming server's step: eight utterances, one new position each
        {"name": "tables_8_single", "op": "tables", "seqs": 8, "cached": 4000, "prompts": 0, "rows": 8},
        # a full server: most utterances one position on, every eighth brings a prompt
        {"name": "tables_515_mixed", "op": "tables", "seqs": 515, "cached": 4000, "prompts": 400, "rows": 32768},
        # one utterance's step in f32: the talker's 16 / 8 heads of 128
        {"name": "post_1_f32", "op": "post", "type": "f32", "rows": 1, "heads": 16, "kv_heads": 8, "dim": 128},
        # a batch of single positions
        {"name": "post_64_bf16", "op": "post", "type": "bf16", "rows": 64, "heads": 16, "kv_heads": 8, "dim": 128},
        # the prompts of a step together: cloned voices' reference rows
        {"name": "post_4001_bf16", "op": "post", "type": "bf16", "rows": 4001, "heads": 16, "kv_heads": 8, "dim": 128},
        # norm and rotation alone: a program with its own cache, heads of 64
        {"name": "norm_rope_1090_f16", "op": "norm", "type": "f16", "rows": 1090, "heads": 16, "kv_heads": 16, "dim": 64},
        # a single utterance's step early on, in f32
        {"name": "attend_1x300_f32", "op": "attend", "type": "f32", "seqs": 1, "length": 300, "fresh": 1,
         "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # a single long sequence
        {"name": "attend_1x16001_bf16", "op": "attend", "type": "bf16", "seqs": 1, "length": 16001, "fresh": 1,
         "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # a full server: utterances of all lengths up to the cache's capacity
        {"name": "attend_64x4096_bf16", "op": "attend", "type": "bf16", "seqs": 64, "length": 4096, "fresh": 1,
         "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # a few rows at a time: the first text rows of a chunk on kept prefixes
        {"name": "attend_16x700_5_f16", "op": "attend", "type": "f16", "seqs": 16, "length": 700, "fresh": 5,
         "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # cloned voices' prompts on kept prefixes
        {"name": "attend_4x2010_1000_bf16", "op": "attend", "type": "bf16", "seqs": 4, "length": 2010, "fresh": 1000,
         "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        # a sliding window over streamed chunks: the speech decoder's heads and window, in f32
        {"name": "attend_8x400_160_window_f32", "op": "attend", "type": "f32", "seqs": 8, "length": 400, "fresh": 160,
         "heads": 16, "kv_heads": 16, "dim": 64, "window": 72},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "post", "norm", "attend", "attend", "attend"])
    if op == "tables":
        seqs = _log_int(rng, 1, 515)
        prompts = rng.choice([0, 0, _log_int(rng, 2, 400)])
        return {"op": op, "seqs": seqs, "cached": _log_int(rng, 1, 4000), "prompts": prompts,
                "rows": min(32768, seqs + seqs * prompts // 8 + prompts + rng.randint(0, 300))}
    case = {"op": op, "type": rng.choice(["f32", "f16", "bf16"])}
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 16, 64), (8, 8, 128), (12, 4, 64), (10, 2, 64), (7, 1, 128)])
    if op != "attend":
        return {**case, "rows": _log_int(rng, 1, 2000 if case["type"] == "f32" else 4001), "heads": heads,
                "kv_heads": kv_heads, "dim": dim}
    fresh = rng.choice([1, 1, rng.randint(2, 9), _log_int(rng, 10, 1000)])
    most = 262144 if fresh < 10 else 8000             # positions in all
    seqs = _log_int(rng, 1, 64 if fresh < 10 else max(2, 4000 // fresh // 2))
    longest = max(fresh, min(16001 if fresh < 10 else 2010, most // seqs))
    return {**case, "seqs": seqs, "length": _log_int(rng, max(fresh, min(8, longest)), longest), "fresh": fresh, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": rng.choice([0, 0, 0, 72, 500])}


# ---------------------------------------------------------------------------
# lengths: of the case alone, so that what a pass has to move is known
# ---------------------------------------------------------------------------

def _spread(n, low, high):
    """n whole numbers between low and high, the last of them high, in no order."""
    r = random.Random(n * 1000003 + high)
    return [r.randint(min(low, high), high) for _ in range(n - 1)] + [high]


def _requests(case):
    """What each request has cached and brings: two lists."""
    n = case["seqs"]
    if case["op"] == "tables":
        cached = _spread(n, 0, case["cached"])
        fresh = [1] * n
        left = case["rows"] - n
        for b in range(0, n, 8):                       # every eighth brings a prompt, on nothing cached
            if case["prompts"] and left >= case["prompts"] - 1:
                cached[b], fresh[b] = 0, case["prompts"]
                left -= case["prompts"] - 1
        return cached, fresh
    fresh = [case["fresh"]] * n if case["fresh"] < 10 else _spread(n, (case["fresh"] + 1) // 2, case["fresh"])
    total = _spread(n, case["length"] // 3, case["length"])
    return [max(0, t - f) for t, f in zip(total, fresh)], fresh


def _pages(length):
    return -(-length // PAGE)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class State:
    pass


def _dev():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind).to(_dev())


def _tables_of(lengths, width, spare, g):
    """Scattered pages for sequences of these lengths: (table, the pages left)."""
    used = sum(_pages(n) for n in lengths)
    order = torch.randperm(used + spare, generator=g).to(torch.int32)
    table = torch.zeros((len(lengths), width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        table[b, :_pages(n)] = order[at:at + _pages(n)]
        at += _pages(n)
    return table.to(_dev()), order[used:].to(_dev())


def _rope(positions, dim):
    """cos and sin [positions][dim / 2] of the standard rotation, made in 64 bits."""
    freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cos(angle).float().to(_dev()), torch.sin(angle).float().to(_dev())


def _filled(pages, case, gd):
    """A layer's pages filled as by earlier steps: keys of unit rms with some
    strong channels, values a few times as large."""
    H, D = case["kv_heads"], case["dim"]
    out = torch.empty((pages, H, 72 * D), dtype=torch.uint8, device=_dev())
    strong = 1 + 3 * (torch.rand((H, 1, D), generator=gd, device=_dev()) < 0.05)
    for at in range(0, pages, 256):
        n = min(256, pages - at)
        k, v = (torch.randn((n, H, PAGE, D), generator=gd, device=_dev()) for _ in "kv")
        out[at:at + n] = _pack(_quantise((k * strong).double()), _quantise(4.0 * v.double()))
    return out


def prepare(case, seed):
    s = State()
    s.case = case
    g = torch.Generator().manual_seed(int(seed))
    gd = torch.Generator(device=_dev()).manual_seed(int(seed) + 1)
    if case["op"] == "tables":
        cached, fresh = _requests(case)
        width = max(_pages(c + n) for c, n in zip(cached, fresh)) + 2
        new = sum(_pages(c + n) - _pages(c) for c, n in zip(cached, fresh))
        s.table, s.free = _tables_of(cached, width, new + 5, g)
        s.cached, s.fresh = _ints(cached), _ints(fresh)
        return s
    H, HK, D, t = case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    if case["op"] == "attend":
        cached, fresh = _requests(case)
        lengths = [c + n for c, n in zip(cached, fresh)]
        s.longest = max(lengths)
        s.table, _ = _tables_of(lengths, _pages(s.longest) + 1, 3, g)
        s.pages = _filled(sum(_pages(n) for n in lengths) + 3, case, gd)
        s.lengths = _ints(lengths)
        s.row_start = _ints([0] + fresh).cumsum(0).to(torch.int32)
        s.most = max(fresh)
        s.q = (2 * torch.randn((sum(fresh), H, D), generator=gd, device=_dev())).to(t)
        return s
    rows = case["rows"]
    qkv = torch.randn((rows, (H + 2 * HK) * D), generator=gd, device=_dev()).to(t)     # a linear map's rows
    s.q, s.k, s.v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, HK * D, HK * D], dim=1))
    s.q_norm, s.k_norm = (1 + 0.2 * torch.randn(D, generator=gd, device=_dev()).half() for _ in "qk")
    s.cos, s.sin = _rope(8192, D)
    s.positions = torch.randint(0, 8192, (rows,), generator=g, dtype=torch.int32).to(_dev())
    if case["op"] == "post":
        pages = _pages(rows) + 3
        s.pages = torch.zeros((pages, HK, 72 * D), dtype=torch.uint8, device=_dev())
        s.slots = torch.randperm(pages * PAGE, generator=g)[:rows].to(_dev())
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _quantise(x):
    """x [..., D] in 64 bits: (codes [..., D], scales [..., D / 32] f16)."""
    g = x.clamp(-MOST, MOST).unflatten(-1, (-1, 32))
    high, low = g.amax(-1), g.amin(-1)
    d = (torch.where(high >= -low, high, low) * -0.125).float().half()
    d = ((d.view(torch.int16) + 4) & ~7).view(torch.float16)
    step = d.double()[..., None]
    codes = (torch.round(torch.where(step == 0, 0.0, g / step)) + 8).clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), d


def _values(codes, scales):
    return (codes.float().unflatten(-1, (-1, 32)) - 8) * scales.float()[..., None]


def _pack(k, v):
    """Blocks [..., 72 D] of 64 positions' codes and scales [..., 64, :]."""
    (kc, ks), (vc, vs) = k, v
    kb, vb = kc[..., 0::2] | kc[..., 1::2] << 4, vc[..., 0::2] | vc[..., 1::2] << 4
    kb = kb.unflatten(-2, (16, 4)).transpose(-3, -2)
    vb = vb.unflatten(-1, (-1, 2)).unflatten(-3, (16, 4)).transpose(-3, -2)
    scales = [s.transpose(-1, -2).contiguous().view(torch.uint8).flatten(-2) for s in (ks, vs)]
    return torch.cat([kb.flatten(-3), vb.flatten(-4)] + scales, dim=-1)


def _unpack(blocks):
    """Keys and values [..., 64, D] of blocks [..., 72 D], in 32 bits."""
    D = blocks.shape[-1] // 72
    kb, vb, ks, vs = blocks.split([32 * D, 32 * D, 4 * D, 4 * D], dim=-1)
    kb = kb.unflatten(-1, (4, 16, D // 2)).transpose(-3, -2).flatten(-3, -2)
    vb = vb.unflatten(-1, (16, D // 4, 4, 2)).transpose(-3, -2).flatten(-2).flatten(-3, -2)
    out = []
    for b, s in ((kb, ks), (vb, vs)):
        codes = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)
        out.append(_values(codes, s.contiguous().view(torch.float16).unflatten(-1, (-1, PAGE)).transpose(-1, -2)).flatten(-2))
    return out


def _plain_tables(s):
    rows, n = s.case["rows"], s.cached.shape[0]
    dev = s.cached.device
    lengths = s.cached + s.fresh
    ends = s.fresh.cumsum(0)
    row_start = torch.cat([ends.new_zeros(1), ends])
    old, all_ = (s.cached + PAGE - 1) // PAGE, (lengths + PAGE - 1) // PAGE
    first = (all_ - old).cumsum(0) - (all_ - old)
    column = torch.arange(s.table.shape[1], device=dev)
    take = (first[:, None] + column - old[:, None]).clamp(0, s.free.shape[0] - 1)
    fresh_page = (column >= old[:, None]) & (column < all_[:, None])
    s.table.copy_(torch.where(fresh_page, s.free[take], s.table))
    row = torch.arange(rows, device=dev)
    seq = torch.searchsorted(ends, row, right=True)
    used = seq < n
    seq = seq.clamp(max=n - 1)
    at = s.cached[seq] + row - row_start[seq]
    page = s.table[seq, (at // PAGE).clamp(0, s.table.shape[1] - 1)].long()
    return {"table": s.table, "row_start": row_start.int(), "lengths": lengths.int(),
            "positions": torch.where(used, at, -1).int(), "slots": torch.where(used, page * PAGE + at % PAGE, -1),
            "status": torch.stack([torch.zeros_like(ends[-1]), (all_ - old).sum()]).int()}


def _norm_rope(x, gamma, cos, sin):
    """Each head's row normed by its root mean square, then pairs (i, i + D / 2) rotated."""
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_norm(s):
    at = s.positions.long()
    cos, sin = s.cos[at][:, None], s.sin[at][:, None]
    q = _norm_rope(s.q.float(), s.q_norm.float(), cos, sin).to(s.q.dtype)
    if s.case["op"] == "norm":
        return {"q": q, "k": _norm_rope(s.k.float(), s.k_norm.float(), cos, sin).to(s.k.dtype)}
    # a code is decided where a value lies between two borders: in 64 bits
    kc, ks = _quantise(_norm_rope(s.k.double(), s.k_norm.double(), cos.double(), sin.double()))
    vc, vs = _quantise(s.v.double())
    D, page, p = s.case["dim"], s.slots // PAGE, s.slots % PAGE
    kb, vb = kc[..., 0::2] | kc[..., 1::2] << 4, vc[..., 0::2] | vc[..., 1::2] << 4
    b, vb2 = s.pages, vb.unflatten(-1, (-1, 2))
    b[..., :32 * D].unflatten(-1, (4, 16, D // 2))[page, :, p % 4, p // 4] = kb
    b[..., 32 * D:64 * D].unflatten(-1, (16, D // 4, 4, 2))[page, :, p // 4, :, p % 4] = vb2
    b[..., 64 * D:68 * D].unflatten(-1, (-1, PAGE, 2))[page, :, :, p] = ks[..., None].view(torch.uint8)
    b[..., 68 * D:].unflatten(-1, (-1, PAGE, 2))[page, :, :, p] = vs[..., None].view(torch.uint8)
    return {"q": q, "k": _values(kc, ks).flatten(-2).half(), "v": _values(vc, vs).flatten(-2).half()}


def _plain_attend(s):
    case = s.case
    n, H, HK, D, L = s.lengths.shape[0], case["heads"], case["kv_heads"], case["dim"], s.table.shape[1] * PAGE
    k, v = (x.transpose(1, 2).reshape(n, HK, L, D) for x in _unpack(s.pages[s.table.long()]))
    fresh = s.row_start[1:] - s.row_start[:-1]
    i = torch.arange(s.most, device=s.q.device)
    rows = (s.row_start[:-1, None] + i).clamp(max=s.q.shape[0] - 1).long()
    q = s.q[rows].float().unflatten(2, (HK, H // HK)).permute(0, 2, 3, 1, 4).reshape(n, HK, -1, D)
    score = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(D)).unflatten(2, (H // HK, -1))
    at, key = (s.lengths - fresh)[:, None] + i, torch.arange(L, device=s.q.device)
    hide = key > at[..., None]
    if case["window"]:
        hide = hide | (key <= at[..., None] - case["window"])
    score.masked_fill_(hide[:, None, None], -math.inf)
    p = torch.exp(score.sub_(score.amax(-1, keepdim=True)))
    out = (p.flatten(2, 3) @ v) / p.sum(-1).flatten(2, 3)[..., None]
    out = out.unflatten(2, (H // HK, -1)).permute(0, 3, 1, 2, 4).reshape(n, -1, H, D)
    return out[i < fresh[:, None]].to(s.q.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_made = []                   # the program's context


def _context():
    if not _made:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qora-tts-12hz-1.7b_amd"))
        import qtts
        _made.extend([qtts, qtts.Context(0, kv_capacity=64)])
    return _made


def run(s):
    case = s.case
    if not own:
        return {"tables": _plain_tables, "attend": _plain_attend}.get(case["op"], _plain_norm)(s)
    qtts, ctx = _context()
    if case["op"] == "tables":
        step = ctx.kv4_tables(s.cached, s.fresh, s.free, s.table, case["rows"])
        return {"table": s.table, "row_start": step.row_start, "lengths": step.lengths, "positions": step.positions,
                "slots": step.slots, "status": step.status}
    if case["op"] == "norm":
        q, k = ctx.qk_norm_rope(s.q, s.k, s.positions, s.cos, s.sin, s.q_norm, s.k_norm, EPS)
        return {"q": q, "k": k}
    cache = qtts.Kv4Cache(s.pages, case["kv_heads"], case["dim"])
    if case["op"] == "post":
        q, _ = ctx.qk_norm_rope(s.q, s.k, s.positions, s.cos, s.sin, s.q_norm, s.k_norm, EPS, v=s.v, cache=cache, slots=s.slots)
        k, v = ctx.kv4_gather(cache, s.slots, torch.float16)
        return {"q": q, "k": k, "v": v}
    return ctx.kv4_attention(s.q, cache, s.table, s.row_start, s.lengths, window=case["window"], max_len=s.longest)


# ---------------------------------------------------------------------------
# the least a pass has to move and compute
# ---------------------------------------------------------------------------

def _attended(cached, fresh, window):
    """(positions read, query and key pairs) of one request."""
    lowest = max(0, cached - window + 1) if window else 0
    pairs = sum(min(cached + i + 1, window or cached + i + 1) for i in range(fresh))
    return cached + fresh - lowest, pairs


def work(case):
    if case["op"] == "tables":
        cached, fresh = _requests(case)
        new = sum(_pages(c + n) - _pages(c) for c, n in zip(cached, fresh))
        return {"bytes": 16 * case["seqs"] + 8 * new + 12 * case["rows"] + 12, "flops": 0}
    H, HK, D = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["type"] == "f32" else 2
    row = 2 * HK * (D // 2 + D // 16)                  # a position's keys and values in 4 bits
    if case["op"] == "attend":
        both = [_attended(c, n, case["window"]) for c, n in zip(*_requests(case))]
        rows = sum(_requests(case)[1])
        return {"bytes": row * sum(b[0] for b in both) + 2 * rows * H * D * size, "flops": 4 * H * D * sum(b[1] for b in both)}
    rows = case["rows"]
    read = rows * ((H + HK) * D * size + 4 * D + 4)    # rows, their angles and positions
    if case["op"] == "norm":
        return {"bytes": read + rows * (H + HK) * D * size, "flops": 8 * rows * (H + HK) * D}
    # rows in, q out; codes and scales written, then read back as f16 values
    return {"bytes": read + rows * (HK * D * size + H * D * size + 8 + row + row + 8 + 2 * HK * D * 2),
            "flops": 8 * rows * (H + 2 * HK) * D}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------

def _held(x):
    """What the cache holds of x [..., D]: each 32 values on a grid of
    sixteen steps, -8 of them at the value of largest magnitude (the positive
    one of two), the step rounded to 8 significant bits."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], 32):
        part = x[..., g:g + 32]
        high, low = part.max(-1, keepdim=True).values, part.min(-1, keepdim=True).values
        step = -torch.where(high + low >= 0, high, low) / 8
        fraction, power = torch.frexp(step.float().half().double())
        unit = torch.exp2(power.double() - 8)
        step = torch.floor(torch.abs(fraction) * 256 + 0.5) * unit * torch.sign(fraction)
        out[..., g:g + 32] = torch.clamp(torch.round(part / step), -8, 7) * step
    return out


def _at(blocks, D):
    """Keys and values [..., 64, D] of blocks [..., 72 D], each found by its place."""
    p, d = torch.arange(PAGE, device=blocks.device)[:, None], torch.arange(D, device=blocks.device)[None]
    shift = 4 * (d % 2)
    out = []
    for at, scale in ((((p % 4) * 16 + p // 4) * (D // 2) + d // 2, 64 * D),
                      (32 * D + ((p // 4) * (D // 4) + d // 4) * 8 + (p % 4) * 2 + d % 4 // 2, 68 * D)):
        code = (blocks[..., at].int() >> shift) & 15
        where = scale + 2 * (d // 32 * PAGE + p)
        bits = blocks[..., where].int() | blocks[..., where + 1].int() << 8
        mantissa, power = bits & 1023, (bits >> 10) & 31
        size = torch.where(power == 0, mantissa.double() * 2.0 ** -24, (1024 + mantissa).double() * torch.exp2(power.double() - 25))
        out.append((code - 8).double() * torch.where(bits >= 32768, -size, size))
    return out


def _exact_heads(x, gamma, cos, sin):
    half = x.shape[-1] // 2
    x = x.double()
    x = gamma.double() * x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / (2 * half) + EPS)
    out = torch.empty_like(x)
    out[..., :half] = x[..., :half] * cos - x[..., half:] * sin
    out[..., half:] = x[..., half:] * cos + x[..., :half] * sin
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    D, H, HK = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] != "attend":
        cos, sin = (t[s.positions.long()].double()[:, None] for t in (s.cos, s.sin))
        q, k = _exact_heads(s.q, s.q_norm, cos, sin), _exact_heads(s.k, s.k_norm, cos, sin)
        return {"q": q, "k": k} if case["op"] == "norm" else {"q": q, "k": _held(k), "v": _held(s.v.double())}
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    starts, lengths, table = s.row_start.tolist(), s.lengths.tolist(), s.table.long()
    for b, length in enumerate(lengths):
        k, v = _at(s.pages[table[b, :_pages(length)]], D)
        q = s.q[starts[b]:starts[b + 1]].double()
        at = torch.arange(length - q.shape[0], length, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)[None]
        off = (key > at) | (key <= at - (case["window"] or length + 1))
        for h in range(H):
            kh, vh = (x[:, h // (H // HK)].reshape(-1, D)[:length] for x in (k, v))
            score = (q[:, h] @ kh.T.contiguous() / math.sqrt(D)).masked_fill(off, -math.inf)
            out[starts[b]:starts[b + 1], h] = torch.softmax(score, -1) @ vh
    return out
