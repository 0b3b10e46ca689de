"""The 4-bit cache's operators on the device against 64 bits (kv4_ref.py):
block tables, norms and rotation with the store, read-back, attention.

Codes and scales are compared exactly.  Error bounds of rows are derived where
they are used; a type's half step is EPS relative to the value.
"""
import threading

import numpy as np
import pytest
import torch

import kv4_ref
import qtts
from kv4_ref import PAGE, Pool

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx(ctx_factory):
    return ctx_factory(64)


def say(*a):
    print(*a, flush=True)


def dev(a, dtype=None):
    return torch.as_tensor(np.asarray(a)).to(DEV) if dtype is None else torch.as_tensor(np.asarray(a)).to(dtype).to(DEV)


def i32(a):
    return dev(a, torch.int32)


def host(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------

def run_tables(ctx, cached, fresh, rows, max_pages, spare=3, seed=0):
    r = np.random.default_rng(seed)
    held = [-(-c // PAGE) for c in cached]
    order = r.permutation(sum(held) + 4096 + spare).astype(np.int32)
    table = np.full((len(cached), max_pages), -7, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = order[at:]
    dt = i32(table)
    step = ctx.kv4_tables(i32(cached), i32(fresh), i32(free), dt, rows)
    return table, free, dt, step


@pytest.mark.parametrize("cached,fresh,rows", [
    ([0], [1], 1), ([0], [0], 0), ([0], [0], 5), ([], [], 3), ([63], [1], 4), ([64], [1], 1), ([64], [64], 64), ([1], [200], 300),
    ([5, 0, 64, 63, 128], [1, 0, 1, 2, 65], 80), ([0] * 7, [0, 64, 0, 0, 1, 130, 0], 195),
])
def test_tables_small(ctx, cached, fresh, rows):
    say("tables", cached, fresh, rows)
    table, free, dt, step = run_tables(ctx, cached, fresh, rows, 9)
    want = kv4_ref.tables(cached, fresh, free, table, rows)
    got = (dt, step.row_start, step.lengths, step.positions, step.slots, step.status)
    for g, w, name in zip(got, want, ("table", "row_start", "lengths", "positions", "slots", "status")):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel()), name
    assert step.check() == want[5][1]


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 1023, 1024, 1025, 4096])
def test_tables_many(ctx, seqs):
    say("tables", seqs)
    r = np.random.default_rng(seqs)
    cached = r.integers(0, 500, seqs).tolist()
    fresh = np.where(r.random(seqs) < 0.8, r.integers(0, 3, seqs), r.integers(0, 40, seqs)).tolist()
    rows = sum(fresh) + 1000
    table, free, dt, step = run_tables(ctx, cached, fresh, rows, 11, seed=seqs)
    want = kv4_ref.tables(cached, fresh, free, table, rows)
    for g, w in zip((dt, step.row_start, step.lengths, step.positions, step.slots, step.status), want):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel())


@pytest.mark.parametrize("cached,fresh,rows,free,code", [
    ([3, 4], [5, 6], 10, 5, qtts.ERR_CAPACITY),            # eleven rows, room for ten
    ([60, 64], [5, 6], 20, 1, qtts.ERR_CAPACITY),          # two pages, one free
    ([60, 64], [5, 700], 2000, 50, qtts.ERR_CAPACITY),     # more pages than columns
    ([3, -1], [5, 6], 20, 5, qtts.ERR_INVALID), ([3, 4], [5, -6], 20, 5, qtts.ERR_INVALID),
    ([2 ** 31 - 1, 4], [2 ** 31 - 1, 1], 20, 5, qtts.ERR_CAPACITY),
    ([2 ** 31 - 1, -4], [2 ** 31 - 1, 1], 20, 5, qtts.ERR_INVALID),
    ([0] * 3000, [2 ** 31 - 1] * 3000, 2 ** 12, 5, qtts.ERR_CAPACITY),
])
def test_tables_that_do_not_fit(ctx, cached, fresh, rows, free, code):
    n = len(cached)
    before = i32(np.arange(n * 9).reshape(n, 9))
    table = before.clone()
    step = ctx.kv4_tables(i32(cached), i32(fresh), i32(np.arange(free)), table, rows)
    assert step.status.tolist() == [code, 0]
    assert torch.equal(table, before)
    assert not step.row_start.any() and not step.lengths.any()
    assert bool((step.positions == -1).all()) and bool((step.slots == -1).all())
    with pytest.raises(qtts.QttsError) as e:
        step.check()
    assert e.value.code == code


def test_tables_strided_and_into_given_outputs(ctx):
    wide = i32(np.full((3, 20), -9))
    table = wide[:, 4:10]
    n, rows = 3, 12
    out = qtts.Kv4Step(*(torch.full((k,), 77, dtype=t, device=DEV) for k, t in
                         ((n + 1, torch.int32), (n, torch.int32), (rows, torch.int32), (rows, torch.int64), (2, torch.int32))))
    step = ctx.kv4_tables(i32([0, 0, 0]), i32([3, 4, 5]), i32([2 ** 31 - 1, 8, 9]), table, rows, out=out)
    assert step is out and step.check() == 3
    assert table[:, 0].tolist() == [2 ** 31 - 1, 8, 9] and int((wide == -9).sum()) == 57
    assert step.slots.tolist() == [(2 ** 31 - 1) * 64 + i for i in range(3)] + [8 * 64 + i for i in range(4)] + [9 * 64 + i for i in range(5)]


# ---------------------------------------------------------------------------
# norms, rotation, store and read-back
# ---------------------------------------------------------------------------

def rope_tables(n, D):
    ang = np.arange(n)[:, None] * 1e4 ** (-np.arange(0, D, 2) / D)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


class Post:
    """Inputs of one call as device views of a joint buffer, and in 64 bits."""

    def __init__(self, kind, rows, H, HK, D, seed=0, pad=0, shift=0, scale=1.0):
        r = np.random.default_rng(seed)
        width = (H + 2 * HK) * D + pad
        x = scale * r.standard_normal((rows, width))
        self.buf = torch.empty(rows * width + shift, dtype=TYPES[kind], device=DEV)[shift:].view(rows, width)
        self.buf.copy_(torch.as_tensor(x))
        cut = [0, H * D, (H + HK) * D, (H + 2 * HK) * D]
        self.q, self.k, self.v = (self.buf[:, a:b].unflatten(1, (-1, D)) for a, b in zip(cut, cut[1:]))
        self.qn, self.kn = ((1 + 0.3 * r.standard_normal(D)).astype(np.float16) for _ in "qk")
        cos, sin = rope_tables(200, D)
        self.pos = r.integers(0, 200, rows)
        self.cos, self.sin, self.c, self.s = dev(cos), dev(sin), cos.astype(np.float64), sin.astype(np.float64)

    def want(self, eps=1e-6, norm=True, rope=True):
        c, s = (self.c[self.pos], self.s[self.pos]) if rope else (None, None)
        return [kv4_ref.norm_rope(host(x), g.astype(np.float64) if norm else None, eps, c, s) for x, g in ((self.q, self.qn), (self.k, self.kn))]

    def args(self, norm=True, rope=True):
        a = {}
        if norm:
            a.update(q_norm=dev(self.qn), k_norm=dev(self.kn))
        if rope:
            a.update(positions=i32(self.pos), cos=self.cos, sin=self.sin)
        return a


def near(got, want, kind, D):
    """f32 arithmetic: a sum of D squares (relative D/2 2^-24 after the root), three
    products and a division a value (4 2^-24), then a difference of two products
    (3 2^-24 of their magnitudes, at most sqrt(2) times the pair's length), and
    one rounding to the type."""
    a, b = np.split(want, 2, -1)
    length = np.concatenate([np.hypot(a, b)] * 2, -1)
    tol = (D / 2 + 7) * 2.0 ** -24 * np.sqrt(2) * length + EPS[kind] * np.abs(want) * (1 + 1e-3) + (6e-8 if kind == "f16" else 0)
    err = np.abs(host(got) - want)
    assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-300)):.3f} of the bound"


HEADS = [(16, 8, 128), (16, 16, 64), (3, 1, 128), (10, 2, 64), (1, 1, 64), (7, 7, 128)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,HK,D", HEADS)
@pytest.mark.parametrize("rows", [1, 5, 131])
def test_norm_rope(ctx, kind, H, HK, D, rows):
    say("norm_rope", kind, H, HK, D, rows)
    p = Post(kind, rows, H, HK, D, seed=rows)
    q, k = ctx.qk_norm_rope(p.q, p.k, **p.args())
    for g, w in zip((q, k), p.want()):
        near(g, w, kind, D)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,HK,D", HEADS)
@pytest.mark.parametrize("rows", [1, 5, 131])
def test_store_and_gather(ctx, kind, H, HK, D, rows):
    say("store", kind, H, HK, D, rows)
    r = np.random.default_rng(rows)
    p = Post(kind, rows, H, HK, D, seed=rows)
    pages = rows // PAGE + 2
    pool = Pool(pages, HK, D, fill=0x3C)
    cache = qtts.Kv4Cache(dev(pool.b), HK, D)
    slots = r.permutation(pages * PAGE)[:rows]
    k_out = torch.empty_like(p.k.contiguous())
    q, k = ctx.qk_norm_rope(p.q, p.k, v=p.v, cache=cache, slots=dev(slots), k_out=k_out, **p.args())
    wq, wk = p.want()
    near(q, wq, kind, D)
    near(k, wk, kind, D)
    pool.put(slots, wk, host(p.v))
    assert np.array_equal(cache.pages.cpu().numpy(), pool.b)          # what no row touched included
    ask = np.concatenate([slots, [-1, pages * PAGE, 0]])
    for dt in TYPES.values():
        for g, w in zip(ctx.kv4_gather(cache, dev(ask), dt), pool.get(ask)):
            assert torch.equal(g.cpu(), torch.as_tensor(w).to(dt))


@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_parts_left_out(ctx, norm, rope, kind):
    p = Post(kind, 40, 4, 2, 64, seed=3)
    pool = Pool(1, 2, 64)
    cache = qtts.Kv4Cache(dev(pool.b), 2, 64)
    q, _ = ctx.qk_norm_rope(p.q, p.k, v=p.v, cache=cache, slots=dev(np.arange(40)), **p.args(norm, rope))
    wq, wk = p.want(norm=norm, rope=rope)
    near(q, wq, kind, 64)
    pool.put(np.arange(40), wk, host(p.v))
    assert np.array_equal(cache.pages.cpu().numpy(), pool.b)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 0), (4, 1), (5, 3)])
def test_in_place_at_any_alignment(ctx, kind, pad, shift):
    """Views of a joint buffer whose rows start anywhere, q and k in place; the
    columns between them and v stay as they were."""
    p = Post(kind, 33, 6, 2, 128, seed=pad, pad=pad, shift=shift)
    before = p.buf.clone()
    want = p.want()
    pool = Pool(1, 2, 128)
    cache = qtts.Kv4Cache(dev(pool.b), 2, 128)
    q, k = ctx.qk_norm_rope(p.q, p.k, v=p.v, cache=cache, slots=dev(np.arange(33)), q_out=p.q, k_out=p.k, **p.args())
    assert q.data_ptr() == p.q.data_ptr() and k.data_ptr() == p.k.data_ptr()
    near(q, want[0], kind, 128)
    near(k, want[1], kind, 128)
    assert torch.equal(p.buf[:, 8 * 128:], before[:, 8 * 128:])
    pool.put(np.arange(33), want[1], host(p.v))
    assert np.array_equal(cache.pages.cpu().numpy(), pool.b)


def test_rows_left_out_and_past_the_tables(ctx):
    p = Post("f32", 12, 4, 2, 128, seed=9)
    pos, slots = p.pos.copy(), np.arange(12)
    pos[[2, 11]] = -1
    pos[5] = 200                       # one past the tables
    pos[7] = 2 ** 31 - 1
    slots[3], slots[4] = -1, 64 * 2    # stored nowhere
    want = p.want()
    pool = Pool(2, 2, 128, fill=0x5A)
    cache = qtts.Kv4Cache(dev(pool.b), 2, 128)
    q_out, k_out = torch.full_like(p.q.contiguous(), 3.0), torch.full_like(p.k.contiguous(), 4.0)
    a = {**p.args(), "positions": i32(pos)}
    ctx.qk_norm_rope(p.q, p.k, v=p.v, cache=cache, slots=dev(slots), q_out=q_out, k_out=k_out, **a)
    q, k = host(q_out), host(k_out)
    assert (q[[2, 11]] == 3).all() and (k[[2, 11]] == 4).all()
    assert np.isnan(q[[5, 7]]).all() and np.isnan(k[[5, 7]]).all()
    rest = [0, 1, 3, 4, 6, 8, 9, 10]
    near(q_out[rest], want[0][rest], "f32", 128)
    near(k_out[rest], want[1][rest], "f32", 128)
    want[1][[5, 7]] = np.nan
    keep = [0, 1, 5, 6, 7, 8, 9, 10]
    pool.put(slots[keep], want[1][keep], host(p.v)[keep])
    k, v = (host(x) for x in ctx.kv4_gather(cache, dev(np.arange(128)), torch.float32))
    wk, wv = pool.get(np.arange(128))
    assert np.array_equal(k, wk, equal_nan=True) and np.array_equal(v, wv)
    assert np.isnan(k[[5, 7]]).all() and (v[[5, 7]] == 0).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_values_at_the_borders(ctx, kind):
    """Ties between steps, groups of zeros, tiny and huge magnitudes,
    infinities; NaN in either row of a head."""
    r = np.random.default_rng(4)
    x = r.integers(-16, 17, (64, 2, 2, 128)) / 2.0 * 2.0 ** r.integers(-3, 4, (64, 2, 2, 1))   # many quotients end in a half
    x[1] = 0
    x[2] = r.standard_normal((2, 2, 128)) * 2e-6
    x[3] = r.standard_normal((2, 2, 128)) * 1e-9
    x[4, :, :, :40] = 6e4
    x[5, :, :, 3] = np.inf
    x[6, :, :, 70] = -np.inf
    x[7, 0, 1, 9] = np.nan               # k of head 1
    x[8, 1, 0, 9] = np.nan               # v of head 0
    if kind != "f16":
        x[9] *= 1e30
        x[10] *= 1e-42 if kind == "f32" else 1e-36
    t = torch.as_tensor(x).to(TYPES[kind]).to(DEV)
    k, v = t[:, 0].contiguous(), t[:, 1].contiguous()
    pool = Pool(1, 2, 128)
    cache = qtts.Kv4Cache(dev(pool.b), 2, 128)
    ctx.qk_norm_rope(torch.zeros_like(k), k, v=v, cache=cache, slots=dev(np.arange(64)))
    pool.put(np.arange(64), host(k), host(v))
    got, want = ctx.kv4_gather(cache, dev(np.arange(64)), torch.float32), pool.get(np.arange(64))
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w, equal_nan=True)
    assert np.isnan(host(got[0])[7, 1]).all() and not np.isnan(host(got[0])[7, 0]).any() and (host(got[1])[8, 0] == 0).all()


def test_values_next_to_a_half(ctx):
    """Halves between codes, exactly and by one f32 step either way, for scales
    of 8 bits and either sign."""
    r = np.random.default_rng(5)
    d = (r.integers(128, 256, (64, 2, 2, 4, 1)) * 2.0 ** r.integers(-12, 4, (64, 2, 2, 4, 1)) * r.choice([-1, 1], (64, 2, 2, 4, 1)))
    x = (d * (r.integers(-15, 16, (64, 2, 2, 4, 32)) / 2)).astype(np.float32)
    x = np.nextafter(x, x + r.integers(-1, 2, x.shape).astype(np.float32), dtype=np.float32)
    x[..., :1] = -8 * d                  # the extreme: code 0
    x = x.reshape(64, 2, 2, 128).astype(np.float64)
    t = torch.as_tensor(x).to(torch.float32).to(DEV)
    k, v = t[:, 0].contiguous(), t[:, 1].contiguous()
    pool = Pool(1, 2, 128)
    cache = qtts.Kv4Cache(dev(pool.b), 2, 128)
    ctx.qk_norm_rope(torch.zeros_like(k), k, v=v, cache=cache, slots=dev(np.arange(64)))
    pool.put(np.arange(64), host(k), host(v))
    for g, w in zip(ctx.kv4_gather(cache, dev(np.arange(64)), torch.float32), pool.get(np.arange(64))):
        assert np.array_equal(host(g), w)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

class Served:
    """A pool with sequences of these lengths on scattered pages."""

    def __init__(self, lengths, HK, D, seed=0, columns=None, fill=0xFF, spread=1.0):
        r = np.random.default_rng(seed)
        held = [-(-n // PAGE) for n in lengths]
        ids = r.permutation(sum(held) + 2)
        self.pool = Pool(sum(held) + 2, HK, D, fill=fill)       # 0xFF: every scale nobody stored is NaN
        self.table = np.full((len(lengths), columns or max(held + [1])), -1, np.int64)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = ids[at:at + n]
            at += n
            slots = [self.table[b, p // PAGE] * PAGE + p % PAGE for p in range(lengths[b])]
            self.pool.put(slots, spread * r.standard_normal((lengths[b], HK, D)), 3 * r.standard_normal((lengths[b], HK, D)))
        self.lengths, self.HK, self.D = lengths, HK, D
        self.cache = qtts.Kv4Cache(dev(self.pool.b), HK, D)


def bound(kind, want, mag, big, lengths):
    """How far a row may be off.  A score is a sum of at most 128 exact products
    in f32 (128 2^-24 of their magnitudes `big`; f32 queries are held to 2^-22 of
    the row's largest) and is scaled and shifted (4 2^-24); exp2 and the log2 factor
    add 2^-21; so a weight is off by d relative to its own size.  Weights enter the
    product with V rounded to f16 (2^-11), or to two f16 (2^-22) for f32 rows; sums of
    weights and products in f32 run over at most pages + 96 additions in a row.
    Numerator and denominator each carry these: twice.  A weight is held as f16 at
    2^14 (f32 rows) or 2^9 times its share of a weight that is at most the largest, so
    one below f16's smallest normal is off by half of the subnormal step 2^-24: 2^-39 or
    2^-34 of the largest weight, for each key.  Then the type's rounding."""
    d = (128 * 2.0 ** -24 + (2.0 ** -22 if kind == "f32" else 0) + 4 * 2.0 ** -24) * big + 2.0 ** -21
    w = 2.0 ** -22 if kind == "f32" else 2.0 ** -11
    chain = (96 + max(lengths) / 64) * 2.0 ** -24
    return 2 * (d[..., None] + w + chain) * mag[..., 0] + 2.0 ** (-39 if kind == "f32" else -34) * mag[..., 1] + EPS[kind] * np.abs(want) * 1.001 + (6e-8 if kind == "f16" else 0)


def off_rms(kind, big):
    """What errors that do not all point one way come to: the same roundings, as a
    root of their number, times four."""
    d = (np.sqrt(128) * 2.0 ** -24) * big.mean() + 2.0 ** -21
    return 4 * (d + (2.0 ** -22 if kind == "f32" else 2.0 ** -11) + EPS[kind])


def attend(ctx, sv, fresh, H, kind, scale=None, window=0, pad=0, shift=0, extra=0, out=None, seed=1, max_len=None, qscale=1.0, check=True):
    """One call, compared with 64 bits; the output."""
    r = np.random.default_rng(seed)
    rows = sum(fresh) + extra
    width = H * sv.D + pad
    q = torch.empty(rows * width + shift, dtype=TYPES[kind], device=DEV)[shift:].view(rows, width)
    q.copy_(torch.as_tensor(qscale * r.standard_normal((rows, width))))
    q = q[:, :H * sv.D].unflatten(1, (H, sv.D))
    row_start = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int64)
    scale = sv.D ** -0.5 if scale is None else scale
    got = ctx.kv4_attention(q, sv.cache, i32(sv.table), i32(row_start), i32(sv.lengths), scale=scale, window=window, max_len=max_len, out=out)
    if check:
        want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, row_start, sv.lengths, np.float64(np.float32(scale)), window)
        n = sum(fresh)
        compare(host(got)[:n], want[:n], mag[:n], big[:n], kind, sv.lengths)
    return got


def compare(got, want, mag, big, kind, lengths):
    if not want.size:
        return
    tol, err = bound(kind, want, mag, big, lengths), np.abs(got - want)
    assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-300)):.3g} of the bound at {np.unravel_index(np.argmax(err / np.maximum(tol, 1e-300)), err.shape)}"
    if np.abs(want).max() > 0:
        rms = np.sqrt((err ** 2).mean() / (mag[..., 0] ** 2).mean())
        assert rms <= off_rms(kind, big), f"rms {rms:.3g} of the weighted values, expected below {off_rms(kind, big):.3g}"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,HK,D", HEADS + [(40, 2, 64), (17, 1, 128)])
def test_attention_single_tokens(ctx, kind, H, HK, D):
    lengths = [1, 63, 64, 65, 200, 2, 129]
    say("attention single", kind, H, HK, D)
    attend(ctx, Served(lengths, HK, D, seed=H), [1] * len(lengths), H, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("window", [0, 1, 72, 64])
@pytest.mark.parametrize("H,HK,D", [(4, 2, 128), (3, 3, 64), (10, 2, 64)])
def test_attention_ragged(ctx, kind, window, H, HK, D):
    """Prompts, parts of prompts, single rows, none, and sequences that are
    empty, in one call; rows behind the last sequence stay."""
    lengths, fresh = [90, 0, 64, 130, 1, 33, 70], [90, 0, 1, 9, 1, 0, 70]
    say("attention ragged", kind, window, H, HK, D)
    out = torch.full((sum(fresh) + 6, H, D), 5.0, dtype=TYPES[kind], device=DEV)
    attend(ctx, Served(lengths, HK, D, seed=window), fresh, H, kind, window=window, extra=6, out=out)
    assert bool((out[sum(fresh):] == 5).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("length", [4096, 1000])
def test_attention_long(ctx, kind, length):
    say("attention long", kind, length)
    attend(ctx, Served([length], 1, 128, seed=5), [3], 2, kind)


def test_max_len_is_only_a_hint(ctx):
    sv = Served([700, 40], 2, 128, seed=6)
    for hint in (0, 1, 64, 700, 10 ** 9):
        attend(ctx, sv, [2, 1], 4, "f32", max_len=hint)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_prompt_rows(ctx, kind):
    """Many rows a sequence: every tile of the prompt path, ends inside tiles."""
    say("attention prompt", kind)
    attend(ctx, Served([150, 257, 131], 1, 128, seed=7), [150, 131, 128], 2, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,shift", [(3, 0), (0, 1), (8, 4)])
def test_attention_any_alignment_in_place(ctx, kind, pad, shift):
    sv = Served([77, 5], 2, 64, seed=8)
    attend(ctx, sv, [3, 2], 4, kind, pad=pad, shift=shift)
    q = torch.randn((5, 4, 64), generator=torch.Generator().manual_seed(1)).to(TYPES[kind]).to(DEV)
    args = (sv.cache, i32(sv.table), i32([0, 3, 5]), i32(sv.lengths))
    apart = ctx.kv4_attention(q, *args)
    assert torch.equal(ctx.kv4_attention(q, *args, out=q), apart) and torch.equal(q, apart)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale,qscale", [(-0.3, 1.0), (1e-4, 1.0), (3.0, 2.0), (1e-3, 1e4), (1e6, 1e-6)])
def test_attention_scales(ctx, kind, scale, qscale):
    """Sharp and flat softmaxes, and query rows far from 1 (f16 ones in its
    range)."""
    if kind == "f16":
        qscale = max(qscale, 1e-3)
    say("scales", kind, scale, qscale)
    attend(ctx, Served([150], 1, 64, seed=9), [2], 2, kind, scale=scale, qscale=qscale)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,H", [(5, 6), (180, 120), (420, 120)])
def test_attention_query_without_a_value(ctx, kind, rows, H):
    """NaN and infinite query values: NaN for their row and head, and only there."""
    sv = Served([430], 1, 64, seed=60)
    q = torch.randn((rows, H, 64), generator=torch.Generator().manual_seed(9)).to(TYPES[kind]).to(DEV)
    args = (sv.cache, i32(sv.table), i32([0, rows]), i32([430]))
    want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, [0, rows], [430], 0.125, 0)
    q[1, 2, 5], q[rows - 1, 0, 63], q[3, 5, 0] = float("nan"), float("inf"), -float("inf")
    got, bad = host(ctx.kv4_attention(q, *args)), np.zeros((rows, H), bool)
    bad[[1, rows - 1, 3], [2, 0, 5]] = True
    assert np.isnan(got[bad]).all()
    compare(got[~bad], want[~bad], mag[~bad], big[~bad], kind, [430])


def test_attention_more_rows_than_positions(ctx):
    """Rows whose position lies before the sequence see nothing: zero."""
    sv = Served([3, 0], 2, 64, seed=10)
    got = attend(ctx, sv, [5, 2], 4, "f32")
    assert not got[:2].any() and got[2:5].any(dim=-1).all() and not got[5:].any()


def test_attention_nan_in_masked_positions(ctx):
    """A NaN in a later position, and whatever lies behind the sequence or
    before the window, does not reach the rows that do not see it; the rows
    that do are NaN."""
    sv = Served([100], 1, 64, seed=11)
    slot = lambda p: sv.table[0][p // PAGE] * PAGE + p % PAGE
    k, v = sv.pool.get([slot(p) for p in (60, 10)])
    v[:] = np.nan
    sv.pool.put([slot(60), slot(10)], k, v)
    sv.cache.pages.copy_(torch.as_tensor(sv.pool.b))
    for fresh, window in ((50, 0), (50, 20)):
        q = torch.randn((fresh, 2, 64), generator=torch.Generator().manual_seed(2)).to(DEV)
        got = host(ctx.kv4_attention(q, sv.cache, i32(sv.table), i32([0, fresh]), i32([100]), window=window))
        want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, [0, fresh], [100], np.float64(np.float32(1 / 8)), window)
        bad = np.isnan(want).any(-1)
        assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
        assert 0 < bad.sum() <= bad.size and (window == 0 or not bad.all())
        if not bad.all():
            compare(got[~bad], want[~bad], mag[~bad], big[~bad], "f32", [100])


@pytest.mark.parametrize("entry", [-1, 1000, 2 ** 31 - 1, -2 ** 31])
def test_attention_bad_pages(ctx, entry):
    """A table entry outside the pool: NaN for the rows that see the page and
    for no other; one that no row sees is not read."""
    sv = Served([200, 70], 1, 64, seed=12)
    table = sv.table.copy()
    table[0, 2] = entry                  # positions 128 .. 191
    table[1, 2:] = entry                 # past the sequence
    q = torch.randn((102, 2, 64), generator=torch.Generator().manual_seed(3)).to(DEV)
    row_start = [0, 100, 102]            # positions 100 .. 199 and 68, 69
    for window in (0, 10):
        got = host(ctx.kv4_attention(q, sv.cache, i32(table), i32(row_start), i32([200, 70]), window=window))
        want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, row_start, [200, 70], np.float64(np.float32(1 / 8)), window)
        pos = np.arange(100, 200)
        sees = (pos >= 128) & ((window == 0) | (pos - window < 191))
        assert np.isnan(got[:100][sees]).all()
        ok = np.concatenate([~sees, [True, True]])
        compare(got[ok], want[ok], mag[ok], big[ok], "f32", [200])


def test_attention_short_table_and_bad_sums(ctx):
    """A length beyond the table's columns is NaN where it is seen; row sums
    that are none leave everything as it was."""
    sv = Served([64], 1, 64, seed=13, columns=1)
    q = torch.randn((2, 2, 64), generator=torch.Generator().manual_seed(4)).to(DEV)
    got = ctx.kv4_attention(q, sv.cache, i32(sv.table), i32([0, 2]), i32([65]))
    assert not torch.isnan(got[0]).any() and torch.isnan(got[1]).all()
    for row_start, length in (([0, 3], 64), ([2, 0], 64), ([-5, 1], 64), ([0, 2], -1), ([0, 2], 2 ** 31 - 1), ([2 ** 31 - 1, 2 ** 31 - 1], 64)):
        out = torch.full_like(q, 9.0)
        ctx.kv4_attention(q, sv.cache, i32(sv.table), i32(row_start), i32([length]), out=out)
        assert bool((out == 9).all())


def test_attention_no_rows_and_no_sequences(ctx):
    sv = Served([10], 2, 64, seed=14)
    q = torch.empty((0, 4, 64), device=DEV)
    assert ctx.kv4_attention(q, sv.cache, i32(sv.table), i32([0, 0]), i32([10])).shape == (0, 4, 64)
    q, out = torch.zeros((2, 4, 64), device=DEV), torch.full((2, 4, 64), 2.0, device=DEV)
    ctx.kv4_attention(q, sv.cache, i32(np.zeros((0, 1))), i32([0]), i32([]), out=out)
    assert bool((out == 2).all())


# More than 48 columns a sequence and 16384 in all (f32: 64 and 20480) take
# tiles of 128 columns.

# sequences, rows of each, query heads, kv heads, head width
WIDE = [([150, 257, 131], [150, 131, 128], 51, 1, 128),           # 165 tiles: two groups of waves a tile
        ([300, 0, 64, 200], [190, 0, 1, 180], 60, 2, 64),
        ([400, 450], [400, 400], 66, 2, 128),                    # 414 tiles: one
        ([65, 500, 129], [65, 480, 1], 98, 1, 64)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("window", [0, 72])
@pytest.mark.parametrize("lengths,fresh,H,HK,D", WIDE)
def test_attention_wide_tiles(ctx, kind, window, lengths, fresh, H, HK, D):
    say("wide", kind, window, lengths, H, HK, D)
    out = torch.full((sum(fresh) + 3, H, D), 5.0, dtype=TYPES[kind], device=DEV)
    attend(ctx, Served(lengths, HK, D, seed=H), fresh, H, kind, window=window, extra=3, out=out, pad=3 if window else 0)
    assert bool((out[sum(fresh):] == 5).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_wide_tiles_split(ctx, kind):
    """Pages past a workgroup's 128 go to others; the short sequence beside is
    not split."""
    say("wide split", kind)
    attend(ctx, Served([8700, 50], 1, 64, seed=30), [70, 50], 180, kind)


@pytest.mark.parametrize("rows", [180, 420])
def test_attention_wide_tiles_sharp_and_flat(ctx, rows):
    for scale in (-0.5, 1e-4, 3.0):
        say("wide", rows, scale)
        attend(ctx, Served([420], 1, 64, seed=31), [rows], 120, "f32", scale=scale)


@pytest.mark.parametrize("rows", [180, 420])
@pytest.mark.parametrize("entry", [-1, 2 ** 31 - 1])
def test_attention_wide_tiles_bad_pages(ctx, rows, entry):
    """NaN for the rows that see the page, and for no other."""
    say("wide bad page", rows, entry)
    sv = Served([420], 1, 64, seed=32)
    table = sv.table.copy()
    table[0, 5] = entry                  # positions 320 .. 383
    q = torch.randn((rows, 120, 64), generator=torch.Generator().manual_seed(3)).to(DEV)
    pos = np.arange(420 - rows, 420)
    for window in (0, 10):
        got = host(ctx.kv4_attention(q, sv.cache, i32(table), i32([0, rows]), i32([420]), window=window))
        want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, [0, rows], [420], np.float64(np.float32(1 / 8)), window)
        sees = (pos >= 320) & ((window == 0) | (pos - window < 383))
        assert np.isnan(got[sees]).all() and sees.any() and not sees.all()
        compare(got[~sees], want[~sees], mag[~sees], big[~sees], "f32", [420])


@pytest.mark.parametrize("rows,HK", [(180, 1), (450, 1)])
def test_attention_wide_tiles_nan_and_empty_rows(ctx, rows, HK):
    """Rows before the sequence are zero; a NaN in a position reaches the rows
    that see it."""
    sv = Served([130], HK, 64, seed=33)
    slot = lambda p: sv.table[0][p // PAGE] * PAGE + p % PAGE
    k, v = sv.pool.get([slot(70)])
    v[:] = np.nan
    sv.pool.put([slot(70)], k, v)
    sv.cache.pages.copy_(torch.as_tensor(sv.pool.b))
    q = torch.randn((rows, 120, 64), generator=torch.Generator().manual_seed(2)).to(DEV)
    for window in (0, 20):
        got = host(ctx.kv4_attention(q, sv.cache, i32(sv.table), i32([0, rows]), i32([130]), window=window))
        want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, [0, rows], [130], np.float64(np.float32(1 / 8)), window)
        bad = np.isnan(want).any(-1)
        assert bad.any() and not bad.all() and np.array_equal(np.isnan(got).all(-1), bad)
        assert (got[:rows - 130] == 0).all()
        compare(got[~bad], want[~bad], mag[~bad], big[~bad], "f32", [130])


def test_attention_wide_tiles_short_table_and_bad_sums(ctx):
    sv = Served([128], 1, 64, seed=34, columns=2)
    q = torch.randn((180, 120, 64), generator=torch.Generator().manual_seed(4)).to(DEV)
    got = ctx.kv4_attention(q, sv.cache, i32(sv.table), i32([0, 180]), i32([130]))
    assert not torch.isnan(got[:178]).any() and torch.isnan(got[178:]).all()
    for row_start, length in (([0, 181], 64), ([180, 0], 64), ([-5, 180], 64), ([0, 180], -1), ([0, 180], 2 ** 31 - 1)):
        out = torch.full_like(q, 9.0)
        ctx.kv4_attention(q, sv.cache, i32(sv.table), i32(row_start), i32([length]), out=out)
        assert bool((out == 9).all())


def test_many_sequences_find_their_tiles(ctx):
    """4097 sequences, some without rows: every row must find its own."""
    r = np.random.default_rng(15)
    n = 4097
    fresh = r.integers(0, 4, n)
    pool = Pool(70, 1, 64)
    slots = np.arange(70 * PAGE)
    pool.put(slots, r.standard_normal((len(slots), 1, 64)), np.repeat(np.arange(70.0) + 1, PAGE)[:, None, None] * np.ones((1, 1, 64)))
    cache = qtts.Kv4Cache(dev(pool.b), 1, 64)
    table = r.integers(0, 70, (n, 1))
    q = torch.randn((int(fresh.sum()), 2, 64), generator=torch.Generator().manual_seed(5)).to(DEV)
    got = host(ctx.kv4_attention(q, cache, i32(table), i32(np.concatenate([[0], np.cumsum(fresh)])), i32(np.full(n, 30))))
    held = pool.get(np.arange(70) * PAGE)[1][:, 0, 0]
    want = held[table[np.repeat(np.arange(n), fresh), 0]][:, None, None]      # constant values: the average is the value
    assert (np.abs(got - want) <= want * 2.0 ** -21).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,HK,window", [(16, 8, 0), (21, 7, 40)])
def test_attention_more_workgroups_than_cus(ctx, kind, H, HK, window):
    """Heads of 128 on four waves a tile."""
    say("many", kind, H, HK, window)
    r = np.random.default_rng(H)
    lengths = r.integers(0, 300, 45).tolist()
    attend(ctx, Served(lengths, HK, 128, seed=H), r.integers(1, 4, 45).tolist(), H, kind, window=window)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_many_sequences_split(ctx, kind):
    """Two long sequences among short ones: theirs alone are split."""
    say("many split", kind)
    lengths = np.random.default_rng(3).integers(1, 60, 34)
    lengths[[4, 30]] = 1500, 1437
    attend(ctx, Served(lengths.tolist(), 8, 64, seed=3), [1] * 34, 16, kind, max_len=1500)


# More than 256 workgroups: tiles are taken in order of their pages, if there
# are more than 16 of them (wide tiles: 4).  Sequences, kv heads, query heads,
# most rows, window, longest.
ORDERED = [("bf16", 64, 8, 16, 1, 0, 1100), ("f32", 60, 9, 18, 1, 0, 1100), ("f16", 40, 16, 16, 3, 100, 1100), ("f32", 130, 4, 68, 2, 0, 1100),
           ("bf16", 300, 2, 4, 1, 0, 1100), ("f32", 20, 16, 320, 9, 70, 1100), ("bf16", 9, 4, 480, 60, 0, 500), ("f32", 33, 8, 8, 3, 0, 260)]


@pytest.mark.parametrize("kind,seqs,HK,H,most,window,longest", ORDERED)
def test_attention_ordered_tiles(ctx, kind, seqs, HK, H, most, window, longest):
    """Lengths in no order, some equal, some empty: every row is written, once."""
    say("ordered", kind, seqs, HK, H, most, window)
    r = np.random.default_rng(seqs)
    lengths = (r.integers(0, longest, seqs) // r.choice([1, 8, 64], seqs)).tolist()
    lengths[seqs // 2] = longest
    fresh = r.integers(0 if most > 1 else 1, most + 1, seqs).tolist()
    rows = sum(fresh)
    out = torch.full((rows + 2, H, 64), 5.0, dtype=TYPES[kind], device=DEV)
    attend(ctx, Served(lengths, HK, 64, seed=seqs), fresh, H, kind, window=window, extra=2, out=out)
    assert bool((out[rows:] == 5).all())


def test_attention_ordered_tiles_with_bad_sequences(ctx):
    """Lengths that are none, in the midst of others: their rows stay, the
    others' are written."""
    lengths = np.random.default_rng(1).integers(1, 1100, 64) // 2
    lengths[7] = 1100
    sv = Served(lengths.tolist(), 8, 64, seed=41)
    given = lengths.copy()
    given[[3, 20]], given[41], given[50] = -7, 2 ** 31 - 1, 2 ** 31 - 70
    q = torch.randn((64, 8, 64), generator=torch.Generator().manual_seed(6)).to(DEV)
    out = torch.full_like(q, 9.0)
    ctx.kv4_attention(q, sv.cache, i32(sv.table), i32(np.arange(65)), i32(given), out=out, max_len=1100)
    got, bad = host(out), np.isin(np.arange(64), [3, 20, 41])
    assert (got[bad] == 9).all() and np.isnan(got[50]).all()
    bad[50] = True
    want, mag, big = kv4_ref.attention(host(q), sv.pool, sv.table, np.arange(65), lengths, 0.125, 0)
    compare(got[~bad], want[~bad], mag[~bad], big[~bad], "f32", lengths)


def test_pages_far_into_a_large_pool(ctx):
    """Offsets beyond 32 bits, and layers interleaved page by page."""
    HK, D = 8, 128
    size = qtts.kv4_page_bytes(HK, D)
    n = (5 << 30) // (2 * size)
    both = torch.empty((n, 2, size), dtype=torch.uint8, device=DEV)
    r = np.random.default_rng(16)
    table = np.array([[n - 1, n - 5], [1, 0]])
    q = torch.randn((2, 16, D), generator=torch.Generator().manual_seed(6)).to(DEV)
    row_start, lengths = [0, 1, 2], [100, 70]
    k, v = r.standard_normal((2, 170, HK, D))
    slots = np.concatenate([[table[b][p // PAGE] * PAGE + p % PAGE for p in range(m)] for b, m in enumerate(lengths)])
    for layer in (0, 1):
        cache = qtts.Kv4Cache(both[:, layer], HK, D)
        assert cache.desc.page_stride == 2 * size
        kl, vl = k * (layer + 1), v + layer
        ctx.qk_norm_rope(torch.zeros((170, 16, D), device=DEV), dev(kl, torch.float32), v=dev(vl, torch.float32), cache=cache, slots=dev(slots))
        small = Pool(4, HK, D)
        near_ids = {n - 1: 0, n - 5: 1, 1: 2, 0: 3}
        small.put(np.array([near_ids[s // PAGE] * PAGE + s % PAGE for s in slots]), kl.astype(np.float32).astype(np.float64), vl.astype(np.float32).astype(np.float64))
        got = host(ctx.kv4_attention(q, cache, i32(table), i32(row_start), i32(lengths)))
        want, mag, big = kv4_ref.attention(host(q), small, np.vectorize(near_ids.get)(table), row_start, lengths, np.float64(np.float32(D ** -0.5)), 0)
        compare(got, want, mag, big, "f32", lengths)


# ---------------------------------------------------------------------------
# together, streams and graphs
# ---------------------------------------------------------------------------

class Serving:
    """A step as a program runs it: tables, then per layer norm + rotation +
    store and attention."""

    def __init__(self, ctx, kind="f32", H=4, HK=2, D=64, layers=2, pages=40, seed=20):
        self.ctx, self.kind, self.H, self.HK, self.D = ctx, kind, H, HK, D
        self.pools = [Pool(pages, HK, D) for _ in range(layers)]
        self.caches = [qtts.Kv4Cache(dev(p.b), HK, D) for p in self.pools]
        self.free = list(np.random.default_rng(seed).permutation(pages))
        cos, sin = rope_tables(300, D)
        self.cos, self.sin, self.c, self.s = dev(cos), dev(sin), cos.astype(np.float64), sin.astype(np.float64)
        self.gamma = (1 + 0.2 * np.random.default_rng(seed).standard_normal(D)).astype(np.float16)
        self.weight = dev(self.gamma)

    def rows(self, rows, seed):
        r = np.random.default_rng(seed)
        return [torch.as_tensor(r.standard_normal((rows, h, self.D))).to(TYPES[self.kind]).to(DEV) for h in (self.H, self.HK, self.HK)]

    def call(self, cached, fresh, free, table, rows, qkv):
        step = self.ctx.kv4_tables(cached, fresh, free, table, rows)
        g, outs = self.weight, []
        for cache, (q, k, v) in zip(self.caches, qkv):
            q, _ = self.ctx.qk_norm_rope(q, k, step.positions, self.cos, self.sin, g, g, v=v, cache=cache, slots=step.slots,
                                         q_out=torch.zeros_like(q))
            outs.append(self.ctx.kv4_attention(q, cache, table, step.row_start, step.lengths, out=torch.zeros_like(q)))
        return step, outs

    def want(self, step, table, qkv, outs):
        row_start, lengths = step.row_start.tolist(), step.lengths.tolist()
        n, pos, slots = row_start[-1], step.positions.cpu().numpy(), step.slots.cpu().numpy()
        for pool, (q, k, v), out in zip(self.pools, qkv, outs):
            g, c, s = self.gamma.astype(np.float64), self.c[pos[:n]], self.s[pos[:n]]
            pool.put(slots[:n], kv4_ref.norm_rope(host(k)[:n], g, 1e-6, c, s), host(v)[:n])
            qn = kv4_ref.norm_rope(host(q)[:n], g, 1e-6, c, s)
            want, mag, big = kv4_ref.attention(qn, pool, table.cpu().numpy(), row_start, lengths, np.float64(np.float32(self.D ** -0.5)), 0)
            # the rotated queries' own rounding: EPS and the norm's f32 sums, relative to `big`, doubled as in bound()
            extra = 2 * (EPS[self.kind] + (self.D / 2 + 10) * 2.0 ** -23) * big[..., None] * mag[..., 0]
            got = host(out)
            assert (np.abs(got[:n] - want) <= bound(self.kind, want, mag, big, lengths) + extra).all()
            assert not got[n:].any()


@pytest.mark.parametrize("kind", list(TYPES))
def test_steps_together(ctx, kind):
    """Prompts, then single positions, then a new request beside old ones, rows
    padded: every step against 64 bits over what the steps before it stored."""
    sv = Serving(ctx, kind)
    cached, table = [0, 0, 0], torch.full((3, 6), -1, dtype=torch.int32, device=DEV)
    for i, fresh in enumerate(([70, 5, 0], [1, 1, 0], [1, 60, 130], [1, 1, 1], [1, 1, 1])):
        rows = sum(fresh) + 3 * (i % 2)
        qkv = [sv.rows(rows, 100 * i + j) for j in range(2)]
        step, outs = sv.call(i32(cached), i32(fresh), i32(sv.free), table, rows, qkv)
        sv.free = sv.free[step.check():]
        cached = [c + f for c, f in zip(cached, fresh)]
        assert step.lengths.tolist() == cached
        sv.want(step, table, qkv, outs)


def test_another_stream_and_device_guard(ctx):
    """Rows made on a side stream and read there, without a wait of the host."""
    sv = Served([300, 20], 2, 64, seed=21)
    args = [sv.cache, i32(sv.table), i32([0, 1, 2]), i32(sv.lengths)]
    base = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(7)).to(DEV)
    torch.cuda.synchronize()
    want = ctx.kv4_attention(base * 2, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn((4096, 4096), device=DEV)
        for _ in range(4):
            x = x @ x * 1e-3                                 # keeps the stream busy while the call is queued
        q = base * 2 + 0 * x[0, 0].nan_to_num(0, 0, 0)
        got = ctx.kv4_attention(q, *args)
        total = got + 0
    side.synchronize()
    assert torch.equal(total, want) and torch.cuda.current_device() == 0


def test_graph_replays_a_step(ctx):
    """One captured step replayed over growing sequences, eager steps of a
    second program between the replays, each replay against 64 bits."""
    sv, other = Serving(ctx, "f32"), Serving(ctx, "f32", seed=30)
    cached, fresh = i32([0, 0]), i32([1, 1])
    table, free = torch.full((2, 5), -1, dtype=torch.int32, device=DEV), i32(sv.free)
    qkv = [sv.rows(2, j) for j in range(2)]
    sv.call(cached, fresh, free, table, 2, qkv)
    torch.cuda.synchronize()
    for c in sv.caches:
        c.pages.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, outs = sv.call(cached, fresh, free, table, 2, qkv)
    o_cached, o_table = [0, 0], torch.full((2, 5), -1, dtype=torch.int32, device=DEV)
    used = 0
    for i, n in enumerate([(0, 0), (1, 1), (2, 2), (3, 3)]):
        for j in range(2):
            for t, x in zip(qkv[j], sv.rows(2, 50 * i + j)):
                t.copy_(x)
        cached.copy_(i32(n))
        free[:len(sv.free) - used].copy_(i32(sv.free[used:]))
        graph.replay()
        torch.cuda.synchronize()
        used += step.check()
        sv.want(step, table, qkv, outs)
        o_qkv = [other.rows(2, 70 * i + j) for j in range(2)]
        o_step, o_outs = other.call(i32(o_cached), fresh, i32(other.free), o_table, 2, o_qkv)
        other.free = other.free[o_step.check():]
        o_cached = [c + 1 for c in o_cached]
        other.want(o_step, o_table, o_qkv, o_outs)


def test_two_graphs_of_split_calls(ctx):
    """Calls that use a workspace, captured twice and replayed on two streams at
    once: neither writes into the other's."""
    sv = Served([4000], 1, 128, seed=22)
    runs = []
    for i in range(2):
        q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(i)).to(DEV)
        args = (q, sv.cache, i32(sv.table), i32([0, 1]), i32([4000]))
        want = ctx.kv4_attention(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ctx.kv4_attention(*args)
        runs.append((g, out, want, torch.cuda.Stream(), args))
    for _ in range(5):
        for g, out, _, s, _ in runs:
            out.zero_()
        torch.cuda.synchronize()
        for g, _, _, s, _ in runs:
            with torch.cuda.stream(s):
                for _ in range(20):
                    g.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in runs:
            assert torch.equal(out, want)


def test_calls_from_two_threads(ctx):
    """Calls that need workspaces of different sizes, made at the same time."""
    jobs = []
    for i, n in enumerate((4000, 1500, 70)):
        sv = Served([n], 1, 128, seed=50 + i)
        q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(i)).to(DEV)
        args = (q, sv.cache, i32(sv.table), i32([0, 1]), i32([n]))
        jobs.append((args, ctx.kv4_attention(*args)))
    torch.cuda.synchronize()
    wrong = []

    def work(args, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                out = ctx.kv4_attention(*args)
            torch.cuda.current_stream().synchronize()
            if not torch.equal(out, want):
                wrong.append(args[-1])
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_calls_repeat_bit_for_bit(ctx):
    sv = Served([3000, 700], 2, 128, seed=23)
    q = torch.randn((4, 8, 128), generator=torch.Generator().manual_seed(8)).to(DEV)
    args = (q, sv.cache, i32(sv.table), i32([0, 1, 4]), i32(sv.lengths))
    first = ctx.kv4_attention(*args)
    for _ in range(5):
        assert torch.equal(ctx.kv4_attention(*args), first)


def test_binding_refusals(ctx):
    """What the Python methods refuse before the C ABI sees it, and its codes."""
    sv = Served([10], 2, 64, seed=24)
    q, t, rs, n = torch.zeros((1, 4, 64), device=DEV), i32(sv.table), i32([0, 1]), i32([10])
    for bad in ((q.cpu(), sv.cache, t, rs, n), (q, sv.cache, t.long(), rs, n), (q, sv.cache, t, rs[:1], n), (q, sv.cache, t, rs, n.cpu()),
                (torch.zeros((1, 4, 128), device=DEV), sv.cache, t, rs, n), (q.transpose(1, 2).contiguous().transpose(1, 2), sv.cache, t, rs, n),
                (q[0], sv.cache, t, rs, n)):
        with pytest.raises(ValueError):
            ctx.kv4_attention(*bad)
    with pytest.raises(TypeError):
        ctx.kv4_attention(q.double(), sv.cache, t, rs, n)
    with pytest.raises(qtts.QttsError) as e:
        ctx.kv4_attention(torch.zeros((1, 3, 64), device=DEV), sv.cache, t, rs, n)
    assert e.value.code == qtts.ERR_INVALID
    with pytest.raises(ValueError):
        qtts.Kv4Cache(sv.cache.pages[:, :1], 2, 64)
    k = torch.zeros((1, 2, 64), device=DEV)
    with pytest.raises(ValueError):
        ctx.qk_norm_rope(q, k, cache=sv.cache)
    with pytest.raises(TypeError):
        ctx.qk_norm_rope(q, k.half())
    with pytest.raises(ValueError):
        ctx.qk_norm_rope(q, k, positions=i32([0]), cos=torch.zeros((5, 64), device=DEV), sin=torch.zeros((5, 64), device=DEV))
    with pytest.raises(ValueError):
        ctx.kv4_tables(i32([1]), i32([1, 2]), i32([0]), t, 5)
