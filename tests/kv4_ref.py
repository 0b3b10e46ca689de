"""The 4-bit cache's operators in 64 bits, from their definitions (numpy)."""
import numpy as np

PAGE = 64
MOST = 65280.0


def scale_of(m):
    """The stored scale of groups whose extreme value is m: -m / 8 as f32, f16,
    then 8 significant bits (nearest, halves away from zero)."""
    h = (m * -0.125).astype(np.float32).astype(np.float16)
    bits = (h.view(np.uint16).astype(np.int32) + 4) & 0xFFF8
    return bits.astype(np.uint16).view(np.float16)


def quantise(x):
    """x [..., D] f64: (codes uint8 [..., D], scales f16 [..., D / 32])."""
    g = np.clip(x, -MOST, MOST).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = g.max(-1), g.min(-1)
    s = scale_of(np.where(hi >= -lo, hi, lo))
    d = s.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d == 0, 0.0, g / d)
    return np.clip(np.rint(q) + 8, 0, 15).astype(np.uint8).reshape(x.shape), s


def values(codes, scales):
    return ((codes.astype(np.float64).reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32) - 8) * scales.astype(np.float64)[..., None]).reshape(codes.shape)


class Pool:
    """Host pages [n][kv_heads][72 D] written and read one position at a time."""

    def __init__(self, n, heads, dim, fill=0):
        self.b = np.full((n, heads, 72 * dim), fill, np.uint8)
        self.dim = dim

    def put(self, slots, k, v):
        """k, v [n][heads][D] f64 to slots."""
        D, G = self.dim, self.dim // 32
        nan = np.isnan(k).any(-1) | np.isnan(v).any(-1)
        (kc, ks), (vc, vs) = quantise(np.nan_to_num(k, nan=0.0, posinf=MOST, neginf=-MOST)), quantise(np.nan_to_num(v, nan=0.0, posinf=MOST, neginf=-MOST))
        ks, vs = ks.copy(), vs.copy()
        ks[nan], vs[nan] = np.float16(np.nan), 0
        for i, s in enumerate(slots):
            if s < 0 or s >= len(self.b) * PAGE:
                continue
            blk, p = self.b[s // PAGE], s % PAGE
            at = ((p % 4) * 16 + p // 4) * (D // 2)
            blk[:, at:at + D // 2] = kc[i][:, 0::2] | kc[i][:, 1::2] << 4
            for u in range(D // 4):
                at = 32 * D + ((p // 4) * (D // 4) + u) * 8 + (p % 4) * 2
                c = vc[i][:, 4 * u:4 * u + 4]
                blk[:, at], blk[:, at + 1] = c[:, 0] | c[:, 1] << 4, c[:, 2] | c[:, 3] << 4
            for g in range(G):
                for base, sc in ((64 * D, ks), (68 * D, vs)):
                    at = base + (g * PAGE + p) * 2
                    blk[:, at:at + 2] = sc[i][:, g:g + 1].copy().view(np.uint8)

    def get(self, slots):
        """(k, v) [n][heads][D] f64 held at slots; zero outside."""
        D, heads = self.dim, self.b.shape[1]
        k, v = np.zeros((len(slots), heads, D)), np.zeros((len(slots), heads, D))
        for i, s in enumerate(slots):
            if s < 0 or s >= len(self.b) * PAGE:
                continue
            blk, p = self.b[s // PAGE], s % PAGE
            at = ((p % 4) * 16 + p // 4) * (D // 2)
            kb = blk[:, at:at + D // 2]
            vb = np.stack([blk[:, 32 * D + ((p // 4) * (D // 4) + u) * 8 + (p % 4) * 2 + h] for u in range(D // 4) for h in (0, 1)], -1)
            for out, b, base in ((k, kb, 64 * D), (v, vb, 68 * D)):
                codes = np.stack([b & 15, b >> 4], -1).reshape(heads, D)
                sc = np.stack([np.ascontiguousarray(blk[:, base + (g * PAGE + p) * 2:][:, :2]).view(np.float16)[:, 0] for g in range(D // 32)], -1)
                out[i] = values(codes, sc)
        return k, v


def norm_rope(x, gamma, eps, cos, sin):
    """x [rows][heads][D] f64; gamma None: no norm; cos None: no rotation."""
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma
    if cos is None:
        return x
    a, b = np.split(x, 2, -1)
    c, s = cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attention(q, pool, table, row_start, lengths, scale, window):
    """(out, (sum of weights times |v|, largest weight times sum of |v|), largest
    sum of |q k| times |scale|): the last two for error bounds.  Rows outside
    all sequences are NaN."""
    rows, heads, D = q.shape
    out, mag, big = np.full(q.shape, np.nan), np.zeros((*q.shape, 2)), np.zeros((rows, heads))
    for b, n in enumerate(lengths):
        r0, r1 = row_start[b], row_start[b + 1]
        if r1 <= r0:
            continue
        slots = [table[b][p // PAGE] * PAGE + p % PAGE for p in range(n)]
        k, v = pool.get(slots)
        G = heads // pool.b.shape[1]
        for r in range(r0, r1):
            pos = n - (r1 - r0) + r - r0
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                out[r] = 0
                continue
            for kv in range(heads // G):
                h, kk, vv = slice(kv * G, kv * G + G), k[lo:pos + 1, kv], v[lo:pos + 1, kv]
                s = q[r, h] @ kk.T * scale
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                out[r, h] = w @ vv
                mag[r, h, :, 0], mag[r, h, :, 1] = w @ np.abs(vv), w.max(1)[:, None] * np.abs(vv).sum(0)
                big[r, h] = (np.abs(q[r, h]) @ np.abs(kk).T).max(1) * abs(scale)
    return out, mag, big


def tables(cached, fresh, free, table, rows):
    """(table, row_start, lengths, positions, slots, status) of a step that fits."""
    table, at, take = table.copy(), 0, 0
    row_start, positions, slots = [0], [-1] * rows, [-1] * rows
    for b, (c, f) in enumerate(zip(cached, fresh)):
        for col in range(-(-c // PAGE), -(-(c + f) // PAGE)):
            table[b, col] = free[take]
            take += 1
        for i in range(f):
            positions[at] = c + i
            slots[at] = int(table[b, (c + i) // PAGE]) * PAGE + (c + i) % PAGE
            at += 1
        row_start.append(at)
    return table, row_start, [c + f for c, f in zip(cached, fresh)], positions, slots, [0, take]
