"""Serving many sequences over a 4-bit cache: the methods of Context that take
torch tensors on its device (qtts_kv4_tables, qtts_qk_norm_rope,
qtts_kv4_gather, qtts_kv4_attention of include/qtts.h).

Each call only enqueues kernels, on torch's current stream of the context's
device, and may be captured into a graph.  Results and workspaces come from
torch's allocator unless `out` arguments are given.
"""
import ctypes
import math
import sys

from .hostdesc import Kv4, Kv4AttentionArgs, Kv4TablesArgs, QkNormRopeArgs

PAGE = 64
_DTYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
_by_dtype = {}               # torch dtype -> QTTS_F32 / F16 / BF16


def kv4_page_bytes(n_kv_heads, head_dim):
    """Bytes of one page (64 positions of every kv head)."""
    return n_kv_heads * 72 * head_dim


def _dtype(t):
    code = _by_dtype.get(t)
    if code is None:
        code = _DTYPES.get(str(t))
        if code is None:
            raise TypeError(f"rows are float32, float16 or bfloat16, not {t}")
        _by_dtype[t] = code
    return code


def _torch():
    return sys.modules["torch"]  # whoever passes its tensors has imported it


def _stream(ctx):
    return _torch()._C._cuda_getCurrentRawStream(ctx.device)


def _on(ctx, **tensors):
    for name, t in tensors.items():
        if t is not None and (t.device.type != "cuda" or t.device.index != ctx.device):
            raise ValueError(f"{name} is on {t.device}, the context on cuda:{ctx.device}")


def _vector(name, t, n, dtype):
    """A contiguous vector of n (None: any number) whole numbers of that type."""
    if t.dim() != 1 or (n is not None and t.shape[0] != n) or str(t.dtype) != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} [{'n' if n is None else n}] expected, got {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def _rows(name, t, heads=None, dim=None, dtype=None):
    """[rows][heads][dim] with whole heads next to each other: the row stride."""
    if t.dim() != 3 or (heads is not None and tuple(t.shape[1:]) != (heads, dim)):
        raise ValueError(f"{name}: [rows][{heads or 'heads'}][{dim or 'dim'}] expected, got {list(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, not {dtype}")
    if t.shape[0] and ((t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != t.shape[2])):
        raise ValueError(f"{name}: the heads of a row must lie next to each other")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _table(t, n):
    """[n][max_pages] int32 with the entries of a row next to each other: the row stride."""
    if t.dim() != 2 or t.shape[0] != n or str(t.dtype) != "torch.int32" or (n and t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"table: int32 [{n}][max_pages] expected, got {t.dtype} {list(t.shape)}")
    return t.stride(0) if n > 1 else t.shape[1]


class Kv4Cache:
    """One layer's pages: a uint8 tensor [n_pages][kv_heads * 72 * head_dim]
    (trailing dimensions may be split; pages may lie further apart)."""

    def __init__(self, pages, n_kv_heads, head_dim):
        size = kv4_page_bytes(n_kv_heads, head_dim)
        if str(pages.dtype) != "torch.uint8" or pages.dim() < 2 or pages[0].numel() != size or not pages[0].is_contiguous():
            raise ValueError(f"pages: uint8 [n][{size}] expected, got {pages.dtype} {list(pages.shape)}")
        self.pages, self.n_kv_heads, self.head_dim = pages, n_kv_heads, head_dim
        stride = pages.stride(0) if pages.shape[0] > 1 else size
        self.desc = Kv4(pages.data_ptr(), pages.shape[0], stride, n_kv_heads, head_dim)


class Kv4Step:
    """What one step's rows are: row_start, lengths, positions and slots for the
    operators, and status, which check() reads (it waits for the device)."""

    def __init__(self, row_start, lengths, positions, slots, status):
        self.row_start, self.lengths, self.positions, self.slots, self.status = row_start, lengths, positions, slots, status

    def check(self):
        """The number of pages taken; raises where the step did not fit."""
        from . import QttsError
        code, pages = self.status.tolist()
        if code:
            raise QttsError(code, "negative length" if code == -1 else "rows, table columns or free pages do not suffice")
        return pages


def tables(self, cached, fresh, free_pages, table, rows, out=None):
    """Block tables and slots of a step (qtts_kv4_tables): cached and fresh
    [n_seqs] int32, free_pages [n] int32, table [n_seqs][max_pages] int32
    (written in place), `rows` the room for rows.  Returns a Kv4Step (out: one
    to write into)."""
    n = cached.shape[0]
    _on(self, cached=cached, fresh=fresh, free_pages=free_pages, table=table)
    if out is None:
        i32 = cached.dtype
        out = Kv4Step(cached.new_empty(n + 1), cached.new_empty(n), cached.new_empty(rows),
                      cached.new_empty(rows, dtype=_torch().int64), cached.new_empty(2, dtype=i32))
    else:
        _on(self, row_start=out.row_start, lengths=out.lengths, positions=out.positions, slots=out.slots, status=out.status)
    stride = _table(table, n)
    a = Kv4TablesArgs(n, table.shape[1], _vector("cached", cached, n, "torch.int32"), _vector("fresh", fresh, n, "torch.int32"),
                      _vector("free_pages", free_pages, None, "torch.int32"), free_pages.shape[0], table.data_ptr(), stride,
                      _vector("row_start", out.row_start, n + 1, "torch.int32"), _vector("lengths", out.lengths, n, "torch.int32"),
                      _vector("positions", out.positions, rows, "torch.int32"), _vector("slots", out.slots, rows, "torch.int64"),
                      rows, _vector("status", out.status, 2, "torch.int32"))
    self._check(self.lib.qtts_kv4_tables(self.h, ctypes.byref(a), _stream(self), 0))
    return out


def qk_norm_rope(self, q, k, positions=None, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-6, v=None, cache=None,
                 slots=None, q_out=None, k_out=None):
    """Norm and rotation of q [rows][heads][dim] and k [rows][kv_heads][dim]
    (qtts_qk_norm_rope); with a cache, k so treated and v are stored at `slots`
    [rows] int64 in the same pass.  cos and sin [max_pos][dim / 2] f32,
    positions [rows] int32, q_norm and k_norm [dim] f16; None leaves that part
    out.  Returns (q_out, k_out); with a cache k is only written out where k_out
    is given."""
    _on(self, q=q, k=k, v=v, positions=positions, cos=cos, sin=sin, q_norm=q_norm, k_norm=k_norm, slots=slots, q_out=q_out, k_out=k_out)
    rows, heads, dim = q.shape
    dtype = q.dtype
    code = _dtype(dtype)
    q_stride = _rows("q", q)
    k_stride = _rows("k", k, k.shape[1], dim, dtype)
    if k.shape[0] != rows:
        raise ValueError(f"k has {k.shape[0]} rows, q {rows}")
    if q_out is None:
        q_out = q.new_empty(q.shape)
    if k_out is None and cache is None:
        k_out = k.new_empty(k.shape)
    a = QkNormRopeArgs(code, heads, k.shape[1], dim, rows, q.data_ptr(), k.data_ptr(), None, q_stride, k_stride, 0,
                       q_out.data_ptr(), None, _rows("q_out", q_out, heads, dim, dtype))
    if q_out.shape[0] != rows or (k_out is not None and k_out.shape[0] != rows):
        raise ValueError("outputs must have as many rows as q")
    if k_out is not None:
        a.k_out, a.k_out_stride = k_out.data_ptr(), _rows("k_out", k_out, k.shape[1], dim, dtype)
    if q_norm is not None:
        a.q_norm = _vector("q_norm", q_norm, dim, "torch.float16")
    if k_norm is not None:
        a.k_norm = _vector("k_norm", k_norm, dim, "torch.float16")
    a.eps = eps
    if positions is not None:
        if cos is None or sin is None or cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != dim // 2 or \
                str(cos.dtype) != "torch.float32" or cos.dtype != sin.dtype or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError(f"cos and sin: contiguous float32 [max_pos][{dim // 2}] expected")
        a.rope_cos, a.rope_sin, a.rope_max_pos = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
        a.positions = _vector("positions", positions, rows, "torch.int32")
    if cache is not None:
        if v is None or slots is None:
            raise ValueError("a cache needs v and slots")
        _on(self, pages=cache.pages)
        a.v, a.v_stride = v.data_ptr(), _rows("v", v, k.shape[1], dim, dtype)
        if v.shape[0] != rows:
            raise ValueError(f"v has {v.shape[0]} rows, q {rows}")
        a.cache = ctypes.pointer(cache.desc)
        a.slots = _vector("slots", slots, rows, "torch.int64")
    self._check(self.lib.qtts_qk_norm_rope(self.h, ctypes.byref(a), _stream(self), 0))
    return q_out, k_out


def gather(self, cache, slots, dtype):
    """The keys and values held at `slots` [n] int64 (qtts_kv4_gather): two
    tensors [n][kv_heads][dim] of `dtype`, zero for a slot outside the pages."""
    _on(self, slots=slots, pages=cache.pages)
    n = slots.shape[0]
    shape = (n, cache.n_kv_heads, cache.head_dim)
    K, V = slots.new_empty(shape, dtype=dtype), slots.new_empty(shape, dtype=dtype)
    self._check(self.lib.qtts_kv4_gather(self.h, ctypes.byref(cache.desc), _vector("slots", slots, None, "torch.int64"), n,
                                         _dtype(dtype), K.data_ptr(), V.data_ptr(), _stream(self), 0))
    return K, V


def attention(self, q, cache, table, row_start, lengths, scale=None, window=0, max_len=None, out=None):
    """Attention of q [rows][heads][dim] over the sequences' pages
    (qtts_kv4_attention): table [n_seqs][max_pages], row_start [n_seqs + 1] and
    lengths [n_seqs] int32.  scale None: 1 / sqrt(dim).  max_len, an upper
    bound of the lengths, helps to split the work.  Rows outside all sequences
    are left as they are in `out`."""
    _on(self, q=q, table=table, row_start=row_start, lengths=lengths, out=out, pages=cache.pages)
    rows, heads, dim = q.shape
    n = lengths.shape[0]
    if dim != cache.head_dim:
        raise ValueError(f"q has heads of {dim}, the cache of {cache.head_dim}")
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape[0] != rows:
        raise ValueError(f"out has {out.shape[0]} rows, q {rows}")
    a = Kv4AttentionArgs(_dtype(q.dtype), heads, rows, q.data_ptr(), out.data_ptr(), _rows("q", q),
                         _rows("out", out, heads, dim, q.dtype), ctypes.pointer(cache.desc), n, table.shape[1],
                         _vector("row_start", row_start, n + 1, "torch.int32"), _vector("lengths", lengths, n, "torch.int32"),
                         table.data_ptr(), _table(table, n),
                         PAGE * table.shape[1] if max_len is None else max_len, 1 / math.sqrt(dim) if scale is None else scale,
                         window, None, 0)
    need = ctypes.c_int64()
    rc = self.lib.qtts_kv4_attention_workspace(ctypes.byref(a), ctypes.byref(need))
    if rc == 0 and need.value:
        workspace = q.new_empty(need.value, dtype=_torch().uint8)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
    self._check(self.lib.qtts_kv4_attention(self.h, ctypes.byref(a), _stream(self), 0))
    return out
