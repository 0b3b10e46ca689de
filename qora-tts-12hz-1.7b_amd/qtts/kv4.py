"""Serving many sequences over a 4-bit cache: the methods of Context that take
torch tensors on its device (qtts_kv4_tables, qtts_qk_norm_rope,
qtts_kv4_gather, qtts_kv4_attention of include/qtts.h).

Each call only enqueues kernels, on torch's current stream of the context's
device, and may be captured into a graph.  Results and workspaces come from
torch's allocator unless `out` arguments are given.  They are operators for
serving: no gradient passes through them.

A decode step makes these calls in every layer, so a call's way to its launch
counts as its kernel does: arguments are packed into the C structs' bytes
(their ctypes mirrors are in hostdesc.py), and what a tensor is gets checked by
identity and plain numbers.
"""
import ctypes
import math
import struct
import sys

from .hostdesc import Kv4

PAGE = 64
WHOLE = 16 * PAGE            # attention over no more positions is never split: it needs no workspace
_TABLES = struct.Struct("@iiPPPqPqPPPPqP")                 # qtts_kv4_tables_args
_POST = struct.Struct("@iiiiqPPPqqqPPqqPPfiPPqPPP")        # qtts_qk_norm_rope_args
_ATTENTION = struct.Struct("@iiqPPqqPiiPPPqqfiPq")         # qtts_kv4_attention_args

_torch = None                # the module, once a tensor has come
_codes = {}                  # torch dtype -> QTTS_F32 / F16 / BF16
_stream = None               # device -> torch's current stream


def _load():
    global _torch, _stream
    t = sys.modules["torch"]     # whoever passes its tensors has imported it
    _codes.update({t.float32: 0, t.float16: 1, t.bfloat16: 2})
    _stream = t._C._cuda_getCurrentRawStream
    _torch = t


def kv4_page_bytes(n_kv_heads, head_dim):
    """Bytes of one page (64 positions of every kv head)."""
    return n_kv_heads * 72 * head_dim


def _code(name, t):
    code = _codes.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")
    return code


def _elsewhere(name, t, device):
    return ValueError(f"{name} is on {t.device}, the context on cuda:{device}")


def _vector(name, t, n, dtype, device):
    """The address of a contiguous vector of n values of that type."""
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} [{n}] expected, got {t.dtype} {list(t.shape)}")
    if t.get_device() != device:
        raise _elsewhere(name, t, device)
    return t.data_ptr()


def _rows(name, t, shape, dtype, device):
    """shape = (rows, heads, dim) with whole heads next to each other: the row stride."""
    if t.shape != shape:
        raise ValueError(f"{name}: {list(shape)} expected, got {list(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, not {dtype}")
    if t.get_device() != device:
        raise _elsewhere(name, t, device)
    rows, heads, dim = shape
    if rows == 0:
        return heads * dim
    row, head, one = t.stride()
    if one != 1 or (heads > 1 and head != dim):
        raise ValueError(f"{name}: the heads of a row must lie next to each other")
    return row if rows > 1 else heads * dim


def _table(t, n, device):
    """[n][max_pages] int32 with the entries of a row next to each other: the row stride."""
    if t.dim() != 2 or t.shape[0] != n or t.dtype is not _torch.int32 or (n and t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"table: int32 [{n}][max_pages] expected, got {t.dtype} {list(t.shape)}")
    if t.get_device() != device:
        raise _elsewhere("table", t, device)
    return t.stride(0) if n > 1 else t.shape[1]


class Kv4Cache:
    """One layer's pages: a uint8 tensor [n_pages][kv_heads * 72 * head_dim]
    (trailing dimensions may be split; pages may lie further apart)."""

    def __init__(self, pages, n_kv_heads, head_dim):
        if _torch is None:
            _load()
        size, shape, strides = n_kv_heads * 72 * head_dim, pages.shape, pages.stride()
        n, inner = shape[0] if shape else 0, 1
        for d in range(len(shape) - 1, 0, -1):
            if strides[d] != inner and shape[d] > 1:
                inner = -1
                break
            inner *= shape[d]
        if inner != size or pages.dtype is not _torch.uint8 or len(shape) < 2:
            raise ValueError(f"pages: uint8 [n][{size}] expected, got {pages.dtype} {list(shape)}")
        self.pages, self.n_kv_heads, self.head_dim = pages, n_kv_heads, head_dim
        self.device = pages.get_device()
        self.desc = Kv4(pages.data_ptr(), n, strides[0] if n > 1 else size, n_kv_heads, head_dim)
        self.address = ctypes.addressof(self.desc)


class Kv4Step:
    """What one step's rows are: row_start, lengths, positions and slots for the
    operators, and status, which check() reads (it waits for the device)."""
    __slots__ = ("row_start", "lengths", "positions", "slots", "status")

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
    if _torch is None:
        _load()
    device, i32 = self.device, _torch.int32
    n, free = cached.shape[0], free_pages.shape[0]
    inputs = (_vector("cached", cached, n, i32, device), _vector("fresh", fresh, n, i32, device),
              _vector("free_pages", free_pages, free, i32, device), free, table.data_ptr(), _table(table, n, device))
    if out is None:
        # one allocation for what is held in 32 bits
        both = cached.new_empty(2 * n + rows + 3)
        slots = cached.new_empty(rows, dtype=_torch.int64)
        at = both.data_ptr()
        a = _TABLES.pack(n, table.shape[1], *inputs, at, at + 4 * n + 4, at + 8 * n + 4, slots.data_ptr(), rows,
                         at + 8 * n + 4 * rows + 4)
        row_start, lengths, positions, status = both.split_with_sizes([n + 1, n, rows, 2])
        out = Kv4Step(row_start, lengths, positions, slots, status)
    else:
        a = _TABLES.pack(n, table.shape[1], *inputs, _vector("row_start", out.row_start, n + 1, i32, device),
                         _vector("lengths", out.lengths, n, i32, device), _vector("positions", out.positions, rows, i32, device),
                         _vector("slots", out.slots, rows, _torch.int64, device), rows,
                         _vector("status", out.status, 2, i32, device))
    rc = self.lib.qtts_kv4_tables(self.h, a, _stream(device), 0)
    if rc:
        self._check(rc)
    return out


def qk_norm_rope(self, q, k, positions=None, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-6, v=None, cache=None,
                 slots=None, q_out=None, k_out=None):
    """Norm and rotation of q [rows][heads][dim] and k [rows][kv_heads][dim]
    (qtts_qk_norm_rope); with a cache, k so treated and v are stored at `slots`
    [rows] int64 in the same pass.  cos and sin [max_pos][dim / 2] f32,
    positions [rows] int32, q_norm and k_norm [dim] f16; None leaves that part
    out.  Returns (q_out, k_out); with a cache k is only written out where k_out
    is given."""
    if _torch is None:
        _load()
    device, dtype = self.device, q.dtype
    rows, heads, dim = shape = q.shape
    kv_heads = k.shape[1] if k.dim() == 3 else 0
    k_shape = (rows, kv_heads, dim)
    code = _code("q", q)
    q_stride, k_stride = _rows("q", q, shape, dtype, device), _rows("k", k, k_shape, dtype, device)
    if q_out is None:
        q_out, qo_stride = _torch.empty_like(q, memory_format=_torch.contiguous_format), heads * dim
    else:
        qo_stride = _rows("q_out", q_out, shape, dtype, device)
    if k_out is None and cache is None:
        k_out = _torch.empty_like(k, memory_format=_torch.contiguous_format)
    ko, ko_stride = (0, 0) if k_out is None else (k_out.data_ptr(), _rows("k_out", k_out, k_shape, dtype, device))
    at = cos_at = sin_at = most = vp = v_stride = desc = slots_at = 0
    if positions is not None:
        if cos is None or sin is None:
            raise ValueError("positions need cos and sin")
        most, f32 = cos.shape[0], _torch.float32
        table = (most, dim // 2)
        if cos.shape != table or sin.shape != table or cos.dtype is not f32 or sin.dtype is not f32 or \
                not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError(f"cos and sin: contiguous float32 [max_pos][{dim // 2}] expected")
        if cos.get_device() != device or sin.get_device() != device:
            raise _elsewhere("cos or sin", cos if cos.get_device() != device else sin, device)
        at, cos_at, sin_at = _vector("positions", positions, rows, _torch.int32, device), cos.data_ptr(), sin.data_ptr()
    if cache is not None:
        if v is None or slots is None:
            raise ValueError("a cache needs v and slots")
        if cache.device != device:
            raise _elsewhere("the cache", cache.pages, device)
        vp, v_stride, desc = v.data_ptr(), _rows("v", v, k_shape, dtype, device), cache.address
        slots_at = _vector("slots", slots, rows, _torch.int64, device)
    f16 = _torch.float16
    a = _POST.pack(code, heads, kv_heads, dim, rows, q.data_ptr(), k.data_ptr(), vp, q_stride, k_stride, v_stride,
                   q_out.data_ptr(), ko, qo_stride, ko_stride,
                   0 if q_norm is None else _vector("q_norm", q_norm, dim, f16, device),
                   0 if k_norm is None else _vector("k_norm", k_norm, dim, f16, device),
                   eps, 0, cos_at, sin_at, most, at, desc, slots_at)
    rc = self.lib.qtts_qk_norm_rope(self.h, a, _stream(device), 0)
    if rc:
        self._check(rc)
    return q_out, k_out


def gather(self, cache, slots, dtype):
    """The keys and values held at `slots` [n] int64 (qtts_kv4_gather): two
    tensors [n][kv_heads][dim] of `dtype`, zero for a slot outside the pages."""
    if _torch is None:
        _load()
    device = self.device
    if cache.device != device:
        raise _elsewhere("the cache", cache.pages, device)
    n = slots.shape[0]
    at = _vector("slots", slots, n, _torch.int64, device)
    both = slots.new_empty((2, n, cache.n_kv_heads, cache.head_dim), dtype=dtype)
    K = both.data_ptr()
    rc = self.lib.qtts_kv4_gather(self.h, cache.address, at, n, _code("values", both), K, K + both.nbytes // 2, _stream(device), 0)
    if rc:
        self._check(rc)
    return both.unbind()


def attention(self, q, cache, table, row_start, lengths, scale=None, window=0, max_len=None, out=None):
    """Attention of q [rows][heads][dim] over the sequences' pages
    (qtts_kv4_attention): table [n_seqs][max_pages], row_start [n_seqs + 1] and
    lengths [n_seqs] int32.  scale None: 1 / sqrt(dim).  max_len, an upper
    bound of the lengths, helps to split the work.  Rows outside all sequences
    are left as they are in `out`."""
    if _torch is None:
        _load()
    device, dtype, i32 = self.device, q.dtype, _torch.int32
    dim, n = cache.head_dim, lengths.shape[0]
    if cache.device != device:
        raise _elsewhere("the cache", cache.pages, device)
    if q.dim() != 3:
        raise ValueError(f"q: [rows][heads][{dim}] expected, got {list(q.shape)}")
    rows, heads = q.shape[0], q.shape[1]
    shape = (rows, heads, dim)
    code, q_stride = _code("q", q), _rows("q", q, shape, dtype, device)
    if out is None:
        out, out_stride = _torch.empty_like(q, memory_format=_torch.contiguous_format), heads * dim
    else:
        out_stride = _rows("out", out, shape, dtype, device)
    columns = table.shape[1] if table.dim() == 2 else 0
    if max_len is None:
        max_len = PAGE * columns
    head = (code, heads, rows, q.data_ptr(), out.data_ptr(), q_stride, out_stride, cache.address, n, columns,
            _vector("row_start", row_start, n + 1, i32, device), _vector("lengths", lengths, n, i32, device), table.data_ptr(),
            _table(table, n, device), max_len, 1 / math.sqrt(dim) if scale is None else scale, window)
    a = _ATTENTION.pack(*head, 0, 0)
    if max_len > WHOLE:
        need = ctypes.c_int64()
        self.lib.qtts_kv4_attention_workspace(a, ctypes.addressof(need))      # what it refuses the call itself names
        if need.value:
            workspace = q.new_empty(need.value, dtype=_torch.uint8)
            a = _ATTENTION.pack(*head, workspace.data_ptr(), need.value)
    rc = self.lib.qtts_kv4_attention(self.h, a, _stream(device), 0)
    if rc:
        self._check(rc)
    return out
