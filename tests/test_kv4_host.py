"""The 4-bit cache's operators without a device: what their calls refuse
(QTTS_CHECK_ONLY), the workspace's size, the descriptors' layout, and the
reference that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import kv4_ref
import qtts

from qtts.hostdesc import Kv4, Kv4AttentionArgs, Kv4TablesArgs, QkNormRopeArgs

LIB = qtts.load_library()
A = 1 << 20                       # addresses, never followed
STEP = 1 << 30


def at(i, off=0):
    return A + i * STEP + off


def test_layouts():
    assert ctypes.sizeof(Kv4) == 32
    assert ctypes.sizeof(Kv4TablesArgs) == 104 and Kv4TablesArgs.status.offset == 96
    assert ctypes.sizeof(QkNormRopeArgs) == 176 and QkNormRopeArgs.rope_max_pos.offset == 144 and QkNormRopeArgs.slots.offset == 168
    assert Kv4AttentionArgs.window.offset == 108 and ctypes.sizeof(Kv4AttentionArgs) == 128
    assert qtts.kv4_page_bytes(8, 128) == 73728
    from qtts import kv4
    for packed, mirror in ((kv4._TABLES, Kv4TablesArgs), (kv4._POST, QkNormRopeArgs), (kv4._ATTENTION, Kv4AttentionArgs)):
        assert packed.size == ctypes.sizeof(mirror)
        fields = [f for f, _ in mirror._fields_]
        got = mirror.from_buffer_copy(packed.pack(*range(1, len(fields) + 1)))
        values = [getattr(got, f) for f in fields]
        values = [ctypes.cast(v, ctypes.c_void_p).value if isinstance(v, ctypes._Pointer) else v for v in values]
        assert values == list(range(1, len(fields) + 1))


def cache(**kw):
    return Kv4(**{"base": at(0), "n_pages": 100, "page_stride": 73728, "n_kv_heads": 8, "head_dim": 128, **kw})


BAD_CACHE = [({"base": None}, qtts.ERR_INVALID), ({"base": at(0, 8)}, qtts.ERR_INVALID), ({"n_pages": 0}, qtts.ERR_INVALID),
             ({"page_stride": 73712}, qtts.ERR_INVALID), ({"page_stride": 73736}, qtts.ERR_INVALID),
             ({"n_kv_heads": 0}, qtts.ERR_INVALID), ({"head_dim": 96}, qtts.ERR_UNSUPPORTED), ({"n_pages": 1 << 31}, qtts.ERR_INVALID)]


def tables(**kw):
    a = Kv4TablesArgs(**{"n_seqs": 5, "max_pages": 7, "cached": at(0), "fresh": at(1), "free_pages": at(2), "n_free": 9,
                         "table": at(3), "table_stride": 7, "row_start": at(4), "lengths": at(5), "positions": at(6),
                         "slots": at(7), "n_rows": 30, "status": at(8), **kw})
    return LIB.qtts_kv4_tables(None, ctypes.byref(a), None, qtts.CHECK_ONLY)


@pytest.mark.parametrize("kw,code", [
    ({}, qtts.OK), ({"n_seqs": 0, "cached": None, "fresh": None, "lengths": None, "table": None}, qtts.OK),
    ({"n_rows": 0, "positions": None, "slots": None}, qtts.OK), ({"n_free": 0, "free_pages": None}, qtts.OK),
    ({"n_seqs": 4096}, qtts.OK), ({"n_seqs": 4097}, qtts.ERR_CAPACITY), ({"n_seqs": -1}, qtts.ERR_INVALID),
    ({"table_stride": 6}, qtts.ERR_INVALID), ({"n_rows": -1}, qtts.ERR_INVALID), ({"n_rows": 1 << 31}, qtts.ERR_CAPACITY),
    ({"max_pages": 1 << 26, "table_stride": 1 << 26}, qtts.ERR_CAPACITY), ({"cached": None}, qtts.ERR_INVALID),
    ({"status": None}, qtts.ERR_INVALID), ({"slots": None}, qtts.ERR_INVALID), ({"slots": at(7, 4)}, qtts.ERR_INVALID),
    ({"fresh": at(1, 2)}, qtts.ERR_INVALID), ({"lengths": at(0)}, qtts.ERR_INVALID), ({"lengths": at(0, 16)}, qtts.ERR_INVALID),
    ({"row_start": at(5, 8)}, qtts.ERR_INVALID), ({"free_pages": at(3, 20)}, qtts.ERR_INVALID),
    ({"status": at(6, 116)}, qtts.ERR_INVALID), ({"status": at(6, 120)}, qtts.OK),
])
def test_tables_refusals(kw, code):
    assert tables(**kw) == code


def post(c=None, **kw):
    a = QkNormRopeArgs(**{"dtype": 0, "n_heads": 16, "n_kv_heads": 8, "head_dim": 128, "rows": 10, "q": at(1), "k": at(2),
                          "v": at(3), "q_stride": 2048, "k_stride": 1024, "v_stride": 1024, "q_out": at(4), "k_out": at(5),
                          "q_out_stride": 2048, "k_out_stride": 1024, "q_norm": at(6), "k_norm": at(7), "eps": 1e-6,
                          "rope_cos": at(8), "rope_sin": at(9), "rope_max_pos": 50, "positions": at(10), "slots": at(11), **kw})
    if c is not None:
        a.cache = ctypes.pointer(c)
    return LIB.qtts_qk_norm_rope(None, ctypes.byref(a), None, qtts.CHECK_ONLY)


JOINT = {"q": at(1), "k": at(1, 8192), "v": at(1, 12288), "q_stride": 4096, "k_stride": 4096, "v_stride": 4096}


@pytest.mark.parametrize("kw,code", [
    ({}, qtts.OK), ({"rows": 0, "q": None, "k": None, "q_out": None, "k_out": None}, qtts.OK), (JOINT, qtts.OK),
    ({**JOINT, "q_out": at(1), "q_out_stride": 4096, "k_out": at(1, 8192), "k_out_stride": 4096}, qtts.OK),
    ({**JOINT, "q_out": at(1, 4096), "q_out_stride": 4096}, qtts.ERR_INVALID),
    ({"q_out": at(1)}, qtts.OK), ({"q_out": at(1), "q_out_stride": 2052}, qtts.ERR_INVALID), ({"q_out": at(2)}, qtts.ERR_INVALID),
    ({"k_out": at(4, 4096)}, qtts.ERR_INVALID), ({"k_out": None}, qtts.ERR_INVALID), ({"q": None}, qtts.ERR_INVALID),
    ({"dtype": 3}, qtts.ERR_UNSUPPORTED), ({"head_dim": 80}, qtts.ERR_UNSUPPORTED), ({"n_heads": 12}, qtts.ERR_INVALID),
    ({"q_stride": 2047}, qtts.ERR_INVALID), ({"q": at(1, 2)}, qtts.ERR_INVALID), ({"dtype": 1, "q": at(1, 2)}, qtts.OK),
    ({"rows": -1}, qtts.ERR_INVALID), ({"rows": 1 << 27}, qtts.ERR_CAPACITY), ({"rope_cos": None}, qtts.ERR_INVALID),
    ({"rope_max_pos": 0}, qtts.ERR_INVALID), ({"positions": None, "rope_cos": None, "rope_sin": None}, qtts.OK),
    ({"q_norm": None, "k_norm": None}, qtts.OK), ({"eps": -1.0}, qtts.ERR_INVALID), ({"eps": float("nan")}, qtts.ERR_INVALID),
    ({"eps": float("inf")}, qtts.ERR_INVALID), ({"positions": at(10, 2)}, qtts.ERR_INVALID), ({"q_norm": at(6, 1)}, qtts.ERR_INVALID),
])
def test_qk_norm_rope_refusals(kw, code):
    assert post(**kw) == code


@pytest.mark.parametrize("c,kw,code", [
    ({}, {}, qtts.OK), ({}, {"k_out": None}, qtts.OK), ({}, {"v": None}, qtts.ERR_INVALID), ({}, {"slots": None}, qtts.ERR_INVALID),
    ({}, {"slots": at(11, 4)}, qtts.ERR_INVALID), ({"n_kv_heads": 4}, {}, qtts.ERR_INVALID), ({"head_dim": 64}, {}, qtts.ERR_INVALID),
    ({}, {"q_out": at(0, 4096)}, qtts.ERR_INVALID), ({}, {"v": at(0)}, qtts.ERR_INVALID), ({}, {"v_stride": 1000}, qtts.ERR_INVALID),
] + [(c, {}, code) for c, code in BAD_CACHE])
def test_store_refusals(c, kw, code):
    assert post(cache(**c), **kw) == code


@pytest.mark.parametrize("c,n,dtype,K,V,code", [
    ({}, 5, 0, at(1), at(2), qtts.OK), ({}, 5, 2, None, at(2), qtts.OK), ({}, 0, 0, None, None, qtts.OK),
    ({}, 5, 7, at(1), at(2), qtts.ERR_UNSUPPORTED), ({}, -1, 0, at(1), at(2), qtts.ERR_INVALID), ({}, 5, 0, at(1, 8), at(2), qtts.ERR_INVALID),
    ({}, 5, 0, at(1), at(1, 64), qtts.ERR_INVALID), ({}, 5, 0, at(0), at(2), qtts.ERR_INVALID), ({}, 1 << 27, 0, at(1), at(2), qtts.ERR_CAPACITY),
] + [(c, 5, 0, at(1), at(2), code) for c, code in BAD_CACHE])
def test_gather_refusals(c, n, dtype, K, V, code):
    assert LIB.qtts_kv4_gather(None, ctypes.byref(cache(**c)), at(3), n, dtype, K, V, None, qtts.CHECK_ONLY) == code


def attention_args(c, **kw):
    a = Kv4AttentionArgs(**{"dtype": 0, "n_heads": 16, "rows": 10, "q": at(1), "out": at(2), "q_stride": 2048, "out_stride": 2048,
                            "n_seqs": 4, "max_pages": 20, "row_start": at(3), "lengths": at(4), "table": at(5),
                            "table_stride": 20, "max_len": 200, "scale": 0.1, "window": 0, "workspace": at(6),
                            "workspace_bytes": STEP, **kw})
    a.cache = ctypes.pointer(c)
    return a


def attend(c, **kw):
    return LIB.qtts_kv4_attention(None, ctypes.byref(attention_args(c, **kw)), None, qtts.CHECK_ONLY)


@pytest.mark.parametrize("kw,code", [
    ({}, qtts.OK), ({"rows": 0, "q": None, "out": None}, qtts.OK), ({"n_seqs": 0, "row_start": None, "lengths": None, "table": None}, qtts.OK),
    ({"out": at(1)}, qtts.OK), ({"out": at(1), "out_stride": 2052}, qtts.ERR_INVALID), ({"out": at(1, 2048 * 4)}, qtts.ERR_INVALID),
    ({"out": at(0)}, qtts.ERR_INVALID), ({"out": at(5)}, qtts.ERR_INVALID), ({"out": at(4)}, qtts.ERR_INVALID),
    ({"dtype": -1}, qtts.ERR_UNSUPPORTED), ({"n_heads": 20}, qtts.ERR_INVALID), ({"n_heads": 0}, qtts.ERR_INVALID),
    ({"n_heads": 56, "q_stride": 7168, "out_stride": 7168}, qtts.OK), ({"rows": 1 << 24}, qtts.ERR_CAPACITY), ({"n_seqs": (1 << 22) + 1}, qtts.ERR_CAPACITY),
    ({"q_stride": 2000}, qtts.ERR_INVALID), ({"max_pages": 0}, qtts.ERR_INVALID), ({"table_stride": 19}, qtts.ERR_INVALID),
    ({"max_pages": 1 << 26, "table_stride": 1 << 26}, qtts.ERR_INVALID), ({"row_start": None}, qtts.ERR_INVALID),
    ({"lengths": at(4, 2)}, qtts.ERR_INVALID), ({"scale": 0.0}, qtts.ERR_INVALID), ({"scale": float("nan")}, qtts.ERR_INVALID),
    ({"scale": -1.0}, qtts.OK), ({"window": -1}, qtts.ERR_INVALID), ({"max_len": -1}, qtts.ERR_INVALID), ({"max_len": 1 << 40}, qtts.OK),
    ({"max_len": 20000, "workspace": None}, qtts.ERR_CAPACITY), ({"max_len": 20000, "workspace_bytes": 100}, qtts.ERR_CAPACITY),
    ({"max_len": 20000, "workspace": at(6, 8)}, qtts.ERR_CAPACITY), ({"max_len": 20000, "workspace": at(1)}, qtts.ERR_INVALID),
    ({"max_len": 20000, "workspace": at(0)}, qtts.ERR_INVALID),
])
def test_attention_refusals(kw, code):
    assert attend(cache(), **kw) == code


@pytest.mark.parametrize("c,code", BAD_CACHE)
def test_attention_refuses_bad_caches(c, code):
    assert attend(cache(**c)) == code
    n = ctypes.c_int64()
    assert LIB.qtts_kv4_attention_workspace(ctypes.byref(attention_args(cache(**c))), ctypes.byref(n)) == code


@pytest.mark.parametrize("rows,over", [((1 << 27) // 16, False), ((1 << 27) // 16 + 1, True)])
def test_rows_that_a_launch_can_have(rows, over):
    """16 heads: 2^27 rows x heads; what is below is refused for its overlaps
    only, the addresses here being close together."""
    assert (post(rows=rows) == qtts.ERR_CAPACITY) == over
    assert (attend(cache(), rows=rows) == qtts.ERR_CAPACITY) == over
    n = (1 << 26) // 8 + over
    assert (LIB.qtts_kv4_gather(None, ctypes.byref(cache()), at(3), n, 0, at(1), at(2), None, qtts.CHECK_ONLY) == qtts.ERR_CAPACITY) == over


def test_without_context_only_checks():
    assert LIB.qtts_kv4_attention(None, ctypes.byref(attention_args(cache())), None, 0) == qtts.ERR_INVALID
    assert LIB.qtts_kv4_gather(None, ctypes.byref(cache()), at(3), 5, 0, at(1), at(2), None, 0) == qtts.ERR_INVALID


def test_workspace_grows_with_the_split_only():
    def need(**kw):
        n = ctypes.c_int64(-1)
        assert LIB.qtts_kv4_attention_workspace(ctypes.byref(attention_args(cache(), **kw)), ctypes.byref(n)) == qtts.OK
        return n.value
    assert need(rows=1, n_seqs=1, max_len=10) == 0            # one page: nothing to split
    assert need(rows=1, n_seqs=1, max_len=16000) > 0
    assert need(rows=0, max_len=16000) == 0
    assert need(rows=1, n_seqs=1, max_len=1024) == 0          # four pages for each wave
    assert need(rows=4096, n_seqs=4096, max_len=4096) == 0    # the sequences fill the card
    assert need(rows=1, n_seqs=1, max_len=1 << 40) < 1 << 25
    assert need(rows=1, n_seqs=1, max_len=2 ** 63 - 1) == need(rows=1, n_seqs=1, max_len=2 ** 31 - 1)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("window", [0, 70, 5000])
def test_short_calls_need_no_workspace(dtype, window):
    """What the binding takes for granted up to qtts.kv4.WHOLE positions."""
    n = ctypes.c_int64(-1)
    for rows in (0, 1, 7, 300, 5000, 100000):
        for seqs in (0, 1, 2, 9, 33, 64, 257, 4000):
            a = attention_args(cache(), dtype=dtype, rows=rows, n_seqs=seqs, max_len=qtts.kv4.WHOLE, window=window)
            assert LIB.qtts_kv4_attention_workspace(ctypes.byref(a), ctypes.byref(n)) == qtts.OK and n.value == 0


def test_reference_codes():
    """Known answers of the format: the extreme value is code 0, steps of an
    eighth, halves to even, saturation, and what 8 significant bits keep."""
    x = np.zeros((1, 32))
    x[0, :6] = [8.0, -7.0, 0.5, 1.5, -0.5, 3.0]
    c, s = kv4_ref.quantise(x)
    assert s[0, 0] == -1.0 and c[0, :6].tolist() == [0, 15, 8, 6, 8, 5]
    assert kv4_ref.values(c, s)[0, :2].tolist() == [8.0, -7.0]
    x = np.zeros((1, 32))
    x[0, :3] = [4.0, -4.0, 1e9]
    c, s = kv4_ref.quantise(x)
    assert kv4_ref.values(c, s)[0, 2] == 65280.0 and s[0, 0] == -8160.0
    c, s = kv4_ref.quantise(np.where(np.arange(32) == 0, 4.0, np.where(np.arange(32) == 1, -4.0, 0.0))[None])
    assert s[0, 0] == -0.5 and c[0, :2].tolist() == [0, 15]   # of two extremes the positive one
    r = np.random.default_rng(1)
    c, s = kv4_ref.quantise(10 ** r.uniform(-4, 4, (500, 1)) * r.standard_normal((500, 64)))
    v = kv4_ref.values(c, s)
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)


def test_reference_pool_round_trip():
    r = np.random.default_rng(2)
    for dim in (64, 128):
        pool = kv4_ref.Pool(3, 2, dim, fill=0xA5)
        slots = r.permutation(3 * 64)[:100]
        k, v = r.standard_normal((2, 100, 2, dim))
        pool.put(slots, k, v)
        for x, y in zip((k, v), pool.get(slots)):
            assert np.array_equal(kv4_ref.values(*kv4_ref.quantise(x)), y)
