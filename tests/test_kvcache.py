"""What the paged cache's calls refuse, without a device: a cache over the caller's pages and no context checks its
calls' arguments and goes no further."""
import ctypes

import numpy as np
import pytest

from rust_trainer_amd import _ffi

INVALID, UNSUPPORTED = 1, 2
F32, F16, BF16 = _ffi.TYPE_F32, _ffi.TYPE_F16, _ffi.TYPE_BF16


def create(type=F16, layers=2, pages=8, page=32, kv=2, d=64, k=4096, v=8192):
    h = ctypes.c_void_p()
    st = _ffi.lib().rtq_kv_cache_create(None, type, layers, pages, page, kv, d, k, v, ctypes.byref(h))
    return st, h


@pytest.fixture
def cache():
    st, h = create()
    assert st == 0
    yield h
    _ffi.lib().rtq_kv_cache_destroy(h)


@pytest.mark.parametrize("bad, status", [
    (dict(type=F32), UNSUPPORTED), (dict(layers=0), INVALID), (dict(layers=65536), INVALID), (dict(pages=0), INVALID), (dict(pages=2 ** 31), INVALID),
    (dict(page=16), INVALID), (dict(page=48), INVALID), (dict(page=2048), INVALID), (dict(kv=0), INVALID), (dict(kv=1025), INVALID),
    (dict(d=8), INVALID), (dict(d=72), INVALID), (dict(d=272), INVALID), (dict(k=None), INVALID), (dict(k=4100), INVALID),
    (dict(k=None, v=None), INVALID), (dict(layers=65535, pages=2 ** 31 - 1, page=1024, kv=1024, d=256), INVALID)])
def test_a_cache_is_refused(bad, status):
    st, h = create(**bad)
    assert st == status and not h.value


def test_pages_of_a_layer(cache):
    k, v = ctypes.c_void_p(), ctypes.c_void_p()
    assert _ffi.lib().rtq_kv_cache_pages(cache, 1, ctypes.byref(k), ctypes.byref(v)) == 0
    assert (k.value, v.value) == (4096 + 8 * 32 * 2 * 64 * 2, 8192 + 8 * 32 * 2 * 64 * 2)
    for layer in (-1, 2):
        assert _ffi.lib().rtq_kv_cache_pages(cache, layer, ctypes.byref(k), ctypes.byref(v)) == INVALID


def seqs(lens=(3, 40), starts=(0, 2, 5), table=((0, 1), (2, 3)), **over):
    a = [np.array(x, np.int32) if x is not None else None for x in (lens, starts, table)]
    s = _ffi.RtqKvSeqs(len(lens), *[None if x is None else x.ctypes.data for x in a], len(table[0]))
    for k, v in over.items():
        setattr(s, k, v)
    s._keep = a
    return s


def rope(dim=64, base=1e4, freq_scale=1.0, neox=1, factors=None, n_factors=0, q_norm=None, k_norm=None, eps=1e-6, offset=0.0):
    return _ffi.RtqRope(dim, base, freq_scale, neox, factors, n_factors, q_norm, k_norm, eps, offset)


def append(cache, s, n=5, layer=0, type=F32, r=None, positions=None, ldk=128, ldv=128, heads=4, ldq=256, ldo=256, q=True, k=True, off=0, d=False):
    rows = np.zeros(5 * 256 + 1, np.float32)
    p = rows.ctypes.data
    args = [cache, layer, None if s is None else ctypes.byref(s), n, type, None if r is False else ctypes.byref(r or rope()),
            None if positions is None else positions.ctypes.data, p + off if k else None, ldk, p, ldv, heads, p if q else None, ldq, p, ldo]
    L = _ffi.lib()
    st = L.rtq_kv_append_d(*args, None) if d else L.rtq_kv_append(*args)
    return st, L.rtq_last_error().decode()


def attend(cache, s, n=5, layer=0, type=F32, heads=4, scale=0.0, parents=None, ldq=256, ldo=256, q=True, d=False):
    rows = np.zeros(5 * 256, np.float32)
    p = rows.ctypes.data
    args = [cache, layer, None if s is None else ctypes.byref(s), n, type, heads, scale, None if parents is None else parents.ctypes.data, p if q else None,
            ldq, p, ldo]
    L = _ffi.lib()
    st = L.rtq_kv_attend_d(*args, None) if d else L.rtq_kv_attend(*args)
    return st, L.rtq_last_error().decode()


@pytest.mark.parametrize("d", [False, True])
@pytest.mark.parametrize("what", [dict(layer=-1), dict(layer=2), dict(n=-1), dict(n=2 ** 24 + 1), dict(type=BF16), dict(type=7), dict(heads=3), dict(heads=0),
                                  dict(ldq=255), dict(ldo=255), dict(s=None)])
def test_both_refuse(cache, what, d):
    what = dict(what)
    s = what.pop("s", seqs())
    bad = UNSUPPORTED if "type" in what else INVALID
    for call in (append, attend):
        st, msg = call(cache, s, d=d, **what)
        assert st == bad and "context" not in msg, msg


@pytest.mark.parametrize("d", [False, True])
def test_what_passes_meets_the_missing_context(cache, d):
    for call in (append, attend):
        assert call(cache, seqs(), d=d) == (INVALID, "null context")
        assert call(cache, seqs(starts=None), n=4, d=d) == (INVALID, "null context")
        assert call(None, seqs(), d=d) == (INVALID, "null cache")


@pytest.mark.parametrize("over", [dict(b=0), dict(b=65537), dict(ld=-1), dict(ld=2 ** 30 + 1), dict(lens=None), dict(table=None)])
def test_sequences_are_refused(cache, over):
    for d in (False, True):
        for call in (append, attend):
            st, msg = call(cache, _with(over), d=d)
            assert st == INVALID and "context" not in msg, msg


def _with(over):
    s = seqs()
    for k, v in over.items():
        setattr(s, k, v)
    return s


def test_rows_need_starts_or_equal_shares(cache):
    for call in (append, attend):
        st, msg = call(cache, seqs(starts=None), n=5)
        assert st == INVALID and "starts" in msg


@pytest.mark.parametrize("s, word", [(dict(starts=(0, 3, 2)), "rows"), (dict(starts=(-1, 2, 5)), "rows"), (dict(starts=(0, 2, 6)), "rows"), (dict(lens=(-1, 0)), "holds"),
                                     (dict(lens=(3, 62)), "table"), (dict(table=((0, 1), (2, 8))), "page"), (dict(table=((-1, 1), (2, 3))), "page")])
def test_the_host_versions_refuse_lists(cache, s, word):
    for call in (append, attend):
        st, msg = call(cache, seqs(**s))
        assert st == INVALID and word in msg, msg


@pytest.mark.parametrize("what", [dict(r=False), dict(r=rope(dim=65)), dict(r=rope(dim=66)), dict(r=rope(dim=-2)), dict(r=rope(base=0.0)), dict(r=rope(base=float("inf"))),
                                  dict(r=rope(freq_scale=float("nan"))), dict(r=rope(n_factors=1)), dict(r=rope(factors=64, n_factors=33)),
                                  dict(r=rope(q_norm=64, eps=-1.0)), dict(r=rope(k_norm=64, offset=float("nan"))), dict(k=False), dict(ldk=127), dict(ldv=127), dict(off=2)])
@pytest.mark.parametrize("d", [False, True])
def test_append_refuses(cache, what, d):
    st, msg = append(cache, seqs(), d=d, **what)
    assert st == INVALID and "context" not in msg, msg


def test_append_refuses_negative_positions_on_the_host(cache):
    st, msg = append(cache, seqs(), positions=np.array([0, 1, -1, 3, 4], np.int32))
    assert st == INVALID and "position" in msg


@pytest.mark.parametrize("scale", [-1.0, float("nan"), float("inf"), 3e38])
def test_attend_refuses_scales(cache, scale):
    for d in (False, True):
        st, msg = attend(cache, seqs(), scale=scale, d=d)
        assert st == INVALID and "scale" in msg


@pytest.mark.parametrize("parents", [(0, 0, -1, 0, 1), (-1, 0, -1, 0, 2), (-1, 0, -3, 0, 1), (-1, 1, -1, 0, 1)])
def test_attend_refuses_parents_on_the_host(cache, parents):
    st, msg = attend(cache, seqs(), parents=np.array(parents, np.int32))
    assert st == INVALID and "parent" in msg


def test_unused_nodes_pass(cache):
    assert attend(cache, seqs(), parents=np.array((-1, 0, -2, 0, -1), np.int32)) == (INVALID, "null context")


def test_a_large_tree_is_refused_on_the_host():
    st, h = create(pages=64)
    n = 1025
    rows = np.zeros((n, 256), np.float32)
    s = seqs(lens=(0,), starts=(0, n), table=(tuple(range(33)),))
    par = np.arange(-1, n - 1, dtype=np.int32)
    st = _ffi.lib().rtq_kv_attend(h, 0, ctypes.byref(s), n, F32, 4, 0.0, par.ctypes.data, rows.ctypes.data, 256, rows.ctypes.data, 256)
    assert st == INVALID and "tree" in _ffi.lib().rtq_last_error().decode()
    st = _ffi.lib().rtq_kv_attend(h, 0, ctypes.byref(s), n, F32, 4, 0.0, None, rows.ctypes.data, 256, rows.ctypes.data, 256)
    assert st == INVALID and "context" in _ffi.lib().rtq_last_error().decode()  # a run may be longer
    _ffi.lib().rtq_kv_cache_destroy(h)


def test_calls_of_more_threads_than_a_launch_holds():
    st, h = create(kv=1024, d=16)
    L, b, n = _ffi.lib(), 65536, 65536
    lens, table = np.zeros(b, np.int32), np.zeros((b, 1), np.int32)
    s = _ffi.RtqKvSeqs(b, lens.ctypes.data, None, table.ctypes.data, 1)
    p, ld = lens.ctypes.data, 1024 * 16
    for n_big, call in ((n, lambda n: L.rtq_kv_attend_d(h, 0, ctypes.byref(s), n, F32, 1024, 0.0, None, p, ld, p, ld, None)),
                        (2 ** 20, lambda n: L.rtq_kv_append_d(h, 0, ctypes.byref(s), n, F32, ctypes.byref(rope(dim=16)), None, p, ld, p, ld, 0, None, 0, None, 0, None)),
                        (0, lambda n: L.rtq_kv_keep_d(h, ctypes.byref(s), p, 1, None, None))):
        assert call(n_big) == UNSUPPORTED and "workgroups" in L.rtq_last_error().decode()
    s.b = 4096
    assert L.rtq_kv_keep_d(h, ctypes.byref(s), p, 1, None, None) == INVALID and "context" in L.rtq_last_error().decode()
    L.rtq_kv_cache_destroy(h)


def keep(cache, s, kept, ldk=None, after=True, d=False, alias=False):
    a = np.array(kept, np.int32)
    out = np.zeros(2, np.int32)
    p = s._keep[0].ctypes.data + 4 if alias else out.ctypes.data
    L = _ffi.lib()
    args = [cache, ctypes.byref(s), a.ctypes.data, ldk if ldk is not None else a.shape[1], p if after else None]
    return (L.rtq_kv_keep_d(*args, None) if d else L.rtq_kv_keep(*args)), L.rtq_last_error().decode()


def test_keep_refuses(cache):
    ok = ((0, 2, -1), (1, -1, -1))
    for d in (False, True):
        assert keep(cache, seqs(), ok, d=d) == (INVALID, "null context")
        assert keep(cache, seqs(), ok, after=False, d=d) == (INVALID, "null context")
        for bad in (dict(ldk=0), dict(ldk=1025), dict(alias=True)):
            st, msg = keep(cache, seqs(), ok, d=d, **bad)
            assert st == INVALID and "context" not in msg, msg
        assert keep(cache, _with(dict(b=0)), ok, d=d)[0] == INVALID
    for kept in (((0, 0, -1), (1, -1, -1)), ((2, 1, -1), (1, -1, -1)), ((0, -2, -1), (1, -1, -1)), ((0, 61, -1), (1, -1, -1))):
        st, msg = keep(cache, seqs(), kept)
        assert st == INVALID and "kept" in msg, msg
    st, msg = keep(cache, seqs(table=((0, 9), (2, 3))), ((30, -1), (1, -1)))
    assert st == INVALID and "page" in msg


def test_rows_of_no_sequence_are_not_looked_at(cache):
    """Positions of rows before the first sequence and behind the last may be anything."""
    for starts, pos in (((0, 2, 4), (0, 1, 2, 3, -1)), ((1, 2, 5), (-7, 1, 2, 3, 4))):
        assert append(cache, seqs(starts=starts), positions=np.array(pos, np.int32)) == (INVALID, "null context")
    st, msg = append(cache, seqs(starts=(1, 2, 5)), positions=np.array((0, 1, 2, 3, -1), np.int32))
    assert st == INVALID and "position" in msg


def test_sequences_longer_than_the_attention_looks_are_refused():
    """2^30 slots pass, one more does not (one page stands for all of a table's)."""
    st, h = create(pages=1, page=1024, kv=1, d=16)
    table = np.zeros((1, 2 ** 20 + 1), np.int32)
    L = _ffi.lib()
    for held, word in ((2 ** 30 - 2, "context"), (2 ** 30 - 1, "table")):
        lens, starts = np.array([held], np.int32), np.array([0, 2], np.int32)
        s = _ffi.RtqKvSeqs(1, lens.ctypes.data, starts.ctypes.data, table.ctypes.data, table.shape[1])
        for call, what in ((append, dict(r=rope(dim=16))), (attend, {})):
            st, msg = call(h, s, n=2, heads=1, **what)
            assert st == INVALID and word in msg, msg
        kept, after = np.array([[1]], np.int32), np.zeros(1, np.int32)
        st = L.rtq_kv_keep(h, ctypes.byref(s), kept.ctypes.data, 1, after.ctypes.data)
        assert st == INVALID and ("context" if word == "context" else "kept") in L.rtq_last_error().decode()
    L.rtq_kv_cache_destroy(h)
