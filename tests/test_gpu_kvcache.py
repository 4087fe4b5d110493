"""The paged cache's operators on the GPU against their definitions in 64 bits: appending with the rotation, attention of
runs and trees, keeping accepted tokens, and a run of them together."""
import numpy as np
import pytest

import rust_trainer_amd as rt
from kv_cases import EPS, TINY, TYPES, Layout, attend, norm, one_plane, rotate, to_type, tree, value, visible
from rust_trainer_amd.kvcache import KvCache, Rope, Seqs, rope_d, seqs_d

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
TT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.int16}
PAIRS = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]  # rows, cache


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def host(t, ty):
    a = t.cpu().numpy()
    return a.view(np.uint16) if ty == "bf16" else a


def rows_d(a, gap=0, off=0):
    """An array's rows on the device, `gap` elements further apart than they are long, `off` elements into an allocation."""
    n, w = a.shape
    t = dev(a)
    out = torch.zeros(off + n * (w + gap), dtype=t.dtype, device="cuda")
    v = out[off:].as_strided((n, w), (w + gap, 1))
    v.copy_(t)
    return v


class Pages:
    """A cache over torch tensors, filled with numbers (or NaN)."""

    def __init__(self, ctx, lay, kv, d, ct, layers=1, seed=0, fill=None):
        rng = np.random.default_rng(seed + 99)
        self.ct, self.kv, self.d, self.lay = ct, kv, d, lay
        ks, vs = (layers, lay.n_pages, kv, lay.page, d), (layers, lay.n_pages, kv, d, lay.page)
        self.k0 = to_type(rng.standard_normal(ks) if fill is None else np.full(ks, fill), ct)
        self.v0 = to_type(rng.standard_normal(vs) if fill is None else np.full(vs, fill), ct)
        self.k, self.v = dev(self.k0), dev(self.v0)
        self.cache = KvCache(layers, lay.n_pages, lay.page, kv, d, type=TYPES[ct], ctx=ctx, pages_d=(self.k.data_ptr(), self.v.data_ptr()))
        self.lens, self.starts, self.table = dev(lay.lens), dev(lay.starts), dev(lay.table)
        self.seqs = seqs_d(lay.b, self.lens.data_ptr(), self.table.data_ptr(), lay.table.shape[1], self.starts.data_ptr())

    def rows(self, i, count=None, layer=0, now=False):
        """(keys, values) [slots x kv x d] of sequence i, in 64 bits."""
        p, s = self.lay.slots(i, count)
        k, v = (host(self.k, self.ct), host(self.v, self.ct)) if now else (self.k0, self.v0)
        return value(k[layer][p, :, s], self.ct), value(v[layer][p, :, :, s], self.ct)


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ append
APPEND = [  # lens, counts, heads, kv, d, rot, neox, normed, page, gap, off, far
    ([5], [1], 4, 2, 128, 128, True, True, 64, 0, 0, False),
    ([0, 31, 32, 7], [3, 1, 40, 0], 6, 3, 80, 32, True, False, 32, 5, 1, False),
    ([100, 0], [33, 65], 5, 5, 64, 64, False, True, 32, 0, 0, True),
    ([9, 2], [2, 2], 8, 1, 256, 256, True, True, 128, 3, 3, True),
    ([1], [7], 2, 2, 96, 44, True, True, 32, 1, 0, False),   # a rotation that ends inside eight elements
    ([1], [7], 2, 2, 48, 6, False, False, 32, 1, 0, True),
    ([63], [2], 3, 3, 16, 0, False, False, 64, 0, 0, False),  # none
    ([40] * 70, [1] * 70, 2, 1, 32, 32, True, False, 32, 0, 0, False),
]


@pytest.mark.parametrize("xt, ct", PAIRS)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(ctx, case, xt, ct):
    lens, counts, heads, kv, d, rot, neox, normed, page, gap, off, far = APPEND[case]
    lay = Layout(lens, counts, page, seed=case)
    rng = np.random.default_rng(case)
    pg = Pages(ctx, lay, kv, d, ct, seed=case)
    n, extra = lay.n, 2  # rows behind the last sequence
    mk = lambda h: to_type(rng.standard_normal((n + extra, h * d)), xt)
    q, k, v = mk(heads), mk(kv), mk(kv)
    qn, kn = (to_type(rng.uniform(0.5, 1.5, (2, d)), "f32")) if normed else (None, None)
    seq = np.repeat(np.arange(lay.b), lay.counts)
    idx = np.arange(n) - lay.starts[seq]
    slot = lay.lens[seq] + idx
    pos = rng.integers(0, 1 << 20, n + extra).astype(np.int32) if far else None
    factors = rng.uniform(0.5, 8.0, rot // 4).astype(np.float32) if case % 2 and rot else None
    base, scale, eps, offset = 5e5, 0.25 if far else 1.0, 1e-6, 1.0 if case == 2 else 0.0
    qd, kd, vd = rows_d(q, gap, off), rows_d(k, gap, off), rows_d(v, gap, off)
    out = rows_d(np.full((n + extra, heads * d), 7, NP[xt]), gap, off)
    qnd, knd = (dev(qn), dev(kn)) if normed else (None, None)
    r = rope_d(rot, base, neox, scale, factors, qnd.data_ptr() if normed else 0, knd.data_ptr() if normed else 0, eps, offset)
    pd = dev(pos) if far else None
    pg.cache.append_d(0, pg.seqs, n + extra, TYPES[xt], r, kd.data_ptr(), kd.stride(0), vd.data_ptr(), vd.stride(0), heads, qd.data_ptr(), qd.stride(0),
                      out.data_ptr(), out.stride(0), 0 if pd is None else pd.data_ptr(), stream())
    torch.cuda.synchronize()
    at = pos[:n] if far else slot

    def want(x, h, w):
        x = value(x[:n], xt).reshape(n, h, d)
        y = rotate(norm(x, w, eps, offset), at, rot, base, neox, scale, factors)
        size = np.abs(norm(x, w, eps, offset))
        if rot:  # the other side of each pair
            i = np.arange(rot // 2)
            ia, ib = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
            pair = size[..., ia] + size[..., ib]
            size[..., ia] = size[..., ib] = pair
        # turns rounded to 2^-26 (2 pi of that), sine and cosine and two products and their sum in 32 bits; the norm: squares
        # summed by 16 lanes and their roots and quotient
        return y, size * ((6.3 * 2.0 ** -26 + 5 * 2.0 ** -24 if rot else 0.0) + ((d / 16 + 12) * 2.0 ** -24 if normed else 0.0))

    yq, bq = want(q, heads, qn)
    got = host(out, xt)
    assert np.all(got[n:] == 7), "rows behind the last sequence were written"
    err = np.abs(value(got[:n], xt).reshape(n, heads, d) - yq)
    assert np.all(err <= bq + EPS[xt] * (np.abs(yq) + bq) + TINY[xt]), (err - bq).max()
    yk, bk = want(k, kv, kn)
    yv = value(v[:n], xt).reshape(n, kv, d)
    page_id, in_page = lay.table[seq, slot // page], slot % page
    k1, v1 = host(pg.k, ct), host(pg.v, ct)
    gk, gv = value(k1[0][page_id, :, in_page], ct), value(v1[0][page_id, :, :, in_page], ct)
    assert np.all(np.abs(gk - yk) <= bk + EPS[ct] * (np.abs(yk) + bk) + TINY[ct])
    assert np.all(np.abs(gv - yv) <= EPS[ct] * np.abs(yv) + TINY[ct])
    k1[0][page_id, :, in_page] = pg.k0[0][page_id, :, in_page]
    v1[0][page_id, :, :, in_page] = pg.v0[0][page_id, :, :, in_page]
    assert np.array_equal(k1, pg.k0) and np.array_equal(v1, pg.v0), "other slots were written"


def test_append_host_in_place_and_alone(ctx):
    """The host call, the device call, queries written over themselves and no queries at all: the same cache."""
    lay = Layout([5, 40], [3, 30], 32, seed=1)
    rng = np.random.default_rng(2)
    kv, d, heads, n = 2, 64, 4, 33
    q, k, v = [rng.standard_normal((n, h * d)).astype(np.float32) for h in (heads, kv, kv)]
    qn, kn = rng.uniform(0.5, 1.5, (2, d)).astype(np.float32)
    a, b, c = [Pages(ctx, lay, kv, d, "f16", layers=2) for _ in range(3)]
    out = a.cache.append(1, Seqs(lay.lens, lay.table, lay.starts), k, v, Rope(64, 1e6, q_norm=qn, k_norm=kn), q=q)
    qd, kd, vd, qnd, knd = dev(q), dev(k), dev(v), dev(qn), dev(kn)
    r = rope_d(64, 1e6, q_norm_ptr=qnd.data_ptr(), k_norm_ptr=knd.data_ptr())
    b.cache.append_d(1, b.seqs, n, 0, r, kd.data_ptr(), kv * d, vd.data_ptr(), kv * d, heads, qd.data_ptr(), heads * d, qd.data_ptr(), heads * d, stream=stream())
    c.cache.append_d(1, c.seqs, n, 0, r, kd.data_ptr(), kv * d, vd.data_ptr(), kv * d, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(out, qd.cpu().numpy())
    for x in (b, c):
        assert torch.equal(a.k, x.k) and torch.equal(a.v, x.v)
    assert np.array_equal(host(a.k, "f16")[0], a.k0[0])  # the other layer


def test_append_skips_pages_that_are_not_there(ctx):
    lay = Layout([30, 10], [5, 2], 32, seed=3)
    pg = Pages(ctx, lay, 2, 64, "f16")
    pages = lay.table[0, 1], lay.table[1, 0]
    table = lay.table.copy()
    table[0, 1], table[1, 0] = pg.lay.n_pages, -5
    pg.table.copy_(dev(table))
    x = rows_d(np.ones((7, 128), np.float32))
    pg.cache.append_d(0, pg.seqs, 7, 0, rope_d(64), x.data_ptr(), 128, x.data_ptr(), 128, stream=stream())
    short = seqs_d(2, pg.lens.data_ptr(), pg.table.data_ptr(), 0, pg.starts.data_ptr())
    pg.cache.append_d(0, short, 7, 0, rope_d(64), x.data_ptr(), 128, x.data_ptr(), 128, stream=stream())  # no pages at all
    torch.cuda.synchronize()
    k1, v1 = host(pg.k, "f16"), host(pg.v, "f16")
    for p in pages:
        assert np.array_equal(k1[0][p], pg.k0[0][p]) and np.array_equal(v1[0][p], pg.v0[0][p])
    first = lay.table[0, 0]
    assert np.all(v1[0][first, :, :, 30:] == 1) and np.array_equal(v1[0][first, :, :, :30], pg.v0[0][first, :, :, :30])


# ------------------------------------------------------------------ attend
ATTEND = [  # lens, counts, heads, kv, d, page, tree, gap, off
    ([1], [1], 2, 2, 64, 32, False, 0, 0),
    ([0], [1], 4, 2, 128, 32, False, 0, 0),
    ([31, 32, 33, 0, 128], [1, 1, 1, 1, 1], 8, 2, 128, 32, False, 0, 0),
    ([500, 0, 1300], [1, 0, 1], 7, 1, 64, 64, False, 3, 1),
    ([200, 77, 0, 5], [9, 16, 17, 0], 6, 3, 80, 32, True, 5, 1),
    ([60, 300], [33, 64], 8, 2, 128, 64, True, 0, 0),
    ([3], [100], 4, 4, 96, 32, False, 0, 0),
    ([130], [70], 16, 2, 64, 128, False, 0, 0),
    ([2100, 40], [2, 3], 4, 2, 256, 256, True, 1, 0),
    ([10], [90], 2, 1, 256, 32, False, 0, 0),
    ([5] * 130, [1] * 130, 2, 2, 32, 32, False, 0, 0),
    ([40] * 66 + [700], [2] * 66 + [5], 2, 1, 16, 32, True, 0, 0),
    ([3000], [1], 32, 8, 128, 128, False, 0, 0),
    ([20, 5], [3, 1], 200, 1, 64, 32, False, 0, 0),  # more query heads a KV head than a tile has rows
    ([50], [60], 6, 2, 16, 32, False, 0, 0),
    ([50, 0], [60, 33], 6, 2, 48, 1024, True, 0, 0),
    ([33], [45], 4, 1, 112, 32, True, 2, 1),
    ([700, 900], [40, 40], 8, 1, 64, 32, True, 0, 0),
    ([1500], [50], 8, 2, 256, 64, False, 0, 0),
    ([3] * 3000, [1] * 3000, 1, 1, 16, 32, False, 0, 0),
    ([515, 130, 511, 512, 513], [1] * 5, 5, 1, 128, 32, False, 0, 0),
]


def check_attend(pg, lay, got, q, xt, heads, parents, scale=0.0):
    weights = one_plane(xt, q.shape[0], lay.b, heads, pg.kv, pg.d)
    for i in range(lay.b):
        a, z = lay.starts[i], lay.starts[i + 1]
        if a == z:
            continue
        k, v = pg.rows(i)
        want, bound = attend(value(q[a:z], xt), k, v, int(lay.lens[i]), heads, None if parents is None else parents[a:z], scale, weights)
        err = np.abs(value(got[a:z], xt) - want)
        lim = bound + EPS[xt] * (np.abs(want) + bound) + TINY[xt]
        assert np.all(err <= lim), (i, (err / lim).max())


@pytest.mark.parametrize("xt, ct", PAIRS)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(ctx, case, xt, ct):
    lens, counts, heads, kv, d, page, is_tree, gap, off = ATTEND[case]
    lay = Layout(lens, counts, page, seed=case)
    rng = np.random.default_rng(case)
    pg = Pages(ctx, lay, kv, d, ct, seed=case)
    n, extra = lay.n, 1
    q = to_type(2.0 * rng.standard_normal((n + extra, heads * d)), xt)
    parents = np.array([p for m in counts for p in tree(rng, m)[0]] + [0] * extra, np.int32) if is_tree else None
    qd, out = rows_d(q, gap, off), rows_d(np.full((n + extra, heads * d), 7, NP[xt]), gap, off)
    pd = dev(parents) if is_tree else None
    scale = 0.05 if case % 3 == 1 else 0.0
    pg.cache.attend_d(0, pg.seqs, n + extra, TYPES[xt], heads, qd.data_ptr(), qd.stride(0), out.data_ptr(), out.stride(0), pd.data_ptr() if is_tree else 0, scale,
                      stream())
    torch.cuda.synchronize()
    got = host(out, xt)
    assert np.all(got[n:] == 7), "rows behind the last sequence were written"
    check_attend(pg, lay, got, q, xt, heads, parents, scale)


@pytest.mark.parametrize("first, counts", [(70, [20, 6, 40]), (2500, [20, 6, 40]), (1500, [6, 6, 5])])
@pytest.mark.parametrize("xt, ct", PAIRS)
def test_what_is_not_seen_does_not_matter(ctx, xt, ct, first, counts):
    """NaN in every slot that holds no token, and NaN and infinities in the keys and values of tokens that others do not see:
    in tiles of one part and of several."""
    lens, heads, kv, d = [first, 3, 0], 4, 2, 128
    lay = Layout(lens, counts, 32, seed=5)
    rng = np.random.default_rng(6)
    pg = Pages(ctx, lay, kv, d, ct, fill=np.nan)
    parents = np.array([p for m in counts for p in tree(rng, m)[0]], np.int32)
    bad = {0: [4, counts[0] - 1], 1: [5], 2: [counts[2] - 1, counts[2] // 2]}
    for i in range(3):
        p, s = lay.slots(i)
        pg.k0[0][p, :, s] = to_type(rng.standard_normal((p.size, kv, d)), ct)
        pg.v0[0][p, :, :, s] = to_type(rng.standard_normal((p.size, kv, d)), ct)
        for j, node in enumerate(bad[i]):
            at = lens[i] + node
            what = to_type(np.array([np.nan, np.inf, -np.inf]), ct)[j % 3]
            pg.k0[0][p[at], :, s[at], ::2] = what
            pg.v0[0][p[at], :, 1::3, s[at]] = to_type(np.array([-np.inf, np.nan, np.inf]), ct)[j % 3]
    pg.k.copy_(dev(pg.k0)), pg.v.copy_(dev(pg.v0))
    q = to_type(rng.standard_normal((lay.n, heads * d)), xt)
    for par in (parents, None):
        out = rows_d(np.zeros((lay.n, heads * d), NP[xt]))
        qd, pd = rows_d(q), dev(parents)
        pg.cache.attend_d(0, pg.seqs, lay.n, TYPES[xt], heads, qd.data_ptr(), heads * d, out.data_ptr(), heads * d, pd.data_ptr() if par is not None else 0, 0.0, stream())
        torch.cuda.synchronize()
        got = value(host(out, xt), xt)
        for i in range(3):
            a, m = lay.starts[i], counts[i]
            seen, _ = visible(m, None if par is None else par[a:a + m])
            hit = seen[:, bad[i]].any(1)
            assert not np.isfinite(got[a:a + m][hit]).all(1).any(), "a row that sees NaN is NaN"
            k, v = pg.rows(i)
            want, bound = attend(value(q[a:a + m], xt), k, v, lens[i], heads, None if par is None else par[a:a + m],
                                 weights=one_plane(xt, lay.n, 3, heads, kv, d))
            err = np.abs(got[a:a + m] - want)[~hit]
            assert np.all(err <= (bound + EPS[xt] * (np.abs(want) + bound) + TINY[xt])[~hit])


@pytest.mark.parametrize("value_, where", [(np.inf, "v"), (-np.inf, "v"), (np.nan, "v")])
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(ctx, value_, where):
    lay = Layout([40], [5], 32)
    pg = Pages(ctx, lay, 1, 64, "f16")
    p, s = lay.slots(0)
    pg.v[0, p[42], 0, 9, s[42]] = value_
    q = rows_d(np.random.default_rng(0).standard_normal((5, 64)).astype(np.float32))
    out = torch.zeros(5, 64, device="cuda")
    pg.cache.attend_d(0, pg.seqs, 5, 0, 1, q.data_ptr(), 64, out.data_ptr(), 64, 0, 0.0, stream())
    got = out.cpu().numpy()
    assert np.isfinite(got[:2]).all() and np.isfinite(np.delete(got, 9, 1)).all()
    assert all(np.isnan(x) if np.isnan(value_) else x == value_ for x in got[2:, 9])


@pytest.mark.parametrize("xt, ct", PAIRS)
def test_infinities_that_are_seen(ctx, xt, ct):
    """An infinite value is its column's sum, an infinite key leaves its row one key less or NaN, as in the formula."""
    lay = Layout([700], [1], 32)
    pg = Pages(ctx, lay, 1, 64, ct)
    rng = np.random.default_rng(0)
    q = to_type(np.abs(rng.standard_normal((1, 128))) + 0.1, xt)
    q[:, 64:] = to_type(-np.abs(rng.standard_normal((1, 64))) - 0.1, xt)  # the second head: the signs turned
    p, s = lay.slots(0)
    pg.v0[0][p[100], 0, 5, s[100]], pg.v0[0][p[300], 0, 6, s[300]] = to_type(np.array([np.inf, -np.inf]), ct)
    pg.k0[0][p[500], 0, s[500]] = to_type(np.array([-np.inf]), ct)[0]
    pg.k.copy_(dev(pg.k0)), pg.v.copy_(dev(pg.v0))
    qd, out = rows_d(q), rows_d(np.zeros((1, 128), NP[xt]))
    pg.cache.attend_d(0, pg.seqs, 1, TYPES[xt], 2, qd.data_ptr(), 128, out.data_ptr(), 128, 0, 0.0, stream())
    got = value(host(out, xt), xt).reshape(2, 64)
    assert got[0, 5] == np.inf and got[0, 6] == -np.inf and np.isfinite(np.delete(got[0], (5, 6))).all()
    assert np.isnan(got[1]).all()
    k, v = pg.rows(0)
    k, v = np.delete(k, 500, 0), np.delete(v, 500, 0)
    v[~np.isfinite(v)] = 0
    want, bound = attend(value(q, xt)[:, :64], k, v, 699, 1)
    err = np.delete(np.abs(got[0] - want[0]) - bound[0] - EPS[xt] * (np.abs(want[0]) + bound[0]), (5, 6))
    assert (err <= 0).all()


@pytest.mark.parametrize("long", [False, True])
def test_rows_that_see_nothing_are_zero(ctx, long):
    """Unused nodes and what hangs from them, keys of -inf alone, pages that are not there, a tree that is too large."""
    held = 4000 if long else 20
    lay = Layout([held, 0], [6, 2], 32)
    pg = Pages(ctx, lay, 2, 64, "bf16")
    q = rows_d(np.random.default_rng(1).standard_normal((8, 256)).astype(np.float32))
    par = dev(np.array([-1, -2, 1, 0, 7, 3, -1, 1], np.int32))  # 1: unused, 2 hangs from it, 4: after itself; 7: itself
    out = torch.full((8, 256), 7.0, device="cuda")
    run = lambda s, p: (pg.cache.attend_d(0, s, 8, 0, 4, q.data_ptr(), 256, out.data_ptr(), 256, p, 0.0, stream()), torch.cuda.synchronize())
    run(pg.seqs, par.data_ptr())
    zero = (out == 0).all(1).tolist()
    assert zero == [False, True, True, False, True, False, False, True]
    none = seqs_d(2, pg.lens.data_ptr(), pg.table.data_ptr(), 0, pg.starts.data_ptr())
    out.fill_(7.0)
    run(none, 0)
    assert (out == 0).all()
    # pages of the held tokens that are not there: the rows are those of a sequence without them
    table = lay.table.copy()
    table[0, :held // 32] = [-1, pg.lay.n_pages, 2 ** 31 - 1, -2 ** 31][:1] * (held // 32)
    pg.table.copy_(dev(table))
    run(pg.seqs, 0)
    k, v = pg.rows(0)
    lo = held // 32 * 32
    want, bound = attend(q.cpu().numpy()[:6].astype(np.float64), k[lo:], v[lo:], held - lo, 4)
    assert np.all(np.abs(out.cpu().numpy()[:6] - want) <= bound + EPS["f32"] * (np.abs(want) + bound))
    pg.table.copy_(dev(lay.table))
    pg.k.fill_(-128)  # bf16 -inf (0xff80)
    q.copy_(q.abs())
    run(pg.seqs, 0)
    assert (out == 0).all()


def test_a_tree_that_is_too_large_gives_zeros(ctx):
    lay = Layout([8, 8], [1025, 3], 64)
    pg = Pages(ctx, lay, 1, 64, "f16")
    q = torch.randn(lay.n, 64, device="cuda")
    par = torch.tensor(list(range(-1, 1024)) + [-1, 0, 1], dtype=torch.int32, device="cuda")
    out = torch.full((lay.n, 64), 7.0, device="cuda")
    pg.cache.attend_d(0, pg.seqs, lay.n, 0, 1, q.data_ptr(), 64, out.data_ptr(), 64, par.data_ptr(), 0.0, stream())
    torch.cuda.synchronize()
    assert (out[:1025] == 0).all() and (out[1025:] != 0).any(1).all()


def test_the_largest_tree_is_a_run_when_it_is_one(ctx):
    """1024 nodes in one branch, and the same tokens as a run: the same rows, to the bit."""
    lay = Layout([70], [1024], 64)
    pg = Pages(ctx, lay, 2, 64, "f16")
    q = torch.randn(1024, 256, device="cuda")
    par = torch.arange(-1, 1023, dtype=torch.int32, device="cuda")
    a, b = torch.zeros(1024, 256, device="cuda"), torch.zeros(1024, 256, device="cuda")
    pg.cache.attend_d(0, pg.seqs, 1024, 0, 4, q.data_ptr(), 256, a.data_ptr(), 256, par.data_ptr(), 0.0, stream())
    pg.cache.attend_d(0, pg.seqs, 1024, 0, 4, q.data_ptr(), 256, b.data_ptr(), 256, 0, 0.0, stream())
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e30])
def test_queries_of_any_size(ctx, size):
    """f32 queries far outside f16's range, over keys that bring the scores back into a usual one."""
    lay = Layout([300], [2], 32)
    rng = np.random.default_rng(3)
    pg = Pages(ctx, lay, 1, 64, "f16", seed=4)
    q = (rng.standard_normal((2, 128)) * size).astype(np.float32)
    qd, out = rows_d(q), torch.zeros(2, 128, device="cuda")
    scale = float(np.float32(0.125 / size))
    pg.cache.attend_d(0, pg.seqs, 2, 0, 2, qd.data_ptr(), 128, out.data_ptr(), 128, 0, scale, stream())
    torch.cuda.synchronize()
    check_attend(pg, lay, out.cpu().numpy(), q, "f32", 2, None, scale)


def test_small_weights_keep_their_bits(ctx):
    """One key far above thousands of others: their share, of weights near 2^-17, is right."""
    lay = Layout([6000], [1], 64)
    pg = Pages(ctx, lay, 1, 64, "f16", seed=4)
    p, s = lay.slots(0)
    pg.k0[0][:] = 0
    pg.k0[0][p[17], 0, s[17]] = 1.0
    pg.v0[0][:] = (1 + np.random.default_rng(0).uniform(0, 1, pg.v0[0].shape)).astype(np.float16)
    pg.v0[0][p[17], 0, :, s[17]] = 0.0
    pg.k.copy_(dev(pg.k0)), pg.v.copy_(dev(pg.v0))
    q = np.full((1, 64), 12 / 64, np.float32)
    qd, out = rows_d(q), torch.zeros(1, 64, device="cuda")
    pg.cache.attend_d(0, pg.seqs, 1, 0, 1, qd.data_ptr(), 64, out.data_ptr(), 64, 0, 1.0, stream())
    torch.cuda.synchronize()
    check_attend(pg, lay, out.cpu().numpy(), q, "f32", 1, None, 1.0)


def test_attend_host_in_place_and_streams(ctx):
    """The host call, the device call on a stream of its own, and rows written over the queries: the same bits."""
    lay = Layout([900, 40, 3], [4, 9, 2], 64, seed=2)
    rng = np.random.default_rng(2)
    pg = Pages(ctx, lay, 2, 128, "f16")
    q = rng.standard_normal((15, 4 * 128)).astype(np.float16)
    par = np.concatenate([tree(rng, m)[0] for m in (4, 9, 2)]).astype(np.int32)
    want = pg.cache.attend(0, Seqs(lay.lens, lay.table, lay.starts), q, parents=par)
    qd, pd = rows_d(q), dev(par)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        pg.cache.attend_d(0, pg.seqs, 15, 1, 4, qd.data_ptr(), 512, qd.data_ptr(), 512, pd.data_ptr(), 0.0, side.cuda_stream)
    side.synchronize()
    assert np.array_equal(qd.cpu().numpy(), want)
    check_attend(pg, lay, want, q, "f16", 4, par)


def test_offsets_past_32_bits(ctx):
    """The last pages of a pool of more than 2^32 elements, written and read."""
    page, kv, d = 1024, 8, 128
    n_pages = 2 ** 32 // (page * kv * d) + 3
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("not enough device memory")
    k = torch.zeros(n_pages, kv, page, d, dtype=torch.float16, device="cuda")
    v = torch.zeros(n_pages, kv, d, page, dtype=torch.float16, device="cuda")
    cache = KvCache(1, n_pages, page, kv, d, ctx=ctx, pages_d=(k.data_ptr(), v.data_ptr()))
    last = n_pages - 1
    rng = np.random.default_rng(0)
    rows = {h: rng.standard_normal((40, h * d)).astype(np.float16) for h in (16, 8)}
    s = Seqs([1000], [[last, n_pages - 2]], [0, 40])
    held = rng.standard_normal((2, 1000, kv, d)).astype(np.float16)
    k[last, :, :1000] = torch.from_numpy(held[0].transpose(1, 0, 2).copy()).cuda()
    v[last, :, :, :1000] = torch.from_numpy(held[1].transpose(1, 2, 0).copy()).cuda()
    cache.append(0, s, rows[8], rows[8][::-1].copy(), Rope(0), q=rows[16])
    got = cache.attend(0, s, rows[16])
    assert torch.equal(k[last, :, 1000:].cpu(), torch.from_numpy(rows[8][:24].reshape(24, kv, d).transpose(1, 0, 2).copy()))
    assert torch.equal(v[n_pages - 2, :, :, :16].cpu(), torch.from_numpy(rows[8][::-1][24:].reshape(16, kv, d).transpose(1, 2, 0).copy()))
    kk = np.concatenate((held[0], rows[8].reshape(40, kv, d))).astype(np.float64)
    vv = np.concatenate((held[1], rows[8][::-1].reshape(40, kv, d))).astype(np.float64)
    want, bound = attend(rows[16].astype(np.float64), kk, vv, 1000, 16, weights=one_plane("f16", 40, 1, 16, 8, 128))
    assert np.all(np.abs(got - want) <= bound + EPS["f16"] * (np.abs(want) + bound) + TINY["f16"])
    cache.close()


def test_rows_of_no_sequence(ctx):
    """Rows before the first sequence, behind the last, and a call whose sequences have none."""
    lay = Layout([40, 7], [3, 2], 32)
    kv, d, heads = 2, 64, 4
    rng = np.random.default_rng(1)
    q, k, v = [rng.standard_normal((9, h * d)).astype(np.float32) for h in (heads, kv, kv)]
    a, b = Pages(ctx, lay, kv, d, "f16"), Pages(ctx, lay, kv, d, "f16")
    shifted = dev(lay.starts + 2)
    sa = seqs_d(2, a.lens.data_ptr(), a.table.data_ptr(), lay.table.shape[1], shifted.data_ptr())
    qd, kd, vd = rows_d(q), rows_d(k), rows_d(v)
    out, o2 = [torch.full((9, heads * d), 7.0, device="cuda") for _ in range(2)]
    a.cache.append_d(0, sa, 9, 0, rope_d(64), kd.data_ptr(), kv * d, vd.data_ptr(), kv * d, heads, qd.data_ptr(), heads * d, out.data_ptr(), heads * d, stream=stream())
    a.cache.attend_d(0, sa, 9, 0, heads, out.data_ptr(), heads * d, o2.data_ptr(), heads * d, 0, 0.0, stream())
    s = Seqs(lay.lens, lay.table, lay.starts)
    want = b.cache.append(0, s, k[2:7], v[2:7], Rope(64), q=q[2:7])
    assert np.array_equal(out[2:7].cpu().numpy(), want) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert np.array_equal(o2[2:7].cpu().numpy(), b.cache.attend(0, s, want))
    for t in (out, o2):
        assert (t[:2] == 7).all() and (t[7:] == 7).all()
    host_out = b.cache.attend(0, Seqs(lay.lens, lay.table, lay.starts + 2), np.concatenate((q[:2], want, q[7:])))
    assert np.array_equal(host_out[2:7], o2[2:7].cpu().numpy()) and not host_out[:2].any()
    k0, v0 = a.k.clone(), a.v.clone()
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    sn = seqs_d(2, a.lens.data_ptr(), a.table.data_ptr(), lay.table.shape[1], none.data_ptr())
    out.fill_(7.0)
    a.cache.append_d(0, sn, 9, 0, rope_d(64), kd.data_ptr(), kv * d, vd.data_ptr(), kv * d, heads, qd.data_ptr(), heads * d, out.data_ptr(), heads * d, stream=stream())
    a.cache.attend_d(0, sn, 9, 0, heads, qd.data_ptr(), heads * d, out.data_ptr(), heads * d, 0, 0.0, stream())
    torch.cuda.synchronize()
    assert torch.equal(a.k, k0) and torch.equal(a.v, v0) and (out == 7).all()


def test_more_tokens_than_the_table_holds(ctx):
    """A held length past the table's end: new tokens are not stored, their queries turn by their own positions, and see what
    the table holds."""
    lay = Layout([64], [0], 32, wide=0)
    pg = Pages(ctx, lay, 1, 64, "f16")
    pg.lens.fill_(1000)
    starts = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    s = seqs_d(1, pg.lens.data_ptr(), pg.table.data_ptr(), 2, starts.data_ptr())
    q = np.random.default_rng(0).standard_normal((2, 64)).astype(np.float32)
    qd, out, after = rows_d(q), torch.zeros(2, 64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    pg.cache.append_d(0, s, 2, 0, rope_d(64), qd.data_ptr(), 64, qd.data_ptr(), 64, 1, qd.data_ptr(), 64, out.data_ptr(), 64, stream=stream())
    pg.cache.keep_d(s, kept.data_ptr(), 2, after.data_ptr(), stream())
    torch.cuda.synchronize()
    want = rotate(q.astype(np.float64)[:, None], [1000, 1001], 64, 1e4, True)[:, 0]
    assert np.abs(out.cpu().numpy() - want).max() <= 2 * np.abs(q).max() * (6.3 * 2.0 ** -26 + 5 * 2.0 ** -24)
    assert np.array_equal(host(pg.k, "f16"), pg.k0) and np.array_equal(host(pg.v, "f16"), pg.v0) and after.item() == 1002
    pg.cache.attend_d(0, s, 2, 0, 1, qd.data_ptr(), 64, out.data_ptr(), 64, 0, 0.0, stream())
    k, v = pg.rows(0, 64)
    for i in range(2):  # (the last held token as the one new token of its row: the row sees all 64)
        want, bound = attend(q[i:i + 1].astype(np.float64), k, v, 63, 1)
        assert np.all(np.abs(out[i:i + 1].cpu().numpy() - want) <= bound + EPS["f32"] * (np.abs(want) + bound))
    # a tree whose tokens have no slots: chains that end well see the held tokens, others nothing (small and large tiles)
    for heads in (1, 70):
        par = torch.tensor([-1, 5], dtype=torch.int32, device="cuda")
        q2 = rows_d(np.random.default_rng(1).standard_normal((2, heads * 64)).astype(np.float32))
        o2 = torch.full((2, heads * 64), 7.0, device="cuda")
        pg.cache.attend_d(0, s, 2, 0, heads, q2.data_ptr(), heads * 64, o2.data_ptr(), heads * 64, par.data_ptr(), 0.0, stream())
        got = o2.cpu().numpy()
        want, bound = attend(q2[:1].cpu().numpy().astype(np.float64), k, v, 63, heads)
        assert np.all(np.abs(got[:1] - want) <= bound + EPS["f32"] * (np.abs(want) + bound)) and not got[1].any()


def test_sequences_that_overlap_stay_in_bounds(ctx):
    """Starts that fall and rise name the same rows for many sequences, more tiles than the call was planned for: rows are left
    out or written more than once, and nothing behind them is touched.  With the long sequence split tiles are left out."""
    b, n = 64, 40
    for long in (20000, 700):
        lay = Layout([700] * (b - 2) + [long, 700], [0] * b, 32, wide=2)
        pg = Pages(ctx, lay, 1, 64, "f16")
        starts = torch.tensor([0, n] * (b // 2) + [0], dtype=torch.int32, device="cuda")
        s = seqs_d(b, pg.lens.data_ptr(), pg.table.data_ptr(), lay.table.shape[1], starts.data_ptr())
        for heads in (1, 8):
            q = torch.randn(n, heads * 64, device="cuda")
            buf = torch.full((n + 8, heads * 64), 7.0, device="cuda")
            pg.cache.attend_d(0, s, n, 0, heads, q.data_ptr(), heads * 64, buf[4:].data_ptr(), heads * 64, 0, 0.0, stream())
            torch.cuda.synchronize()
            assert (buf[:4] == 7).all() and (buf[n + 4:] == 7).all()
    # a call of an ordinary sequence after it is as ever
    s1 = seqs_d(1, pg.lens.data_ptr(), pg.table.data_ptr(), lay.table.shape[1])
    q, out = torch.randn(1, 64, device="cuda"), torch.zeros(1, 64, device="cuda")
    pg.cache.attend_d(0, s1, 1, 0, 1, q.data_ptr(), 64, out.data_ptr(), 64, 0, 0.0, stream())
    k, v = pg.rows(0, 701)
    want, bound = attend(q.cpu().numpy().astype(np.float64), k, v, 700, 1)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound + EPS["f32"] * (np.abs(want) + bound))


# ------------------------------------------------------------------ keep
@pytest.mark.parametrize("ct", ["f16", "bf16"])
@pytest.mark.parametrize("d, page, kv, layers", [(128, 32, 2, 3), (80, 64, 3, 1), (256, 32, 1, 2), (16, 32, 2, 2)])
def test_keep(ctx, ct, d, page, kv, layers):
    lens, counts = [30, 0, 31, 64, 5, 7], [40, 9, 3, 30, 33, 0]
    kept = [[1, 2, 3, 9, 11, 12, 13, 14, 15, 39], [0, 1, 2], [], [29], list(range(1, 33)), []]
    lay = Layout(lens, counts, page, seed=d)
    pg = Pages(ctx, lay, kv, d, ct, layers=layers)
    want_k, want_v = pg.k0.copy(), pg.v0.copy()
    for i, row in enumerate(kept):
        p, s = lay.slots(i)
        for j, x in enumerate(row):
            to, fr = lens[i] + j, lens[i] + x
            want_k[:, p[to], :, s[to]] = pg.k0[:, p[fr], :, s[fr]]
            want_v[:, p[to], :, :, s[to]] = pg.v0[:, p[fr], :, :, s[fr]]
    after = pg.cache.keep(Seqs(lay.lens, lay.table), kept)
    assert after.tolist() == [a + len(r) for a, r in zip(lens, kept)]
    assert np.array_equal(host(pg.k, ct), want_k) and np.array_equal(host(pg.v, ct), want_v)


def test_keep_on_the_device_ends_lists_that_do_not_ascend(ctx):
    lay = Layout([3] * 5, [20] * 5, 32)
    pg = Pages(ctx, lay, 1, 64, "f16")
    lists = [[2, 5, 5, 7], [4, 3, 9, 10], [-7, 1, 2, 3], [2 ** 31 - 1, 0, 1, 2], [1, 2, 2 ** 31 - 1, -1]]
    kd, after = dev(np.array(lists, np.int32)), torch.zeros(5, dtype=torch.int32, device="cuda")
    pg.cache.keep_d(pg.seqs, kd.data_ptr(), 4, after.data_ptr(), stream())
    torch.cuda.synchronize()
    assert after.tolist() == [5, 4, 3, 4, 6]
    got = host(pg.k, "f16")
    p = [lay.slots(i) for i in range(5)]
    for i, moves in enumerate([[(0, 2), (1, 5)], [(0, 4)], [], [], [(0, 1), (1, 2)]]):
        for to, fr in moves:
            assert np.array_equal(got[0][p[i][0][3 + to], :, p[i][1][3 + to]], pg.k0[0][p[i][0][3 + fr], :, p[i][1][3 + fr]])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("xt, ct", [("f32", "f16"), ("bf16", "bf16")])
def test_drafting_with_a_tree(ctx, xt, ct):
    """A prompt, a drafted tree, its accepted branch kept, and the next token: each token's row is that of plain attention
    over the tokens before it, with the keys that the cache holds."""
    kv, heads, d, page, layers = 2, 6, 64, 32, 2
    rng = np.random.default_rng(8)
    b, prompt, nodes = 3, [45, 1, 130], 12
    trees = [tree(rng, nodes, deep=5) for _ in range(b)]
    lay = Layout([0] * b, [m + nodes + 4 for m in prompt], page)
    pg = Pages(ctx, lay, kv, d, ct, layers=layers, fill=np.nan)
    lens = np.zeros(b, np.int32)
    tokens = [[] for _ in range(b)]  # the accepted tokens' (k, v) rows of each layer
    rope = Rope(d, 1e4, neox=False)

    def step(counts, parents=None, depth=None):
        nonlocal lens
        starts = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        n = starts[-1]
        seqs = Seqs(lens, lay.table, starts)
        pos = None if depth is None else np.concatenate([lens[i] + np.array(depth[i]) for i in range(b)]).astype(np.int32)
        new = [[[None] * layers for _ in range(c)] for c in counts]
        for layer in range(layers):
            q, k, v = [to_type(rng.standard_normal((n, h * d)), xt) for h in (heads, kv, kv)]
            qr = pg.cache.append(layer, seqs, k, v, rope, q=q, positions=pos, type=TYPES[xt])
            par = None if parents is None else np.concatenate(parents).astype(np.int32)
            out = pg.cache.attend(layer, seqs, qr, parents=par, type=TYPES[xt])
            for i in range(b):
                a, m = starts[i], counts[i]
                at = lens[i] + np.arange(m) if depth is None else lens[i] + np.array(depth[i])
                kk = rotate(value(k[a:a + m], xt).reshape(m, kv, d), at, d, 1e4, False)
                vv = value(v[a:a + m], xt).reshape(m, kv, d)
                for j in range(m):
                    new[i][j][layer] = (value(to_type(kk[j], ct), ct), value(to_type(vv[j], ct), ct))
                allk = np.array([t[layer][0] for t in tokens[i]] + [t[layer][0] for t in new[i]])
                allv = np.array([t[layer][1] for t in tokens[i]] + [t[layer][1] for t in new[i]])
                qq = rotate(value(q[a:a + m], xt).reshape(m, heads, d), at, d, 1e4, False).reshape(m, -1)
                want, bound = attend(qq, allk, allv, int(lens[i]), heads, None if parents is None else parents[i], weights=one_plane(xt, n, b, heads, kv, d))
                # the keys and queries that the cache's call rounds (and, once in a thousand, to the other side of a
                # border than these) leave the scores within 2 half steps of both: weights and rows within that
                qmax = np.abs(qq.reshape(m, heads, d)).sum(2).max()
                slack = 2 * (EPS[ct] + EPS[xt]) * qmax * np.abs(allk).max() / np.sqrt(d) * np.abs(allv).max()
                err = np.abs(value(out[a:a + m], xt) - want)
                assert np.all(err <= bound + slack + EPS[xt] * np.abs(want)), (layer, i, err.max())
        return new

    first = step(prompt)
    for i in range(b):
        tokens[i] += first[i]
    lens = lens + np.array(prompt, np.int32)
    drafted = step([nodes] * b, [t[0] for t in trees], [t[1] for t in trees])
    kept = []
    for i in range(b):
        node, branch = int(rng.integers(nodes // 2, nodes)), []
        while node >= 0:
            branch.append(node)
            node = trees[i][0][node]
        kept.append(branch[::-1])
        tokens[i] += [drafted[i][x] for x in kept[i]]
    lens = pg.cache.keep(Seqs(lens, lay.table), kept)
    assert lens.tolist() == [len(t) for t in tokens]
    step([1] * b)


def test_a_captured_step_replays(ctx):
    """append, attend and keep in one graph, with lengths, tables and rows changed between replays."""
    lay = Layout([100, 20], [8, 8], 32)
    kv, heads, d, n = 2, 4, 128, 16
    pg, ref = Pages(ctx, lay, kv, d, "f16", layers=2), Pages(ctx, lay, kv, d, "f16", layers=2)
    rng = np.random.default_rng(0)
    par = dev(np.array([-1, 0, 0, 1, 2, 2, 4, 5] * 2, np.int32))
    kept = dev(np.array([[0, 2, 4, 6], [1, -1, -1, -1]], np.int32))
    x = torch.zeros(n, (heads + 2 * kv) * d, device="cuda")
    ld, rope = x.stride(0), rope_d(d, 1e6)

    def call(p, out, q, after, st):
        for layer in range(2):
            p.cache.append_d(layer, p.seqs, n, 0, rope, x.data_ptr() + 4 * heads * d, ld, x.data_ptr() + 4 * (heads + kv) * d, ld, heads, x.data_ptr(), ld, q.data_ptr(),
                             heads * d, stream=st)
            p.cache.attend_d(layer, p.seqs, n, 0, heads, q.data_ptr(), heads * d, out.data_ptr(), heads * d, par.data_ptr(), 0.0, st)
        p.cache.keep_d(p.seqs, kept.data_ptr(), 4, after.data_ptr(), st)

    bufs = [[torch.zeros(n, heads * d, device="cuda"), torch.zeros(n, heads * d, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")] for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call(pg, *bufs[0], side.cuda_stream)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call(pg, *bufs[0], torch.cuda.current_stream().cuda_stream)
    pg.k.copy_(ref.k), pg.v.copy_(ref.v)
    for lens in ([100, 20], [7, 27], [0, 0], [101, 24]):
        for p in (pg, ref):
            p.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
            call(ref, *bufs[1], side.cuda_stream)
        side.synchronize()
        assert torch.equal(pg.k, ref.k) and torch.equal(pg.v, ref.v)
        assert all(torch.equal(a, b) for a, b in zip(*bufs))
        assert torch.isfinite(bufs[0][0]).all() and (x.sum() * 0 == 0).item()  # the program's own work between the replays


def test_two_graphs_share_the_workspace(ctx):
    """Calls whose parts are joined by the last workgroup, and by a kernel, captured apart and replayed in turn."""
    lay = Layout([900, 2000, 700], [1, 1, 1], 32)
    pg = Pages(ctx, lay, 2, 64, "f16")
    big = Layout([3000], [40], 32, seed=3)
    pb = Pages(ctx, big, 2, 64, "f16", seed=3)
    q = [torch.randn(n, 256, device="cuda") for n in (3, 40)]
    out = [torch.zeros_like(x) for x in q]
    side = torch.cuda.Stream()

    def call(i, st):
        p, n = ((pg, 3), (pb, 40))[i]
        p.cache.attend_d(0, p.seqs, n, 0, 4, q[i].data_ptr(), 256, out[i].data_ptr(), 256, 0, 0.0, st)

    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(side):
        for i in (1, 0):
            call(i, side.cuda_stream)
        side.synchronize()
        for i in (0, 1):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                call(i, torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        for x in q:
            x.normal_()
        torch.cuda.synchronize()
        for i in (0, 1):
            out[i].fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for i in ((0, 1), (1, 0), (0, 0, 1), (1, 1, 0))[turn]:
                graphs[i].replay()
        side.synchronize()
        got = [x.clone() for x in out]
        with torch.cuda.stream(side):
            for i in (0, 1):
                call(i, side.cuda_stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, out)) and torch.isfinite(got[0]).all()


def test_calls_from_two_threads(ctx):
    """Host calls on one cache from two threads: each as it is alone."""
    import threading

    lay = Layout([700, 90], [2, 2], 32)
    pg = Pages(ctx, lay, 2, 64, "f16")
    q = [np.random.default_rng(i).standard_normal((4, 256)).astype(np.float32) for i in range(2)]
    s = [Seqs(lay.lens, lay.table, lay.starts) for _ in range(2)]
    want = [pg.cache.attend(0, s[i], q[i]) for i in range(2)]
    ok = [True, True]

    def work(i):
        for _ in range(20):
            ok[i] = ok[i] and np.array_equal(pg.cache.attend(0, s[i], q[i]), want[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(ok)


def test_growing_under_capture_is_refused():
    own = rt.Context(0)
    lay = Layout([10], [1], 32)
    pg = Pages(own, lay, 1, 64, "f16")
    q, out = torch.zeros(1, 64, device="cuda"), torch.zeros(1, 64, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            with pytest.raises(rt.RtqError, match="capture"):
                pg.cache.attend_d(0, pg.seqs, 1, 0, 1, q.data_ptr(), 64, out.data_ptr(), 64, 0, 0.0, torch.cuda.current_stream().cuda_stream)
            out.zero_()
    own.close()


def test_an_owned_cache_starts_with_zeros_and_goes_with_its_context():
    own = rt.Context(0)
    cache = KvCache(2, 3, 32, 2, 64, ctx=own)
    s = Seqs([10], [[0]], [0, 1])
    assert (cache.attend(1, s, np.ones((1, 128), np.float32)) == 0).all()
    cache.append(1, s, np.ones((1, 128), np.float32), np.full((1, 128), 11, np.float32), Rope(0))
    got = cache.attend(1, s, np.zeros((1, 128), np.float32))
    assert np.allclose(got, 1.0, atol=2.0 ** -20)
    k0, _ = cache.pages(0)
    k1, _ = cache.pages(1)
    assert k1 - k0 == 3 * 32 * 2 * 64 * 2
    own.close()
    with pytest.raises(RuntimeError, match="destroyed"):
        cache.pages(0)
