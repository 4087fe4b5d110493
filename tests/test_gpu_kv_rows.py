"""Rows of the cache's attention where its plan is at its ends: how exact 16-bit rows are in tiles of either size, tiles of so many
parts that the join's tables are full."""
import numpy as np
import pytest

from kv_cases import EPS, TINY, TYPES, Layout, attend, to_type, tree, value, visible
from rust_trainer_amd.kvcache import rope_d, seqs_d
from test_gpu_kvcache import NP, Pages, dev, host, rows_d, stream

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def planes(xt):
    """What two planes of a weight leave of it: half a step of the half step that the first leaves (f32 rows take as many planes
    as their bound of 2^-22 asks for)."""
    return 0.0 if xt == "f32" else EPS[xt] ** 2


def run(pg, q, xt, heads, parents=None, scale=0.0):
    """The call's rows, over 7s."""
    n, d = q.shape[0], pg.d
    qd, out = rows_d(q), rows_d(np.full((n, heads * d), 7, NP[xt]))
    pd = None if parents is None else dev(np.asarray(parents, np.int32))
    pg.cache.attend_d(0, pg.seqs, n, TYPES[xt], heads, qd.data_ptr(), heads * d, out.data_ptr(), heads * d, 0 if pd is None else pd.data_ptr(), scale, stream())
    torch.cuda.synchronize()
    return host(out, xt)


def check(pg, got, q, xt, heads, parents=None, scale=0.0, only=None):
    lay = pg.lay
    for i in range(lay.b) if only is None else only:
        a, z = lay.starts[i], lay.starts[i + 1]
        if a == z:
            continue
        k, v = pg.rows(i)
        want, bound = attend(value(q[a:z], xt), k, v, int(lay.lens[i]), heads, None if parents is None else parents[a:z], scale, planes(xt))
        err = np.abs(value(got[a:z], xt) - want)
        lim = bound + EPS[xt] * (np.abs(want) + bound) + TINY[xt]
        assert np.all(err <= lim), (i, (err / lim).max(), np.argwhere((err > lim).any(1)).ravel()[:8])


EXACT = [  # lens, counts, heads, kv, d, tree
    ([300], [40], 4, 1, 128, False),     # tiles of 128 rows: whole,
    ([3000], [40], 4, 1, 64, False),     # split,
    ([1500], [40], 4, 1, 256, True),
    ([900, 40], [60, 33], 8, 2, 80, True),
    ([200, 100], [6, 5], 4, 1, 128, False),  # more than 16 rows of short sequences: tiles of 16
    ([2000], [4], 4, 1, 128, False),
]


@pytest.mark.parametrize("xt, ct", [("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("case", range(len(EXACT)))
def test_weights_of_16_bit_rows_keep_two_planes(ctx, case, xt, ct):
    """Small scores, so that weights are what is rounded: a row is within a weight's two planes in a tile of either size."""
    lens, counts, heads, kv, d, is_tree = EXACT[case]
    lay = Layout(lens, counts, 32, seed=case)
    rng = np.random.default_rng(case)
    pg = Pages(ctx, lay, kv, d, ct, seed=case)
    q = to_type(0.05 * rng.standard_normal((lay.n, heads * d)), xt)
    parents = np.array([p for m in counts for p in tree(rng, m)[0]], np.int32) if is_tree else None
    check(pg, run(pg, q, xt, heads, parents), q, xt, heads, parents)


JOINED = [  # sequences, the one with new tokens: held, new, then heads, kv, d, tree: parts x rows past 1024 in one small tile
    (12, 10898, 2, 12, 2, 128, False),  # 86 parts of 12 rows
    (16, 9358, 2, 28, 4, 128, False),   # 74 of 14
    (16, 10069, 13, 1, 1, 128, False),  # 79 of 13
    (16, 10069, 13, 1, 1, 64, True),
    (16, 8705, 15, 4, 4, 64, True),     # 69 of 15
    (16, 14500, 9, 1, 1, 128, True),    # 114 of 9
]


@pytest.mark.parametrize("xt, ct", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("case", range(len(JOINED)))
def test_tiles_of_many_parts_in_a_batch_of_idle_sequences(ctx, case, xt, ct):
    """One sequence with some rows, joined by its last workgroup (the call's mean is a row a sequence or less)."""
    b, held, new, heads, kv, d, is_tree = JOINED[case]
    lay = Layout([40] * 3 + [held] + [7] * (b - 4), [0] * 3 + [new] + [0] * (b - 4), 64, seed=case)
    rng = np.random.default_rng(case)
    pg = Pages(ctx, lay, kv, d, ct, seed=case)
    q = to_type(2.0 * rng.standard_normal((new, heads * d)), xt)
    parents = np.array(tree(rng, new)[0], np.int32) if is_tree else None
    check(pg, run(pg, q, xt, heads, parents), q, xt, heads, parents)


def test_fifteen_rows_beside_a_token(ctx):
    lay = Layout([8705, 100] + [3] * 14, [15, 1] + [0] * 14, 64)
    rng = np.random.default_rng(1)
    pg = Pages(ctx, lay, 4, 64, "f16")
    q = to_type(rng.standard_normal((16, 4 * 64)), "f16")
    parents = np.array(tree(rng, 15)[0] + [-1], np.int32)
    check(pg, run(pg, q, "f16", 4, parents), q, "f16", 4, parents)


DEAD = [  # held, counts, heads: whole tiles, joined by the last workgroup (small, large tiles) and by a kernel (small, large)
    (20, [6, 2], 4), (4000, [6, 2], 1), (800, [9, 8], 2), (4000, [6, 2], 4), (4000, [6, 2], 16)]


@pytest.mark.parametrize("xt, ct", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("held, counts, heads", DEAD)
def test_rows_that_see_nothing_are_zero_beside_infinite_scores(ctx, held, counts, heads, xt, ct):
    """A held key of +inf is no key of an unused node's row, nor of what hangs from it: those are 0, the others what
    the formula makes of an infinite score, and the next sequence's are as ever."""
    lay = Layout([held, 0], counts, 32)
    rng = np.random.default_rng(4)
    pg = Pages(ctx, lay, 1, 64, ct)
    p, s = lay.slots(0)
    pg.k0[0][p[10], 0, s[10]] = to_type(np.array([np.inf]), ct)[0]
    pg.k.copy_(dev(pg.k0))
    parents = np.array([-1, -2, 1, 0, 7, 3, 4, -1, 8][:counts[0]] + [-1, 1, 0, 2, 3, -1, 9, 5][:counts[1]], np.int32)
    q = to_type(np.abs(rng.standard_normal((lay.n, heads * 64))), xt)
    got = value(run(pg, q, xt, heads, parents), xt)
    _, alive = visible(counts[0], parents[:counts[0]])
    assert not got[:counts[0]][~alive].any() and np.isnan(got[:counts[0]][alive]).all()
    _, alive = visible(counts[1], parents[counts[0]:])
    assert not got[counts[0]:][~alive].any()
    check(pg, to_type(got, xt), q, xt, heads, parents, only=[1])


@pytest.mark.parametrize("first", [0, 3, 40])
def test_append_takes_its_sequences_rows_alone(ctx, first):
    """A call of up to 300 rows, as a captured step makes it, whose sequences have 73 of them: the cache and the queries are those
    of a call of 73, and the rows before and behind, NaN here, are left."""
    lay = Layout([5, 31, 0], [40, 0, 33], 32, seed=2)
    kv, heads, d, n = 3, 6, 80, 300
    rng = np.random.default_rng(first)
    a, b = Pages(ctx, lay, kv, d, "f16"), Pages(ctx, lay, kv, d, "f16")
    rows = [rng.standard_normal((lay.n, h * d)).astype(np.float32) for h in (heads, kv, kv)]
    wide = [np.full((n, r.shape[1]), np.nan, np.float32) for r in rows]
    for w, r in zip(wide, rows):
        w[first:first + lay.n] = r
    starts = dev(lay.starts + first)
    seqs = seqs_d(lay.b, a.lens.data_ptr(), a.table.data_ptr(), lay.table.shape[1], starts.data_ptr())
    outs = []
    for pg, s, (q, k, v) in ((a, seqs, wide), (b, b.seqs, rows)):
        qd, kd, vd = dev(q), dev(k), dev(v)
        outs.append(torch.full((len(q), heads * d), 7.0, device="cuda"))
        pg.cache.append_d(0, s, len(q), 0, rope_d(32), kd.data_ptr(), kv * d, vd.data_ptr(), kv * d, heads, qd.data_ptr(), heads * d, outs[-1].data_ptr(),
                          heads * d, stream=stream())
        torch.cuda.synchronize()
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(outs[0][first:first + lay.n], outs[1])
    assert (outs[0][:first] == 7).all() and (outs[0][first + lay.n:] == 7).all()
