"""Rows of the cache's attention at the ends of its tables: how exact 16-bit rows are in tiles of either size."""
import numpy as np
import pytest

from kv_cases import EPS, TINY, TYPES, Layout, attend, to_type, tree, value
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
