"""Paged caches for tests: sequences in shuffled pages, and the cache operators' definitions in 64 bits."""
import numpy as np

TYPES = {"f32": 0, "f16": 1, "bf16": 30}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the subnormals


def to_type(x, t):
    """An array's values in type t (bfloat16: its bits)."""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x
    if t == "f16":
        return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def value(x, t):
    """The values of an array in type t, in 64 bits."""
    return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if t == "bf16" else x.astype(np.float64)


class Layout:
    """Sequences of `lens` held and `counts` new tokens, their pages shuffled over a pool with spare pages."""

    def __init__(self, lens, counts, page, seed=0, spare=3, wide=1):
        rng = np.random.default_rng(seed)
        self.lens, self.counts, self.page = np.array(lens, np.int32), np.array(counts, np.int32), page
        self.starts = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        self.n, self.b = int(self.starts[-1]), len(lens)
        pages = -(-(self.lens + self.counts) // page)
        self.n_pages = int(pages.sum()) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((self.b, int(pages.max()) + wide), -1, np.int32)  # behind a sequence's end: no page
        at = 0
        for i, p in enumerate(pages):
            self.table[i, :p] = order[at:at + p]
            at += p

    def slots(self, i, count=None):
        """(page, slot in the page) of the first `count` slots of sequence i (all of them)."""
        s = np.arange(self.lens[i] + self.counts[i] if count is None else count)
        return self.table[i, s // self.page], s % self.page


def rotate(x, pos, dim, base, neox, scale=1.0, factors=None):
    """x [n x heads x d] in 64 bits, rotated."""
    i = np.arange(dim // 2)
    freq = float(np.float32(base)) ** (-2.0 * i / max(dim, 1)) * float(np.float32(scale))
    if factors is not None:
        f = np.ones(dim // 2)
        f[:len(factors)] = np.where(np.asarray(factors) != 0, factors, 1.0)
        freq = freq / f
    a = np.asarray(pos, np.float64)[:, None] * freq
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    y = x.copy()
    ia, ib = (i, i + dim // 2) if neox else (2 * i, 2 * i + 1)
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ib] * c + x[..., ia] * s
    return y


def norm(x, w, eps, offset):
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * (w.astype(np.float64) + float(np.float32(offset)))


def visible(m, parents=None):
    """[m x m] which new tokens each new token sees, and which rows see anything at all (the cache included)."""
    if parents is None:
        return np.tril(np.ones((m, m), bool)), np.ones(m, bool)
    seen, alive = np.zeros((m, m), bool), np.ones(m, bool)
    for i in range(m):
        node = i
        while node >= 0:
            seen[i, node] = True
            p = int(parents[node])
            if p < -1 or p >= node:
                alive[i], seen[i] = False, False
                break
            node = p
    return seen, alive


def one_plane(xt, n, b, heads, kv, d):
    """The half step by which the weights of a call are rounded: large tiles (some of the calls of more than 16 rows a sequence
    and KV head) of 16-bit rows hold each weight in one number of that type; the others'
    planes are counted with the scores' below."""
    large = n * (heads // kv) > 16 * b
    return EPS[xt] if large and xt != "f32" else 0.0


def attend(q, k, v, held, heads, parents=None, scale=0.0, weights=0.0):
    """(out, bound): attention of one sequence in 64 bits, and what rounding may make of it in the kernels' 32.
    q [m x heads d], k and v [slots x kv x d]; weights: what each weight may be off by (``one_plane``): the weights' sum is
    of the unrounded ones, so a row's error is at most that share of its weighted values' sizes."""
    m, kv, d = q.shape[0], k.shape[1], k.shape[2]
    scale = float(np.float32(scale)) or 1.0 / np.sqrt(d)
    seen, alive = visible(m, parents)
    vis = np.concatenate((np.ones((m, held), bool) & alive[:, None], seen), 1)
    out, bound = np.zeros((m, heads, d)), np.zeros((m, heads, d))
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        qh = q.reshape(m, heads, d)[:, h]
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(vis, qh @ np.where(np.isfinite(kh), kh, 0.0).T * scale, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0.0)) * vis
        l = p.sum(1, keepdims=True)
        p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
        fin = np.where(np.isfinite(vh), vh, 0.0)
        out[:, h] = p @ fin
        # scores: planes of q within 2^-22 of the row's largest element, d products of which each sum rounds by 2^-24, the
        # product with the scale and the difference from the maximum (2^-23 of both sizes); weights: v_exp_f32 and their
        # planes (2^-22); sums over the slots in 32 bits: a step of 32 per 128 slots, planes, waves and parts joined
        kabs = np.abs(np.where(np.isfinite(kh), kh, 0.0))
        es = (np.abs(qh) @ kabs.T * d * 2.0 ** -24 + np.abs(qh).max(1, keepdims=True) * kabs.sum(1) * 2.0 ** -22) * scale
        size = np.where(vis, np.abs(np.where(vis, s, 0.0)), 0.0).max(1, keepdims=True)
        e = (es * vis).max(1, keepdims=True) + 2.0 ** -22 * size
        bound[:, h] = (2 * e + 2.0 ** -21 + (k.shape[0] / 32 + 64) * 2.0 ** -24 + weights) * (p @ np.abs(fin))
    return out.reshape(m, -1), bound.reshape(m, -1)


def tree(rng, m, deep=8, back=12):
    """Parents of a random tree of m nodes, no branch longer than deep, and the nodes' depths."""
    parents, depth = [], []
    for i in range(m):
        p = int(rng.integers(max(-1, i - back), i))
        while p >= 0 and depth[p] >= deep - 1:
            p = parents[p]
        parents.append(p)
        depth.append(0 if p < 0 else depth[p] + 1)
    return parents, depth
