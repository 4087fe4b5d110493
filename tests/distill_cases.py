"""Plain 64-bit forms of the operators on rows of vocabulary logits, and inputs for their tests."""
import numpy as np

NEG = -np.inf
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}  # half a subnormal step (f16); flushed below (others)
# Relative error of a sum of f32 exponentials: 2^-22 for an exponential (its instruction and two
# roundings), 2^-22 for a vector's eight f32 additions, the rounding of its argument, |z - max| 2^-24 / T,
# and of the scale 1 / T, |z - max| 2^-25 / T, averaged over the softmax (|z - max| / T at most log of the
# vocabulary, 12.6: weights below e^-12.6 count less).
SUM = 2.0 ** -21 + 12.6 * 1.5 * 2.0 ** -24


def lse(x, axis=-1):
    with np.errstate(all="ignore"):
        m = np.max(x, axis=axis, keepdims=True)
        m0 = np.where(np.isfinite(m), m, 0.0)
        r = np.log(np.sum(np.exp(x - m0), axis=axis, keepdims=True)) + m0
        r = np.where(m == np.inf, np.inf, r)
    return np.squeeze(r, axis)


def top(z, k, temp):
    """(vals, ids, rest) of f64 rows; NaN above every number, equal values by the lower id."""
    z = np.asarray(z, np.float64)
    order = np.argsort(np.where(np.isnan(z), NEG, -z), axis=1, kind="stable")
    ids = order[:, :k]
    left = np.take_along_axis(z, order[:, k:], 1)
    rest = lse(left / temp) if left.shape[1] else np.full(z.shape[0], NEG)
    return np.take_along_axis(z, ids, 1), ids, rest


def distill(z, ids, vals, rest, temp, tok=None, w=None, hard=0.0):
    """One row at a time: (kl, logp, gradient, scale): scale bounds, per element, the magnitudes that the
    gradient is a difference of."""
    z = np.asarray(z, np.float64)
    n, V = z.shape
    with np.errstate(all="ignore"):  # from the maximum: beside one of -1e20 the logarithms would be lost
        m = z.max(1, keepdims=True)
        z = z - np.where(np.isfinite(m), m, 0.0)
    kl, logp, g, sc = np.zeros(n), np.full(n, np.nan), np.zeros((n, V)), np.zeros((n, V))
    with np.errstate(all="ignore"):
        for i in range(n):
            held = [s for s in range(len(ids[i])) if 0 <= ids[i][s] < V]
            t = np.array([float(vals[i][s]) / temp for s in held] + [NEG if rest is None else float(rest[i])])
            listed = np.zeros(V, bool)
            listed[[ids[i][s] for s in held]] = True
            lq, q1 = z[i] / temp - lse(z[i] / temp), np.exp(z[i] - lse(z[i]))
            q = np.exp(lq)
            wi = 0.0 if w is None else float(w[i])
            taught = not np.all(t == NEG)
            if taught:
                p = np.exp(t - lse(t))
                lr = lse(lq[~listed]) if (~listed).any() else NEG
                for j in {ids[i][s] for s in held}:  # slots of one token are one bucket
                    pj = sum(p[b] for b, s in enumerate(held) if ids[i][s] == j)
                    if pj > 0 or np.isnan(pj):
                        kl[i] += pj * (np.log(pj) - lq[j])
                if p[-1] > 0 or np.isnan(p[-1]):
                    kl[i] += p[-1] * (np.log(p[-1]) - lr)
                d = q.copy()
                s_ = q.copy()
                if p[-1] > 0:
                    share = np.where(listed, 0.0, p[-1] * np.exp(np.where(listed, NEG, lq - lr)))
                    if lr == NEG:
                        share[:] = 0.0
                    d -= share
                    s_ += share
                for b, s in enumerate(held):
                    d[ids[i][s]] -= p[b]
                    s_[ids[i][s]] += p[b]
                g[i] += wi * (1 - hard) * temp * d
                sc[i] += abs(wi) * (1 - hard) * temp * s_
            if tok is not None and 0 <= tok[i] < V:
                logp[i] = z[i, tok[i]] - lse(z[i])
                one = np.arange(V) == tok[i]
                g[i] += wi * hard * (q1 - one)
                sc[i] += abs(wi) * hard * (q1 + one)
            if wi == 0.0:
                g[i], sc[i] = 0.0, 0.0
    return kl, logp, g, sc


def verify(z, q, drafted, lens, u, temp):
    b, d = drafted.shape
    V = z.shape[1]
    z = np.asarray(z, np.float64).reshape(b, d + 1, V)
    q = None if q is None else np.asarray(q, np.float64).reshape(b, d, V)
    acc, out = np.zeros(b, np.int32), np.full((b, d + 1), -1, np.int32)
    soft = lambda x: np.exp(x / temp - lse(x / temp)) if np.isfinite(x.max()) else np.full(V, np.nan)  # noqa: E731

    def best(row):  # of the logits, -1 without a distribution
        v, j, _ = top(row[None], 1, 1.0)
        return j[0, 0] if v[0, 0] > NEG else -1

    with np.errstate(all="ignore"):
        for i in range(b):
            n = d if lens is None else min(max(int(lens[i]), 0), d)
            a, w = 0, None
            while a < n:
                x = int(drafted[i, a])
                ok = 0 <= x < V
                if temp == 0:
                    ok = ok and x == best(z[i, a])
                else:
                    p = soft(z[i, a])
                    qa = np.arange(V) == x if q is None else soft(q[i, a])
                    ok = bool(ok and float(u[i, a]) * (qa[x] if q is not None else 1.0) < p[x])
                    if not ok:
                        w = np.maximum(p - qa, 0.0)
                        if not w.sum() > 0:
                            w = p
                if not ok:
                    break
                out[i, a] = x
                a += 1
            acc[i] = a
            if temp == 0:
                out[i, a] = best(z[i, a])
                continue
            if w is None:
                w = soft(z[i, a])
            c = np.cumsum(w)
            if c[-1] > 0:
                hit = np.nonzero(c > float(u[i, d]) * c[-1])[0]
                out[i, a] = hit[0] if hit.size else np.nonzero(w > 0)[0][-1]
    return acc, out


def logits(rng, n, V, near=None):
    """Rows of a decoder's head: a spread of a few units and a few tokens far above."""
    z = rng.normal(0, 1.5, (n, V)) if near is None else near + rng.normal(0, 0.7, (n, V))
    for i in range(n):
        z[i, rng.integers(0, V, 4)] += rng.uniform(2, 9, 4)
    return z


def rounded(z, ty):
    """z in the type's values: (array to hand over, the same as f64).  bf16 arrays are their uint16 bits."""
    if ty == "f32":
        a = z.astype(np.float32)
        return a, a.astype(np.float64)
    if ty == "f16":
        a = np.clip(z, -65504, 65504).astype(np.float16) if np.isfinite(z).all() else z.astype(np.float16)
        return a, a.astype(np.float64)
    bits = z.astype(np.float32).view(np.uint32)
    nan = np.isnan(z)
    r = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(nan, np.uint16(0x7FC0), r).astype(np.uint16)
    return r, values(r, "bf16")


def values(a, ty):
    return a.astype(np.float64) if ty != "bf16" else (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
