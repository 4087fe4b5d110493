"""Rows of vocabulary logits at places where top logits, distillation and draft verification have gone wrong, each
against a form of its own in 64 bits or more."""
import os

import numpy as np
import pytest
import torch

import distill_cases as D
import rust_trainer_amd as rt
from rust_trainer_amd.distill import distill_d, teacher_d, top_logits_d, verify_draft_d

pytestmark = pytest.mark.gpu

TYPES = {"f32": (rt.TYPE_F32, torch.float32), "f16": (rt.TYPE_F16, torch.float16), "bf16": (rt.TYPE_BF16, torch.bfloat16)}
HALF = 2.0 ** -24
# a sum of f32 exponentials, relative: 2^-22 each and 2^-22 for the f32 additions among eight; the roundings of an
# argument and of the scale log2(e) / T, 2^-24 of |z - max| / T each, at most 12.6 on average over a softmax
SUM = 2.0 ** -21 + 12.6 * 2 * 2.0 ** -24


@pytest.fixture(scope="module", params=["-1", "0", "1", "2"])
def each_ctx(request):
    """A context whose distillation runs on slices, or a row a workgroup of 256, 512 or 1024 threads, whatever the size."""
    os.environ["RTQ_DISTILL_ROWS"] = request.param
    c = rt.Context(0)
    del os.environ["RTQ_DISTILL_ROWS"]
    yield c
    c.close()


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def stream():
    return torch.cuda.current_stream().cuda_stream


def losses(ctx, z, ids, vals, rest, temp, tok=None, w=None, hard=0.0, ty="f32"):
    """(kl, logp, gradient) of device rows, as 64-bit numpy arrays (None where there is none)."""
    n, V = z.shape
    z = dev(z.astype(np.float32), TYPES[ty][1])
    keep = [dev(np.asarray(ids, np.int32)), dev(np.asarray(vals, np.float32))]
    keep += [None if a is None else dev(np.asarray(a, t)) for a, t in ((rest, np.float32), (tok, np.int32), (w, np.float32))]
    di, dv, dr, dt, dw = keep
    kl, lp = torch.full((n,), 7.0, device="cuda"), None if tok is None else torch.full((n,), 7.0, device="cuda")
    g = None if w is None else torch.full((n, V), 7.0, dtype=TYPES[ty][1], device="cuda")
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    distill_d(ctx, z.data_ptr(), TYPES[ty][0], n, V, V, teacher_d(di.shape[1], di.data_ptr(), dv.data_ptr(), ptr(dr), temp), ptr(dt), ptr(dw),
              kl.data_ptr(), ptr(lp), ptr(g), V, hard=hard, stream=stream())
    torch.cuda.synchronize()
    return [None if t is None else t.double().cpu().numpy() for t in (kl, lp, g)]


def divergence(z, ids, vals, rest, temp):
    """kl of one row from its definition: a bucket for each token that is listed, one for all others."""
    weights = {}
    for i, v in zip(ids, vals):
        if 0 <= i < len(z):
            weights[int(i)] = np.logaddexp(weights.get(int(i), -np.inf), float(v) / temp)
    others = np.ones(len(z), bool)
    others[list(weights)] = False
    lt = np.array(list(weights.values()) + [-np.inf if rest is None else float(rest)])
    lq = z / temp - D.lse(z / temp)
    lq = np.append(lq[list(weights)], D.lse(lq[others]) if others.any() else -np.inf)
    lp = lt - D.lse(lt)
    on = lp > -np.inf
    return float(np.sum(np.exp(lp[on]) * (lp[on] - lq[on])))


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_slots_of_one_token_are_one_bucket(each_ctx, ty):
    """A token in several slots has the sum of their weights: the divergence is that of the merged list, at least 0."""
    q = np.repeat(np.log([[0.9, 0.1]]), 3, 0)
    kl, _, _ = losses(each_ctx, q, [[0, 0], [0, 0], [1, 1]], [[1.0, 1.0]] * 3, [-np.inf, 1.0, -np.inf], 1.0)
    # p = (1, 0): log(1 / 0.9); p = (2/3, 1/3); p = (1 at the other token, 0): log(1 / 0.1)
    want = [np.log(1 / 0.9), 2 / 3 * np.log(2 / 2.7) + 1 / 3 * np.log(1 / 0.3), np.log(10)]
    assert np.all(np.abs(kl - want) <= 2 * SUM + HALF * np.abs(want) + 2.0 ** -23)  # (and the roundings of the logits handed over)
    V, k, n, temp = 9000, 12, 8, 1.25
    rng = np.random.default_rng(1)
    z = D.logits(rng, n, V)
    vals, ids, rest = D.top(D.logits(rng, n, V, near=z), k, temp)
    ids[0, 1] = ids[0, 0]
    ids[1, [2, 5, 11]] = ids[1, 8]
    ids[2] = ids[2, 0]  # one token alone
    ids[3, 6:] = ids[3, :6]  # each twice
    ids[4, 4], ids[4, 5] = ids[4, 0], -1
    ids[5, 3:] = V - 1
    vals[6, 2], ids[6, 2] = -np.inf, ids[6, 0]
    z[7, ids[7, 0]], ids[7, 3] = 11.0, ids[7, 0]
    _, z64 = D.rounded(z, ty)
    vals, rest = vals.astype(np.float32), rest.astype(np.float32)
    for r in (rest, None):
        for w in (None, np.ones(n)):
            kl, _, _ = losses(each_ctx, z64, ids, vals, r, temp, w=w, ty=ty)
            want = np.array([divergence(z64[i], ids[i], vals[i], None if r is None else r[i], temp) for i in range(n)])
            assert np.all(want >= 0) and np.all(np.abs(kl - want) <= 2 * SUM + HALF * np.abs(want)), kl - want


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,k", [(40, 3), (700, 20), (20000, 8), (40000, 256)])
def test_rest_of_a_nan_beside_infinity_is_nan(ctx, ty, V, k):
    """More NaNs than are listed, and +inf: the log of the sum of the others is NaN, as it is without the infinity;
    of +inf alone it is +inf."""
    rng = np.random.default_rng(V)
    z = rng.normal(0, 1, (8, V))
    spots = rng.permutation(V)
    for i, lead in enumerate((1, 2, V - 2 * k - 2)):
        z[i, spots[:k + lead]] = np.nan
        z[i, spots[k + lead]] = np.inf  # anywhere
    z[3, :k + 1], z[3, k + 1:2 * k + 3] = np.nan, np.inf  # side by side
    z[4, V - 1 - k:], z[4, 0] = np.nan, np.inf
    z[5, spots[:k + 1]] = np.inf
    z[6, spots[:k + 1]] = np.nan
    z[7, spots[:k]], z[7, spots[k]] = np.nan, np.inf
    zd = dev(z, TYPES[ty][1])
    vals, ids = torch.empty(8, k, device="cuda"), torch.empty(8, k, dtype=torch.int32, device="cuda")
    rest = torch.full((8,), 7.0, device="cuda")
    top_logits_d(ctx, zd.data_ptr(), TYPES[ty][0], 8, V, V, k, vals.data_ptr(), ids.data_ptr(), rest.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    rest = rest.cpu().numpy()
    assert np.isnan(rest[:5]).all() and rest[5] == np.inf and np.isnan(rest[6]) and rest[7] == np.inf, rest
    # a NaN is above every number, +inf among them
    order = np.lexsort((np.broadcast_to(np.arange(V), z.shape), -np.nan_to_num(z, nan=0.0, posinf=np.inf), ~np.isnan(z)), axis=1)
    np.testing.assert_array_equal(ids.cpu().numpy(), order[:, :k])


@pytest.mark.parametrize("temp", [1.0, 0.75, 2.0])
@pytest.mark.parametrize("V", [2, 20001])
def test_draws_and_tests_at_the_borders_are_exact_to_64_bits(ctx, V, temp):
    """Two live tokens whose border w0 / (w0 + w1) lies 2e-14 to 1e-12 of itself beside the uniform number (placed with
    a logit next to 0, whose float steps are that fine; expected values in extended precision).  A weight's
    exponential is off by a few 2^-53: of its table and polynomial, and of its argument, 2^-52 |z - max| / T."""
    L = np.longdouble
    rng = np.random.default_rng(int(temp * 100) + V)
    z1 = rng.uniform(-3, 3, 400).astype(np.float32)
    u = (1 / (1 + np.exp(z1.astype(L) / L(temp)))).astype(np.float32)
    off = np.tile([2e-14, -2e-14, 1e-13, -1e-13, 5e-13, -5e-13, 1e-12, -1e-12], 50).astype(L)
    # w0 / w1 = u / (1 - u) (1 + off) (off the border by (1 - u) off of itself)
    z0 = (z1.astype(L) + L(temp) * (np.log(u.astype(L)) - np.log1p(-u.astype(L)) + off)).astype(np.float32)
    e = np.exp((z0.astype(L) - z1.astype(L)) / L(temp))
    border = e / (1 + e)
    ok = np.abs(border / u.astype(L) - 1) > 4e-15
    assert ok.sum() > 300
    z0, z1, u, border = z0[ok], z1[ok], u[ok], border[ok]
    b = len(u)
    i, j = (0, 1) if V == 2 else (4321, 17000)
    z = np.full((b, V), -np.inf, np.float32)
    z[:, i], z[:, j] = z0, z1
    zd, ud = dev(z), dev(u)
    acc, out = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, 1, dtype=torch.int32, device="cuda")
    verify_draft_d(ctx, zd.data_ptr(), rt.TYPE_F32, V, 0, 0, b, 0, V, 0, 0, ud.data_ptr(), acc.data_ptr(), out.data_ptr(), temperature=temp, stream=stream())
    torch.cuda.synchronize()
    # drawn: the first token whose running sum passes u times the total
    np.testing.assert_array_equal(out.cpu().numpy()[:, 0], np.where(border > u, i, j))
    # a looked-up draft of that token is accepted while u < p
    zz, uu, x = dev(np.repeat(z, 2, 0)), dev(np.stack([u, u], 1)), torch.full((b, 1), i, dtype=torch.int32, device="cuda")
    out = torch.empty(b, 2, dtype=torch.int32, device="cuda")
    verify_draft_d(ctx, zz.data_ptr(), rt.TYPE_F32, V, 0, 0, b, 1, V, x.data_ptr(), 0, uu.data_ptr(), acc.data_ptr(), out.data_ptr(), temperature=temp,
                   stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(acc.cpu().numpy(), (u < border).astype(np.int32))


@pytest.mark.parametrize("temp", [1.0, 1.25, 1.44, 2.8848, 0.0907])
def test_large_losses_carry_no_scale_of_32_bits(each_ctx, temp):
    """A teacher that is certain of a token far below the student's best: kl is (max - z) / T to the rounding of the
    result, whatever log2(e) / T rounds to as a float; the same for a label's log-probability."""
    V, n = 3001, 64
    rng = np.random.default_rng(7)
    z = rng.normal(0, 1, (n, V)).astype(np.float32)
    at = rng.integers(0, V, (n, 1))
    np.put_along_axis(z, at, -rng.uniform(2e3, 6e4, (n, 1)).astype(np.float32), 1)
    z64, t = z.astype(np.float64), float(np.float32(temp))
    vals, tok = np.zeros((n, 1)), at[:, 0]
    kl, lp, _ = losses(each_ctx, z, at, vals, None, temp, tok=tok)
    want = -(np.take_along_axis(z64, at, 1)[:, 0] / t - D.lse(z64 / t))
    assert np.all(np.abs(kl - want) <= 2 * SUM + HALF * want), np.abs(kl / want - 1).max() / HALF
    want = np.take_along_axis(z64, at, 1)[:, 0] - D.lse(z64)
    assert np.all(np.abs(lp - want) <= SUM + HALF * np.abs(want)), np.abs(lp / want - 1).max() / HALF


def test_the_rest_does_not_depend_on_the_order_of_gathering(ctx):
    """Rows whose rest is next to 0, where a float's steps are finest: the same bits from call to call."""
    rng = np.random.default_rng(3)
    for V, k in ((6000, 200), (20000, 200), (60000, 256)):
        n = 512
        z = rng.normal(0, 1.0, (n, V))
        z -= D.top(z, k, 1.0)[2][:, None]
        zd = dev(z.astype(np.float32))
        first = None
        for rep in range(6):
            vals, ids, rest = torch.empty(n, k, device="cuda"), torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
            top_logits_d(ctx, zd.data_ptr(), rt.TYPE_F32, n, V, V, k, vals.data_ptr(), ids.data_ptr(), rest.data_ptr(), stream=stream())
            torch.cuda.synchronize()
            assert float(rest.abs().max()) < 1e-3
            first = rest if first is None else first
            assert torch.equal(first, rest), (V, k, rep, int((first != rest).sum()))


def test_many_verification_rows(ctx):
    """More rows than one grid dimension holds."""
    b, d, V = 300, 130, 5
    rng = np.random.default_rng(9)
    zp, zq = rng.normal(0, 1, (b * (d + 1), V)).astype(np.float32), rng.normal(0, 1, (b * d, V)).astype(np.float32)
    zq.reshape(b, d, V)[150:] = zp.reshape(b, d + 1, V)[150:, :d]  # accepted far
    x = np.argmax(zq, 1).reshape(b, d).astype(np.int32)
    u = rng.random((b, d + 1)).astype(np.float32)
    assert b * (2 * d + 1) > 65535
    args = [dev(a) for a in (zp, zq, x, u)]
    for temp, draft in ((1.0, True), (1.0, False), (0.0, False)):
        acc, out = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, d + 1, dtype=torch.int32, device="cuda")
        verify_draft_d(ctx, args[0].data_ptr(), rt.TYPE_F32, V, args[1].data_ptr() if draft else 0, V if draft else 0, b, d, V, args[2].data_ptr(), 0,
                       args[3].data_ptr(), acc.data_ptr(), out.data_ptr(), temperature=temp, stream=stream())
        torch.cuda.synchronize()
        want = D.verify(zp, zq if draft else None, x, None, u, temp)
        np.testing.assert_array_equal(acc.cpu().numpy(), want[0])
        np.testing.assert_array_equal(out.cpu().numpy(), want[1])


@pytest.mark.parametrize("hard", [0.0, 0.5])
def test_rows_without_a_teacher_or_a_weight_beside_bad_logits(each_ctx, hard):
    """What is not asked of a row stays 0 whatever its logits: no teacher, no divergence and none of its gradient; weight
    0, no gradient.  What is asked of it is NaN."""
    V, n, k = 9000, 6, 3
    rng = np.random.default_rng(10)
    z = D.logits(rng, n, V)
    z[0, 5], z[1, 6], z[3, 5], z[4, 5] = np.nan, np.inf, np.nan, np.nan
    z[2] = -np.inf
    ids = np.array([[1, 2, 3]] * n)
    ids[[0, 1, 2, 4]] = -1
    rest = np.zeros(n)
    rest[[0, 1, 2, 4]] = -np.inf
    w = np.array([1.0, 1, 1, 0, 0, 1])
    for ty in ("f32", "bf16"):
        kl, lp, g = losses(each_ctx, z, ids, np.zeros((n, k)), rest, 1.0, rng.integers(0, V, n), w, hard, ty)
        assert not kl[[0, 1, 2, 4]].any() and np.isnan(kl[3]) and np.isfinite(kl[5])
        assert np.isnan(lp[:5]).all() and np.isfinite(lp[5])
        assert np.isnan(g[:3]).all() if hard else not g[:3].any()
        assert not g[3:5].any() and np.isfinite(g[5]).all() and g[5].any()


def test_heads_of_an_empty_sequence(ctx):
    """No hidden states: every position is out of range, so the losses are NaN, the lists empty and dx has no rows."""
    import ctypes

    V, d, n, k = 700, 64, 3, 4
    rng = np.random.default_rng(11)
    f = rt.HipFrozen.f32(rng.normal(0, 0.1, (V, d)), V, d, ctx=ctx)
    norm, x, pos = torch.ones(d, device="cuda"), torch.ones(d, device="cuda"), dev(np.array([0, 1, -1], np.int32))
    tok, w, dx = dev(np.array([1, 2, 3], np.int32)), torch.ones(n, device="cuda"), torch.full((d,), 7.0, device="cuda")
    ids, vals = dev(np.arange(n * k, dtype=np.int32)), torch.zeros(n, k, device="cuda")
    kl, lp, hit = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    te = rt._ffi.RtqTeacher(k, ids.data_ptr(), vals.data_ptr(), None, 1.0)
    head = (ctx.handle, f.handle, norm.data_ptr(), 1e-6, 0.0, x.data_ptr(), 0, pos.data_ptr())
    rt._ffi.check(rt.lib().rtq_lm_distill_d(*head, tok.data_ptr(), w.data_ptr(), n, ctypes.byref(te), 0.5, kl.data_ptr(), lp.data_ptr(), dx.data_ptr(),
                                            stream() or None), "distill")
    torch.cuda.synchronize()
    assert torch.isnan(kl).all() and torch.isnan(lp).all()
    lp.zero_()
    rt._ffi.check(rt.lib().rtq_lm_head_d(*head, tok.data_ptr(), w.data_ptr(), n, lp.data_ptr(), hit.data_ptr(), dx.data_ptr(), stream() or None), "head")
    torch.cuda.synchronize()
    assert torch.isnan(lp).all() and not hit.any()
    rt._ffi.check(rt.lib().rtq_lm_top_logits_d(*head, n, k, 1.0, vals.data_ptr(), ids.data_ptr(), kl.data_ptr(), stream() or None), "top")
    torch.cuda.synchronize()
    assert torch.isnan(vals).all() and (ids == -1).all() and torch.isnan(kl).all()
    assert torch.equal(dx, torch.full_like(dx, 7.0))
    f.close()
