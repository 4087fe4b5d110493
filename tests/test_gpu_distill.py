"""Top logits, distillation and draft verification on the GPU against plain 64-bit forms (distill_cases.py).

Tolerances: whole numbers and selected logits are equal.  A log-sum-exp is off by D.SUM (a relative error of its
sum) and half a step; kl by D.SUM for each of the two it holds and half a step; a gradient element by D.SUM and
one more exponential (2^-22, and its argument's roundings: |z - max| / T of 2^-24 for itself and 2^-25 for the
scale, doubled for the label's at T = 1) of the magnitudes it is a difference of, and half a step of its type."""

import numpy as np
import pytest
import torch

import distill_cases as D
import rust_trainer_amd as rt
from rust_trainer_amd.distill import distill_d, teacher_d, top_logits_d, verify_draft_d

pytestmark = pytest.mark.gpu

TYPES = {"f32": (rt.TYPE_F32, torch.float32), "f16": (rt.TYPE_F16, torch.float16), "bf16": (rt.TYPE_BF16, torch.bfloat16)}
HALF = 2.0 ** -24


def dev(a, ty=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t.view(torch.bfloat16) if ty == "bf16" else t).cuda()


def rows(a, ty, pad=0, shift=0):
    """a on the device in rows V + pad apart, the first `shift` elements into its allocation; what lies between
    holds NaN.  Returns (the allocation, the [n x V] view)."""
    n, V = a.shape
    mem = torch.full((shift + n * (V + pad) + 8,), float("nan"), dtype=TYPES[ty][1], device="cuda")
    view = mem[shift:shift + n * (V + pad)].view(n, V + pad)[:, :V] if n else mem[:0].view(0, V)
    view.copy_(dev(a, ty))
    return mem, view


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def run_top(ctx, view, ty, k, temp, rest=True):
    n, V = view.shape
    vals, ids = torch.full((n, k), 7.0, device="cuda"), torch.full((n, k), -7, dtype=torch.int32, device="cuda")
    r = torch.full((n,), 7.0, device="cuda") if rest else None
    top_logits_d(ctx, view.data_ptr(), TYPES[ty][0], n, V, view.stride(0), k, vals.data_ptr(), ids.data_ptr(),
                 r.data_ptr() if rest else 0, temperature=temp, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return vals.cpu().numpy(), ids.cpu().numpy(), r.cpu().numpy() if rest else None


def check_top(ctx, z, ty, k, temp=1.0, pad=0, shift=0):
    a, z64 = D.rounded(z, ty)
    _, view = rows(a, ty, pad, shift)
    vals, ids, rest = run_top(ctx, view, ty, k, temp)
    v, j, r = D.top(z64, k, float(np.float32(temp)))
    np.testing.assert_array_equal(ids, j)
    np.testing.assert_array_equal(vals.astype(np.float64), v)
    check_lse(rest, r)
    return view


def check_lse(got, want, each=1):
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin].astype(np.float32))
    err = np.abs(got[fin] - want[fin])
    assert np.all(err <= each * D.SUM + HALF * np.abs(want[fin])), float(err.max())


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,V,k,temp,pad,shift", [
    (1, 1, 1, 1.0, 0, 0), (2, 2, 2, 1.0, 1, 1), (3, 7, 5, 0.5, 0, 3), (5, 63, 63, 1.0, 2, 0), (4, 1000, 256, 2.0, 0, 1),
    (3, 8191, 20, 1.0, 0, 0), (3, 8193, 64, 1.0, 5, 7), (2, 16385, 1, 4.0, 0, 2), (37, 50257, 8, 1.0, 0, 0), (2, 151936, 256, 1.0, 0, 0),
    (1, 300001, 100, 1.0, 0, 0), (300, 257, 17, 1.0, 0, 1), (1, 1 << 20, 256, 1.0, 0, 0)])
def test_top_logits(ctx, ty, n, V, k, temp, pad, shift):
    check_top(ctx, D.logits(np.random.default_rng(V + k), n, V), ty, k, temp, pad, shift)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_top_logits_of_rows_that_defeat_the_bound(ctx, ty):
    """All equal, sorted either way, one slice that holds everything, few live logits among -inf or the type's
    lowest value, +-0, blocks of ties: more logits reach the bound than are gathered at once."""
    V, k = 40000, 100
    rng = np.random.default_rng(1)
    z = rng.normal(0, 2, (12, V))
    z[0] = 1.5
    z[1] = np.linspace(-20, 20, V)
    z[2] = np.linspace(20, -20, V)
    z[3, :9000] += 30
    z[4, 50:] = -np.inf
    z[5, 50:] = -3e38
    z[6] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    z[7] = rng.integers(0, 3, V)
    z[8, ::64] += 25  # one lane's logits
    z[9] = -np.inf
    z[9, 39999] = 0.0
    z[10] = -3e38
    z[11, 30000:] = 11.0
    check_top(ctx, z, ty, k)
    check_top(ctx, z, ty, 256, 2.0, pad=1)
    check_top(ctx, z, ty, 1)


def test_top_logits_nan_and_infinity(ctx):
    z = np.random.default_rng(2).normal(0, 1, (4, 20000))
    z[0, [5, 19000]] = np.nan
    z[1, 7] = np.inf
    z[2, :5000] = np.nan
    z[3, :300] = np.inf
    a, z64 = D.rounded(z, "f32")
    _, view = rows(a, "f32")
    vals, ids, rest = run_top(ctx, view, "f32", 8, 1.0)
    v, j, r = D.top(z64, 8, 1.0)
    np.testing.assert_array_equal(ids, j)
    np.testing.assert_array_equal(vals, v.astype(np.float32))
    assert np.isnan(rest[2]) and rest[3] == np.inf
    check_lse(rest[:2], r[:2])
    vals2, ids2, none = run_top(ctx, view, "f32", 8, 1.0, rest=False)
    assert none is None and np.array_equal(ids2, ids)


def check_distill(ctx, z, ids, vals, rest, temp, tok=None, w=None, hard=0.0, ty="f32", pad=0, shift=0, dpad=0, in_place=False, kl_rel=HALF):
    a, z64 = D.rounded(z, ty)
    n, V = a.shape
    k = ids.shape[1]
    mem, view = rows(a, ty, pad, shift)
    ids, vals = np.ascontiguousarray(ids, np.int32), np.ascontiguousarray(vals, np.float32)
    rest = None if rest is None else np.ascontiguousarray(rest, np.float32)
    w = None if w is None else np.ascontiguousarray(w, np.float32)
    di, dv, dr = dev(ids), dev(vals), None if rest is None else dev(rest)
    dt = None if tok is None else dev(np.ascontiguousarray(tok, np.int32))
    dw = None if w is None else dev(w)
    kl, lp = torch.full((n,), 7.0, device="cuda"), None if tok is None else torch.full((n,), 7.0, device="cuda")
    if in_place:
        gmem, gview = mem, view
    else:
        gmem, gview = rows(np.zeros((n, V), a.dtype), ty, dpad, shift)
    before = gmem.clone()
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    distill_d(ctx, view.data_ptr(), TYPES[ty][0], n, V, view.stride(0), teacher_d(k, di.data_ptr(), dv.data_ptr(), ptr(dr), temp), ptr(dt),
              ptr(dw), kl.data_ptr(), ptr(lp), gview.data_ptr() if w is not None else 0, gview.stride(0), hard=hard,
              stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    rk, rl, rg, sc = D.distill(z64, ids, vals.astype(np.float64), rest, float(np.float32(temp)), tok, w, hard)  # (a float in the call)
    got = kl.cpu().numpy().astype(np.float64)
    fin = np.isfinite(rk)
    np.testing.assert_array_equal(got[~fin], rk[~fin])
    assert np.all(np.abs(got[fin] - rk[fin]) <= 2 * D.SUM + kl_rel * np.abs(rk[fin])), float(np.abs(got[fin] - rk[fin]).max())
    if tok is not None:
        got = lp.cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(rl))
        ok = np.isfinite(rl)
        np.testing.assert_array_equal(got[~ok], rl[~ok])
        assert np.all(np.abs(got[ok] - rl[ok]) <= D.SUM + HALF * np.abs(rl[ok]))
    outside = torch.ones_like(gmem, dtype=torch.bool)
    if w is not None:
        inside = outside[shift:shift + n * gview.stride(0)].view(n, gview.stride(0))[:, :V] if n else outside[:0]
        inside[:] = False
        got = host(gview)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(rg))
        with np.errstate(all="ignore"):
            depth = np.abs(z64 - np.where(np.isfinite(z64), z64, -np.inf).max(1, keepdims=True)) * 2 * HALF / min(temp, 1.0)
            bound = np.where(sc > 0, sc * (D.SUM + 2.0 ** -22 + np.minimum(depth, 1.0)), 0.0) + np.abs(rg) * D.EPS[ty] * (1 + 1e-5) + D.TINY[ty]
        bad = ~np.isnan(rg) & ~(np.abs(got - rg) <= bound)
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], rg[bad][:5], bound[bad][:5])
    # what lies outside the gradient's rows is left as it was (NaN equals NaN here)
    assert torch.equal(gmem[outside].view(torch.int16 if ty != "f32" else torch.int32), before[outside].view(torch.int16 if ty != "f32" else torch.int32))
    return kl, gview


def teacher(rng, z, k, temp, ragged=False):
    n, V = z.shape
    t = D.logits(rng, n, V, near=np.where(np.isfinite(z), z, -30.0))
    vals, ids, rest = D.top(t, k, temp)
    if ragged:
        held = rng.integers(0, k + 1, n)
        held[0] = 0
        ids = np.where(np.arange(k) < held[:, None], ids, -1)
        rest = np.where(held == 0, -np.inf, rest)
    return ids, vals, rest


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,V,k,temp,hard,rest,ragged,pad,shift", [
    (1, 1, 1, 1.0, 0.5, True, False, 0, 0), (2, 2, 1, 1.0, 0.0, True, False, 0, 1), (3, 7, 7, 2.0, 0.25, False, False, 1, 0),
    (4, 33, 5, 1.0, 1.0, True, True, 3, 1), (12, 8192, 20, 1.0, 0.0, False, False, 0, 0), (5, 8193, 256, 0.5, 0.5, True, True, 0, 3),
    (3, 16385, 33, 4.0, 0.25, True, False, 7, 0), (2, 50257, 64, 1.25, 0.5, True, False, 0, 5), (2, 151936, 128, 2.0, 0.0, True, False, 0, 0),
    (1, 200003, 100, 1.0, 0.3, True, False, 0, 0), (260, 515, 9, 1.0, 0.3, True, True, 0, 0)])
def test_distill(ctx, ty, n, V, k, temp, hard, rest, ragged, pad, shift):
    rng = np.random.default_rng(V * 3 + k)
    z = D.logits(rng, n, V)
    ids, vals, r = teacher(rng, z, k, temp, ragged)
    tok, w = rng.integers(0, V, n), rng.uniform(0.25, 2.0, n)
    tok[: n // 2] = np.maximum(ids[: n // 2, 0], 0)  # labels among the listed tokens
    r = r if rest else None
    _, g = check_distill(ctx, z, ids, vals, r, temp, tok, w, hard, ty, pad, shift, dpad=pad)
    # the gradient over the logits themselves: the same bits
    _, g2 = check_distill(ctx, z, ids, vals, r, temp, tok, w, hard, ty, pad, shift, in_place=True)
    assert torch.equal(g.contiguous().view(torch.uint8), g2.contiguous().view(torch.uint8))
    # losses alone, without labels
    check_distill(ctx, z, ids, vals, r, temp, ty=ty, pad=pad, shift=shift)


@pytest.fixture(scope="module", params=["-1", "0", "1", "2"])
def each_ctx(request):
    """A context whose distillation runs on slices, or a row a workgroup of 256, 512 or 1024 threads, whatever the size."""
    import os

    os.environ["RTQ_DISTILL_ROWS"] = request.param
    c = rt.Context(0)
    del os.environ["RTQ_DISTILL_ROWS"]
    yield c
    c.close()


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("n,V,k,temp,hard", [(1, 3, 2, 1.0, 0.5), (2, 6143, 30, 2.0, 0.25), (3, 40001, 256, 1.0, 0.5), (1, 170003, 20, 0.5, 0.0), (1, 1 << 20, 64, 1.0, 0.5)])
def test_distill_on_every_kernel(each_ctx, ty, n, V, k, temp, hard):
    rng = np.random.default_rng(V)
    z = D.logits(rng, n, V)
    ids, vals, r = teacher(rng, z, k, temp)
    tok, w = rng.integers(0, V, n), rng.uniform(0.25, 2.0, n)
    _, g = check_distill(each_ctx, z, ids, vals, r, temp, tok, w, hard, ty, pad=3, shift=1)
    _, g2 = check_distill(each_ctx, z, ids, vals, r, temp, tok, w, hard, ty, pad=3, shift=1, in_place=True)
    assert torch.equal(g.contiguous().view(torch.uint8), g2.contiguous().view(torch.uint8))


def test_distill_rows_at_the_edges_on_every_kernel(each_ctx):
    test_distill_rows_at_the_edges(each_ctx)
    test_distill_nan_and_infinite_rows(each_ctx)


def test_distill_rows_at_the_edges(ctx):
    """Empty slots and ids out of range, a token listed twice and three times, no teacher, weight 0, labels out of
    range, masked logits (-inf and the lowest value) outside and inside the list, a student that gives the
    rest nothing, a teacher that is certain, one that lists nothing but has a rest."""
    V, k, n = 9000, 6, 16
    rng = np.random.default_rng(8)
    z = D.logits(rng, n, V)
    ids, vals, rest = teacher(rng, z, k, 1.0)
    tok, w = rng.integers(0, V, n), rng.uniform(0.5, 1.5, n)
    ids[0, 2] = ids[0, 0]
    ids[1, 1] = ids[1, 4] = ids[1, 5] = 8999
    ids[2] = -1
    rest[2] = -np.inf
    ids[3, 3:] = [-5, V, 2 ** 30]
    w[4] = 0.0
    z[4, 5] = np.nan
    tok[5], tok[6] = -100, V
    z[7, 100:8000] = -np.inf
    z[8, 100:8000] = -3.0e38
    others = np.setdiff1d(np.arange(V), ids[9])
    z[9, others] = -np.inf
    tok[9] = ids[9, 0]
    z[10, ids[10, 1]] = -np.inf
    vals[11] = [300, 0, 0, 0, 0, 0]
    rest[11] = -np.inf
    ids[12] = -1
    vals[13] = -np.inf
    rest[14] = 300.0
    z[15, np.setdiff1d(np.arange(V), ids[15])] -= 300.0  # far below: exp underflows against the listed
    for tv in (0.0, 0.5, 1.0):
        for ty in ("f32", "bf16"):
            check_distill(ctx, z, ids, vals, rest, 1.0, tok, w, tv, ty)
    check_distill(ctx, z, ids, vals, None, 2.0, tok, w, 0.5)


@pytest.mark.parametrize("temp", [1.0, 0.25, 3.0])
def test_distill_masks_of_any_size(each_ctx, temp):
    """Masked logits of -1e5 to -1e30 beside live ones, all but the list masked, and whole rows masked: the rest
    is small or nothing but every sum stays finite."""
    V, k = 9000, 6
    sizes = [-1e5, -1e8, -1e9, -1e10, -3e13, -1e20, -1e30]
    rng = np.random.default_rng(15)
    n = 3 * len(sizes)
    z = D.logits(rng, n, V)
    ids, vals, rest = teacher(rng, z, k, temp)
    for i, m in enumerate(sizes):
        z[i, np.setdiff1d(np.arange(100, 8000), ids[i])] = m
        z[len(sizes) + i, np.setdiff1d(np.arange(V), ids[len(sizes) + i])] = m
        rest[len(sizes) + i] = -np.inf
        z[2 * len(sizes) + i] = m
    tok, w = rng.integers(0, V, n), np.ones(n)
    tok[len(sizes):2 * len(sizes)] = ids[len(sizes):2 * len(sizes), 0]
    for ty in ("f32", "bf16"):
        check_distill(each_ctx, z, ids, vals, rest, temp, tok, w, 0.5, ty)
        check_distill(each_ctx, z, ids, vals, rest, temp, None, w, 0.0, ty)


@pytest.mark.parametrize("temp", [1e-4, 1e4])
def test_the_ends_of_the_temperatures(each_ctx, temp):
    """The divergence at 1e-4 is some 1e4 and proportional to 1 / T, whose scale log2(e) / T is a float: 2^-25 of it
    more than its own rounding, 2^-24."""
    V, k, n = 9000, 6, 5
    rng = np.random.default_rng(16)
    z = D.logits(rng, n, V)
    ids, vals, rest = teacher(rng, z, k, temp)
    for ty in ("f32", "f16"):
        check_distill(each_ctx, z, ids, vals, rest, temp, rng.integers(0, V, n), np.ones(n), 0.5, ty, kl_rel=1.5 * HALF)
        test_top_logits(each_ctx, ty, n, V, k, temp, 0, 0)
        test_verify_draft(each_ctx, ty, n, 3, V, temp, True, False, 0, 0)


def test_distill_nan_and_infinite_rows(ctx):
    V, k = 20000, 4
    rng = np.random.default_rng(9)
    z = D.logits(rng, 6, V)
    ids, vals, rest = teacher(rng, z, k, 1.0)
    tok, w = rng.integers(0, V, 6), np.ones(6)
    z[0, 11] = np.nan
    z[1, ids[1, 0]] = np.nan
    z[2] = -np.inf
    z[3, 19999] = np.inf
    vals[4, 1] = np.nan
    a, _ = D.rounded(z, "f32")
    kl, lp, g = rt.distill(a, rt.Teacher(ids, vals, rest), tok, w, hard=0.5, ctx=ctx)
    assert np.isnan(kl[:5]).all() and np.isnan(lp[:4]).all() and np.isnan(g[:4]).all()
    assert np.isfinite(kl[5]) and np.isfinite(lp[4:]).all() and np.isfinite(g[5]).all()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b,d,V,temp,draft,ragged,pad,shift", [
    (1, 0, 5, 1.0, False, False, 0, 0), (1, 1, 1, 1.0, True, False, 0, 1), (3, 2, 2, 1.0, True, True, 1, 0), (1, 4, 151936, 1.0, True, False, 0, 0),
    (9, 3, 50257, 0.75, False, True, 3, 1), (33, 5, 1000, 2.0, True, True, 0, 0), (17, 3, 8193, 0.0, True, True, 0, 3), (5, 40, 300, 0.5, True, False, 0, 0),
    (40, 1, 16385, 4.0, False, False, 0, 0)])
def test_verify_draft(ctx, ty, b, d, V, temp, draft, ragged, pad, shift):
    rng = np.random.default_rng(V + b)
    zp = D.logits(rng, b * (d + 1), V)
    zq = D.logits(rng, b * d, V, near=zp.reshape(b, d + 1, V)[:, :d].reshape(b * d, V)) if b * d else np.zeros((0, V))
    x = np.array([rng.choice(V, p=np.exp(r / max(temp, 0.5) - D.lse(r / max(temp, 0.5)))) if temp else int(np.argmax(r)) for r in zq]).reshape(b, d)
    check_verify(ctx, zp, zq if draft else None, x, rng.integers(0, d + 1, b) if ragged else None, rng.random((b, d + 1)), temp, ty, pad, shift)


def check_verify(ctx, zp, zq, x, lens, u, temp, ty="f32", pad=0, shift=0):
    b, d = x.shape
    a, z64 = D.rounded(zp, ty)
    V = a.shape[1]
    _, view = rows(a, ty, pad, shift)
    q64, qv = None, None
    if zq is not None:
        aq, q64 = D.rounded(zq, ty)
        _, qv = rows(aq, ty, pad, shift)
    x, u = np.ascontiguousarray(x, np.int32), np.ascontiguousarray(np.minimum(u, 1 - 2.0 ** -24), np.float32)
    dx, du = dev(x), dev(u)
    dl = None if lens is None else dev(np.ascontiguousarray(lens, np.int32))
    acc, out = torch.full((b,), -7, dtype=torch.int32, device="cuda"), torch.full((b, d + 1), -7, dtype=torch.int32, device="cuda")
    verify_draft_d(ctx, view.data_ptr(), TYPES[ty][0], V + pad, 0 if qv is None else qv.data_ptr(), V + pad, b, d, V, dx.data_ptr(),
                   0 if dl is None else dl.data_ptr(), du.data_ptr(), acc.data_ptr(), out.data_ptr(), temperature=temp,
                   stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = D.verify(z64, q64, x, lens, u, float(np.float32(temp)))
    np.testing.assert_array_equal(acc.cpu().numpy(), want[0])
    np.testing.assert_array_equal(out.cpu().numpy(), want[1])


def test_verify_draft_at_the_edges(ctx):
    """Uniform numbers of 0 and next to 1, drafted ids out of range, a target that excludes the token, a draft equal
    to the target, masked vocabularies, a certain target, lengths outside [0, d], NaN and -inf rows, equal
    largest logits."""
    b, d, V = 14, 3, 10000
    rng = np.random.default_rng(4)
    zp = D.logits(rng, b * (d + 1), V)
    zq = D.logits(rng, b * d, V, near=zp.reshape(b, d + 1, V)[:, :d].reshape(b * d, V))
    x = np.argmax(zq, 1).reshape(b, d).astype(np.int64)
    u = rng.random((b, d + 1))
    T, Q = zp.reshape(b, d + 1, V), zq.reshape(b, d, V)
    u[0] = 0.0
    u[1] = 1.0
    x[2, 1] = -1
    x[3, 0] = V
    T[4, 0, x[4, 0]] = -np.inf
    Q[5] = T[5, :d]
    T[6, :, 5000:] = -np.inf
    Q[6, :, 5000:] = -np.inf
    x[6] = np.argmax(Q[6], 1)
    T[7, :, 123] = 500.0
    T[8, 1] = -np.inf
    u[8, 0] = 0.0
    T[9, 0, 77] = np.nan
    T[10, 2] = 1.25  # all equal
    T[11, :, :] = -3e38
    T[11, :, 9999] = 0.0
    Q[12, 0, x[12, 0]] = -np.inf  # a token its own draft excludes
    T[13, 3, 4000:] = -np.inf
    u[13, :d] = 0.0
    lens = np.full(b, d)
    for temp in (1.0, 0.0, 2.0):
        for ty in ("f32", "bf16"):
            check_verify(ctx, zp, zq, x, lens, u, temp, ty)
            check_verify(ctx, zp, None, x, None, u, temp, ty)
    lens[0], lens[1] = -3, 9
    check_verify(ctx, zp, zq, x, lens, u, 1.0)


def test_verify_draft_rows_without_a_distribution(ctx):
    """A target row of -inf alone, with a NaN or with +inf draws nothing (at temperature 0 the last has a largest
    logit); a draft row like that accepts nothing and leaves the draw to the target."""
    b, d, V = 7, 2, 5003
    rng = np.random.default_rng(14)
    zp = D.logits(rng, b * (d + 1), V)
    zq = D.logits(rng, b * d, V, near=zp.reshape(b, d + 1, V)[:, :d].reshape(b * d, V))
    T, Q = zp.reshape(b, d + 1, V), zq.reshape(b, d, V)
    x = np.argmax(T[:, :d], 2)
    u = np.zeros((b, d + 1))
    u[:, d] = 0.5
    for i, v in enumerate((np.nan, -np.inf, np.inf)):
        at = slice(None) if v == -np.inf else 4321
        T[i, i % d + (i == 2), at] = v  # rows 0, 1 and the last
        Q[3 + i, 1, at] = v
    for temp in (1.0, 0.0):
        for ty in ("f32", "f16", "bf16"):
            check_verify(ctx, zp, zq, x, None, u, temp, ty)
            check_verify(ctx, zp, None, x, None, u, temp, ty)
    acc, out = D.verify(zp, zq, x, None, u, 1.0)
    assert acc[:6].tolist() == [0, 1, 1, 1, 1, 1] and out[0, 0] == out[1, 1] == out[2, 1] == -1 and (out[3:6, 1] >= 0).all()


def test_host_calls_and_their_refusals(ctx):
    rng = np.random.default_rng(6)
    n, V, k = 5, 1003, 7
    wide = D.logits(rng, n, V + 20).astype(np.float32)
    z = wide[:, :V]  # rows V + 20 apart
    t = rt.top_logits(z, k, 2.0, ctx=ctx)
    v, j, r = D.top(z, k, 2.0)
    np.testing.assert_array_equal(t.ids, j)
    np.testing.assert_array_equal(t.vals, v)
    check_lse(t.rest, r)
    s = (z + rng.normal(0, 0.5, z.shape)).astype(np.float16)
    tok, w = rng.integers(0, V, n), np.ones(n)
    kl, lp, g = rt.distill(s, t, tok, w, hard=0.25, ctx=ctx)
    rk, rl, rg, sc = D.distill(s, t.ids, t.vals, t.rest, 2.0, tok, w, 0.25)
    assert np.all(np.abs(kl - rk) <= 2 * D.SUM + HALF * rk) and g.dtype == np.float16
    assert np.all(np.abs(g - rg) <= sc * 1e-5 + np.abs(rg) * D.EPS["f16"] + D.TINY["f16"])
    kl2, none, nog = rt.distill(s, t, ctx=ctx)
    assert np.array_equal(kl2, kl) and none.size == 0 and nog.shape == (0, V)
    for bad in (lambda: rt.distill(s, rt.Teacher(np.full((n, 1), V), np.zeros((n, 1))), ctx=ctx), lambda: rt.distill(s, t, np.full(n, V), w, ctx=ctx),
                lambda: rt.distill(s, t, np.full(n, -1), w, ctx=ctx), lambda: rt.top_logits(z, V + 1, ctx=ctx),
                lambda: rt.verify_draft(z[:4], [[1], [V]], np.zeros((2, 2)), ctx=ctx), lambda: rt.verify_draft(z[:4], [[1], [2]], np.ones((2, 2)), ctx=ctx),
                lambda: rt.verify_draft(z[:4], [[1], [2]], np.zeros((2, 2)), lens=[1, 2], ctx=ctx), lambda: rt.verify_draft(z[:4], [[1], [2]], ctx=ctx)):
        with pytest.raises(rt.RtqError):
            bad()
    x, u = np.argmax(z[:4].reshape(2, 2, V)[:, 0], 1)[:, None], rng.random((2, 2)).astype(np.float32)
    acc, out = rt.verify_draft(z[:4], x, u, ctx=ctx)
    want = D.verify(z[:4], None, x, None, u, 1.0)
    assert np.array_equal(acc, want[0]) and np.array_equal(out, want[1])
    acc, out = rt.verify_draft(z[:4], x, temperature=0.0, ctx=ctx)
    assert acc.tolist() == [1, 1]
    # no rows
    assert rt.top_logits(z[:0], 3, ctx=ctx).ids.shape == (0, 3)
    assert rt.distill(z[:0], rt.Teacher(np.zeros((0, 3)), np.zeros((0, 3))), ctx=ctx)[0].size == 0
    assert rt.verify_draft(z[:0], np.zeros((0, 2)), np.zeros((0, 3)), ctx=ctx)[1].shape == (0, 3)


def test_a_teacher_a_student_and_a_draft_together_on_a_stream_and_captured():
    """A teacher's top logits, the student's gradient from them and the verification of the student's drafts, eager
    on a side stream and as one replayed graph, with the context's workspace outgrown between replays; a
    capture that would have to grow it is refused."""
    ctx = rt.Context(0)
    rng = np.random.default_rng(11)
    b, d, V, k = 3, 4, 30011, 24
    n = b * (d + 1)
    zt = D.logits(rng, n, V)
    zs = D.logits(rng, n, V, near=zt)
    rows_d = [i * (d + 1) + j for i in range(b) for j in range(d)]
    T, S = dev(zt.astype(np.float32)), dev(zs.astype(np.float32))
    Q = S[rows_d].contiguous()
    x, u = dev(np.argmax(zs[rows_d], 1).astype(np.int32).reshape(b, d)), dev(rng.random((b, d + 1)).astype(np.float32))
    w = dev(np.full(n, 1.0 / n, np.float32))
    vals, ids, rest = torch.empty(n, k, device="cuda"), torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
    kl, g = torch.empty(n, device="cuda"), torch.empty(n, V, device="cuda")
    acc, out = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, d + 1, dtype=torch.int32, device="cuda")
    outs = (vals, ids, rest, kl, g, acc, out)

    def calls(stream):
        s = stream.cuda_stream
        top_logits_d(ctx, T.data_ptr(), rt.TYPE_F32, n, V, V, k, vals.data_ptr(), ids.data_ptr(), rest.data_ptr(), temperature=2.0, stream=s)
        distill_d(ctx, S.data_ptr(), rt.TYPE_F32, n, V, V, teacher_d(k, ids.data_ptr(), vals.data_ptr(), rest.data_ptr(), 2.0), 0, w.data_ptr(),
                  kl.data_ptr(), 0, g.data_ptr(), V, stream=s)
        verify_draft_d(ctx, T.data_ptr(), rt.TYPE_F32, V, Q.data_ptr(), V, b, d, V, x.data_ptr(), 0, u.data_ptr(), acc.data_ptr(), out.data_ptr(),
                       stream=s)

    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(rt.RtqError, match="cannot grow under capture"):
        with torch.cuda.graph(graph, stream=st):
            calls(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        calls(st)
    st.synchronize()
    v, j, r = D.top(zt.astype(np.float32), k, 2.0)
    np.testing.assert_array_equal(ids.cpu().numpy(), j)
    rk = D.distill(zs.astype(np.float32), j, v, r, 2.0)[0]
    assert np.all(np.abs(kl.cpu().numpy() - rk) <= 3 * D.SUM + HALF * rk)
    want = D.verify(zt.astype(np.float32), zs[rows_d].astype(np.float32), x.cpu().numpy(), None, u.cpu().numpy(), 1.0)
    assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(out.cpu().numpy(), want[1])
    first = [t.clone() for t in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        calls(torch.cuda.current_stream())
    big = torch.randn(40, 150000, device="cuda")
    for rep in range(4):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        st.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, first)), rep
        # eager work in between, which outgrows the workspace the graph holds
        bv, bi = torch.empty(40, 256, device="cuda"), torch.empty(40, 256, dtype=torch.int32, device="cuda")
        with torch.cuda.stream(st):
            top_logits_d(ctx, big.data_ptr(), rt.TYPE_F32, 10 * (rep + 1), 150000, 150000, 256, bv.data_ptr(), bi.data_ptr(), stream=st.cuda_stream)
        torch.cuda.synchronize()
    del graph
    ctx.close()


def test_rows_past_32_bit_offsets(ctx):
    """The last rows of 2.3 G elements (9.2 GB): element offsets past 2^31, byte offsets past 2^33."""
    n, V, ld, k = 3, 1000, (1 << 30) + (1 << 27), 5
    mem = torch.empty(2 * ld + V, device="cuda")
    z = D.logits(np.random.default_rng(12), n, V).astype(np.float32)
    view = mem.as_strided((n, V), (ld, 1))
    view.copy_(dev(z))
    vals, ids, rest = run_top(ctx, view, "f32", k, 1.0)
    v, j, r = D.top(z, k, 1.0)
    np.testing.assert_array_equal(ids, j)
    check_lse(rest, r)
    kl, w = torch.empty(n, device="cuda"), torch.ones(n, device="cuda")
    di, dv, dr = dev(ids), dev(vals), dev(rest)
    distill_d(ctx, view.data_ptr(), rt.TYPE_F32, n, V, ld, teacher_d(k, di.data_ptr(), dv.data_ptr(), dr.data_ptr()), 0, w.data_ptr(), kl.data_ptr(), 0,
              view.data_ptr(), ld, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _, _, rg, sc = D.distill(z, ids, vals, rest, 1.0, None, np.ones(n))
    # the teacher is the student: only rounding is left of the gradient
    assert np.all(np.abs(host(view) - rg) <= sc * 1e-5 + 1e-30)
    assert np.all(np.abs(kl.cpu().numpy()) <= 3 * D.SUM)
    del mem, view
    torch.cuda.empty_cache()


def test_results_do_not_depend_on_scheduling(ctx):
    """The same call twice: the same bits (gathered candidates and listed tokens come in any order inside)."""
    rng = np.random.default_rng(13)
    z = D.logits(rng, 20, 60000)
    z[::2] = np.round(z[::2])
    a, _ = D.rounded(z, "bf16")
    _, view = rows(a, "bf16")
    one, two = run_top(ctx, view, "bf16", 200, 1.0), run_top(ctx, view, "bf16", 200, 1.0)
    assert all(np.array_equal(p.view(np.int32), q.view(np.int32)) for p, q in zip(one, two))
    ids, vals, rest = teacher(rng, z, 40, 1.0)
    ids[:, 7] = ids[:, 3]
    g = [check_distill(ctx, z, ids, vals, rest, 1.0, ids[:, 3], np.ones(20), 0.5, "bf16") for _ in range(2)]
    assert torch.equal(g[0][0], g[1][0]) and torch.equal(g[0][1].view(torch.int16), g[1][1].view(torch.int16))
