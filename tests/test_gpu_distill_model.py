"""Distillation, top logits and draft verification through the LM head and through a whole model.

With a teacher of k listed tokens, no rest and temperature 1, the divergence's gradient is the cross-entropy gradient of k
targets a row with weights w p_s (sum_s p_s (q - onehot_s) = q - p), and its value is sum_s p_s (log p_s - logp_s): so both are
held against Model::head and Model::forward_backward, which have oracles of their own.  The two run different
kernels over n and over n k rows, so they agree as the head's own calls of different row counts do (1e-5 of the largest
value for F32 weights, whose products carry 2^-22; 1e-3 through quantised ones and whole models)."""
import numpy as np
import pytest

import distill_cases as D
import oracle as O
import rust_trainer_amd as rt
from model_cases import adapters, sequence, tiny_spec
from rust_trainer_amd import gguf as G
from rust_trainer_amd.packing import pack

pytestmark = pytest.mark.gpu


def close(got, want, tol):
    got, want = np.asarray(got, np.float64).ravel(), np.asarray(want, np.float64).ravel()
    assert got.shape == want.shape
    err = np.abs(got - want).max() / max(np.abs(want).max(), 1e-30)
    assert err <= tol, err


def lists(rng, n, V, k):
    ids = np.array([rng.choice(V, k, replace=False) for _ in range(n)], np.int32)
    vals = rng.normal(0, 2, (n, k)).astype(np.float32)
    p = np.exp(vals.astype(np.float64) - D.lse(vals.astype(np.float64))[:, None])
    return ids, vals, p


@pytest.mark.parametrize("wtype,tol", [(O.F32, 1e-5), (O.Q8_0, 1e-3), (O.Q4_K, 1e-3)])
def test_head_distillation_is_cross_entropy_over_the_list(ctx, wtype, tol):
    V, d, t, n, k = 1500, 256, 20, 11, 5
    rng = np.random.default_rng(1)
    w = O.Rng(1).vec_normal(V * d, 0.05).reshape(V, d)
    f = rt.HipFrozen(wtype, O.quantize(wtype, w) if wtype != O.F32 else w.astype(np.float32), V, d, ctx=ctx)
    x, norm = rng.normal(0, 1, (t, d)).astype(np.float32), (1 + rng.normal(0, 0.1, d)).astype(np.float32)
    pos = rng.integers(0, t, n).astype(np.int32)  # some twice
    ids, vals, p = lists(rng, n, V, k)
    wts = rng.uniform(0.5, 1.5, n)
    tok = rng.integers(0, V, n).astype(np.int32)
    kl, logp, dx = rt.head_distill(f, norm, x, pos, rt.Teacher(ids, vals), tok, wts, hard=0.0)
    targets = [rt.Target(int(pos[i]), int(ids[i, s])) for i in range(n) for s in range(k)]
    lp, dx_ce, _ = rt.head(f, norm, x, targets, (wts[:, None] * p).ravel())
    close(dx, dx_ce, tol)
    close(kl, (p * (np.log(p) - lp.reshape(n, k))).sum(1), tol)
    lp, dx_ce, _ = rt.head(f, norm, x, [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)], wts)
    close(logp, lp, tol)
    kl1, lp1, dx1 = rt.head_distill(f, norm, x, pos, rt.Teacher(ids, vals), tok, wts, hard=1.0)
    close(dx1, dx_ce, tol)
    assert np.array_equal(kl1, kl) and np.array_equal(lp1, logp)
    # mixed: linear in hard
    _, _, dx2 = rt.head_distill(f, norm, x, pos, rt.Teacher(ids, vals), tok, wts, hard=0.25)
    close(dx2, 0.75 * dx + 0.25 * dx1, 1e-5)
    # losses alone, no labels
    kl3, none, nodx = rt.head_distill(f, norm, x, pos, rt.Teacher(ids, vals))
    assert np.array_equal(kl3, kl) and none.size == 0 and nodx.size == 0
    f.close()


def test_head_top_logits_give_back_the_log_probabilities(ctx):
    V, d, t, n, k = 3001, 96, 9, 7, 30
    rng = np.random.default_rng(2)
    f = rt.HipFrozen.f32(rng.normal(0, 0.1, (V, d)), V, d, ctx=ctx)
    x, norm, pos = rng.normal(0, 1, (t, d)).astype(np.float32), np.ones(d, np.float32), rng.integers(0, t, n)
    te = rt.head_top_logits(f, norm, x, pos, k)
    lp, _, _ = rt.head(f, norm, x, [rt.Target(int(pos[i]), int(te.ids[i, s])) for i in range(n) for s in range(k)])
    z = np.concatenate([te.vals.astype(np.float64), te.rest[:, None].astype(np.float64)], 1)
    close(te.vals - D.lse(z)[:, None], lp, 1e-5)
    assert np.all(np.diff(te.vals, axis=1) <= 0)
    # a student that is the teacher: no divergence, no gradient but rounding
    kl, _, dx = rt.head_distill(f, norm, x, pos, te, weights=np.ones(n))
    assert np.abs(kl).max() <= 1e-5 and np.abs(dx).max() <= 1e-4
    # refusals, and no rows
    for bad in (lambda: rt.head_top_logits(f, norm, x, [t], k), lambda: rt.head_top_logits(f, norm, x, [-1], k), lambda: rt.head_top_logits(f, norm, x, pos, 257),
                lambda: rt.head_top_logits(f, norm, x, pos, k, temperature=0.0), lambda: rt.head_distill(f, norm, x, pos, te, hard=0.5),
                lambda: rt.head_distill(f, norm, x, pos, te, labels=np.full(n, V), weights=np.ones(n)),
                lambda: rt.head_distill(f, norm, x, pos, rt.Teacher(np.full((n, 1), V), np.zeros((n, 1))))):
        with pytest.raises(rt.RtqError):
            bad()
    kl, _, dx = rt.head_distill(f, norm, x, [], rt.Teacher(np.zeros((0, 2)), np.zeros((0, 2))), weights=[])
    assert kl.size == 0 and dx.size == t * d and not dx.any()
    f.close()


def test_head_device_calls_mark_positions_out_of_range(ctx):
    import torch

    V, d, t, k = 700, 64, 5, 4
    rng = np.random.default_rng(3)
    f = rt.HipFrozen.f32(rng.normal(0, 0.1, (V, d)), V, d, ctx=ctx)
    x, norm = rng.normal(0, 1, (t, d)).astype(np.float32), np.ones(d, np.float32)
    pos, tok = np.array([1, t, 3, -1], np.int32), np.array([5, 6, -1, 7], np.int32)
    ids, vals, _ = lists(rng, 4, V, k)
    D_ = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    dn, dxs, dp, dt, di, dv, dw = D_(norm), D_(x), D_(pos), D_(tok), D_(ids), D_(vals), torch.ones(4, device="cuda")
    kl, lp, dx = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), torch.full((t, d), 7.0, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    te = rt._ffi.RtqTeacher(k, di.data_ptr(), dv.data_ptr(), None, 1.0)
    import ctypes

    rt._ffi.check(rt.lib().rtq_lm_distill_d(ctx.handle, f.handle, dn.data_ptr(), 1e-6, 0.0, dxs.data_ptr(), t, dp.data_ptr(), dt.data_ptr(),
                                            dw.data_ptr(), 4, ctypes.byref(te), 0.5, kl.data_ptr(), lp.data_ptr(), dx.data_ptr(), st or None), "d")
    tv, ti, tr = torch.zeros(4, k, device="cuda"), torch.zeros(4, k, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    rt._ffi.check(rt.lib().rtq_lm_top_logits_d(ctx.handle, f.handle, dn.data_ptr(), 1e-6, 0.0, dxs.data_ptr(), t, dp.data_ptr(), 4, k, 1.0,
                                               tv.data_ptr(), ti.data_ptr(), tr.data_ptr(), st or None), "t")
    torch.cuda.synchronize()
    kl, lp, dx = kl.cpu().numpy(), lp.cpu().numpy(), dx.cpu().numpy()
    assert np.isnan(kl[[1, 3]]).all() and np.isnan(lp[[1, 2, 3]]).all() and np.isfinite(kl[[0, 2]]).all() and np.isfinite(lp[0])
    assert not dx[[0, 2, 4]].any() and dx[1].any() and dx[3].any() and np.isfinite(dx).all()
    assert torch.isnan(tv[[1, 3]]).all() and (ti[[1, 3]] == -1).all() and torch.isnan(tr[[1, 3]]).all()
    good = rt.head_top_logits(f, norm, x, pos[[0, 2]], k)
    assert np.array_equal(ti.cpu().numpy()[[0, 2]], good.ids)
    f.close()


def load(ctx, wtype=O.F32, n_layer=2, seed=1, **kw):
    g = G.GgufFile.from_bytes(tiny_spec(wtype, n_layer=n_layer, **kw).build())
    m = rt.GpuModel.from_gguf(g, ctx=ctx)
    m.attach_lora(4, 8.0, seed=seed)
    lora = adapters(g, 4, 8.0, seed=10 + seed, b_std=0.05)
    for i in range(m.lora_count()):
        inf = m.lora_info(i)
        m.set_lora(i, *lora[(inf["layer"], O.LINEARS[inf["which"]])])
    return m


def grads(m):
    return np.concatenate([np.concatenate([v.ravel() for v in m.lora(i)[2:]]) for i in range(m.lora_count())])


@pytest.mark.parametrize("wtype", [O.F32, O.Q8_0])
def test_model_distillation_is_cross_entropy_over_the_list(ctx, wtype):
    m = load(ctx, wtype)
    V, n, k = m.config["n_vocab"], 12, 3
    toks, pos, tok = sequence(V, 40, n)
    rng = np.random.default_rng(4)
    ids, vals, p = lists(rng, n, V, k)
    te, wts = rt.Teacher(ids, vals), rng.uniform(0.5, 1.5, n)
    m.zero_grad()
    kl, logp = m.forward_backward_distill(toks, pos, te, tok, wts, hard=0.0)
    g = grads(m)
    m.zero_grad()
    lp, _ = m.forward_backward(toks, [rt.Target(int(pos[i]), int(ids[i, s])) for i in range(n) for s in range(k)], (wts[:, None] * p).ravel())
    close(g, grads(m), 1e-3)
    close(kl, (p * (np.log(p) - lp.reshape(n, k))).sum(1), 1e-3)
    m.zero_grad()
    lp, _ = m.forward_backward(toks, [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)], wts)
    ce = grads(m)
    close(logp, lp, 1e-3)
    # repeated steps run as one graph, with the same bits; gradients accumulate
    before = m.graph_replays
    outs = []
    for _ in range(5):
        m.zero_grad()
        outs.append((*m.forward_backward_distill(toks, pos, te, tok, wts, hard=1.0), grads(m)))
    assert m.graph_replays >= before + 3
    assert all(np.array_equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))
    close(outs[0][2], ce, 1e-3)
    # new inputs of the same sizes replay it too: another teacher, another temperature is another step
    te2 = rt.Teacher(ids[::-1], vals)
    m.zero_grad()
    kl2, _ = m.forward_backward_distill(toks, pos, te2, tok, wts, hard=1.0)
    assert not np.array_equal(kl2, kl)
    kl3, _ = m.forward_backward_distill(toks, pos, rt.Teacher(ids, vals, temperature=2.0), tok, wts, hard=1.0)
    assert not np.array_equal(kl3, kl)
    kl4, none = m.forward_backward_distill(toks, pos, te)
    close(kl4, kl, 1e-6)
    assert none.size == 0
    # an ordinary step after it is as before
    m.zero_grad()
    m.forward_backward(toks, [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)], wts)
    assert np.array_equal(grads(m), ce)
    m.close()


def test_teacher_student_and_packed_batches(ctx):
    """A teacher's pass over a packed batch gives what it gives example by example, and the student's
    gradient on it is the loss's slope."""
    te_m, st_m = load(ctx, seed=1), load(ctx, seed=2)
    V, k = te_m.config["n_vocab"], 16
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, V, 10).tolist()
    seqs = [prompt + rng.integers(0, V, 6).tolist(), prompt + rng.integers(0, V, 9).tolist()]
    pk = pack(seqs)
    pos = [[9, 11, 14], [10, 17]]
    where = [pk.index(i, q) for i in (0, 1) for q in pos[i]]
    both = te_m.top_logits(None, where, k, 2.0, packed=pk)
    one = [te_m.top_logits(seqs[i], pos[i], k, 2.0) for i in (0, 1)]
    close(both.vals, np.concatenate([o.vals for o in one]), 1e-4)
    close(both.rest, np.concatenate([o.rest for o in one]), 1e-4)
    w = np.full(5, 0.2)
    st_m.zero_grad()
    kl, _ = st_m.forward_backward_distill(None, where, both, weights=w, packed=pk)
    kls = np.concatenate([st_m.forward_backward_distill(seqs[i], pos[i], one[i])[0] for i in (0, 1)])
    close(kl, kls, 1e-3)
    # the loss along the gradient against differences: dL = -step |g|^2 to first order
    gs = [st_m.lora(i)[2:] for i in range(st_m.lora_count())]
    g2 = float(sum((a.astype(np.float64) ** 2).sum() + (b.astype(np.float64) ** 2).sum() for a, b in gs))
    base = [st_m.lora(i)[:2] for i in range(st_m.lora_count())]

    def loss(step):
        for i, ((a, b), (ga, gb)) in enumerate(zip(base, gs)):
            st_m.set_lora(i, a - step * ga, b - step * gb)
        return 4.0 * float((st_m.forward_backward_distill(None, where, both, packed=pk)[0].astype(np.float64) * w).sum())

    h = 2e-2 * loss(0.0) / g2
    assert abs((loss(-h) - loss(h)) / (2 * h) / g2 - 1) <= 0.02
    te_m.close()
    st_m.close()


def test_model_verifies_drafts(ctx):
    target, draft = load(ctx, seed=1), load(ctx, seed=2)
    V, d = target.config["n_vocab"], 4
    toks = sequence(V, 20, 4)[0]
    every = lambda m, s: m.score(s, [rt.Target(int(p), v) for p in range(len(s) - d - 1, len(s)) for v in range(V)])[0].reshape(d + 1, V)  # noqa: E731
    rng = np.random.default_rng(6)
    for rep in range(6):
        s = toks.copy()
        if rep % 2:  # a draft that is likely accepted at first
            for j in range(2):
                s[len(s) - d + j] = draft.top_logits(s, [len(s) - d - 1 + j], 1).ids[0, 0]
        u = rng.random(d + 1).astype(np.float32) * (0.2 if rep % 2 else 1.0)
        zt, zq = every(target, s), every(draft, s)[:d]
        for who, rows in ((draft, zq), (None, None)):
            acc, out = target.verify_draft(s, d, u, draft=who)
            want = D.verify(zt, rows, s[None, -d:], None, u[None], 1.0)
            assert acc == want[0][0] and np.array_equal(out, want[1][0])
    # greedy: a draft of the target's own choices is accepted whole
    s = list(toks)
    for _ in range(d):
        s.append(int(target.top_logits(s, [len(s) - 1], 1).ids[0, 0]))
    acc, out = target.verify_draft(s, d, temperature=0.0)
    assert acc == d and np.array_equal(out[:d], s[-d:]) and out[d] == target.top_logits(s, [len(s) - 1], 1).ids[0, 0]
    acc, out = target.verify_draft(s, 0, np.zeros(1, np.float32))
    assert acc == 0 and out.shape == (1,) and out[0] >= 0
    other = load(ctx, n_vocab=300)
    for bad in (lambda: target.verify_draft(s, len(s), np.zeros(len(s) + 1)), lambda: target.verify_draft(s, d), lambda: target.verify_draft(s, d, np.ones(d + 1)),
                lambda: target.verify_draft(s, d, np.zeros(d + 1), draft=other), lambda: target.verify_draft(s, d, np.zeros(d + 1), temperature=-1.0),
                lambda: target.top_logits(s, [len(s)], 2), lambda: target.top_logits(s, [0], V + 1), lambda: target.top_logits(s, [0], 2, temperature=0.0),
                lambda: target.forward_backward_distill(s, [0], rt.Teacher([[V]], [[0.0]])),
                lambda: target.forward_backward_distill(s, [0], rt.Teacher([[1]], [[0.0]]), hard=0.5)):
        with pytest.raises(rt.RtqError):
            bad()
    for m in (target, draft, other):
        m.close()
