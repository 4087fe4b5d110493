"""Rows of vocabulary logits without a GPU: every refusal of the entry points (their arguments are checked
before the context), and the tests' plain forms against differences."""
import ctypes

import numpy as np
import pytest

import distill_cases as D
import rust_trainer_amd as rt
from rust_trainer_amd import _ffi

INVALID, UNSUPPORTED = 1, 2
BUF = np.zeros(4096, np.float32)
P = BUF.ctypes.data
P += -P % 16


def refused(status, text):
    assert status in (INVALID, UNSUPPORTED)
    assert text in _ffi.lib().rtq_last_error().decode()
    return status


def top(**kw):
    a = dict(z=P, ty=0, n=2, V=100, ld=100, k=4, temp=1.0, vals=P, ids=P, rest=P) | kw
    args = (None, a["z"], a["ty"], a["n"], a["V"], a["ld"], a["k"], a["temp"], a["vals"], a["ids"], a["rest"])
    s = _ffi.lib().rtq_top_logits(*args)
    assert s == _ffi.lib().rtq_top_logits_d(*args, None)
    return s


@pytest.mark.parametrize("kw,text", [
    ({"ty": 2}, "type 2"), ({"ty": 264}, "type 264"), ({"n": -1}, "row count"), ({"n": 65536}, "row count"), ({"V": 0}, "vocabulary"),
    ({"V": (1 << 20) + 1, "ld": 1 << 21}, "vocabulary"), ({"ld": 99}, "stride"), ({"z": None}, "null logits"), ({"z": P + 2}, "aligned"),
    ({"ty": 1, "z": P + 1}, "aligned"), ({"k": 0}, "k = 0"), ({"k": 101}, "k = 101"), ({"k": 257, "V": 1000, "ld": 1000}, "k = 257"),
    ({"temp": 0.0}, "temperature"), ({"temp": -1.0}, "temperature"), ({"temp": float("nan")}, "temperature"),
    ({"temp": float("inf")}, "temperature"), ({"vals": None}, "null vals"), ({"ids": None}, "null vals/ids"), ({}, "null context")])
def test_top_logits_refuses(kw, text):
    s = refused(top(**kw), text)
    assert (s == UNSUPPORTED) == ("type" in text)


def distill(**kw):
    a = dict(z=P, ty=0, n=2, V=100, ld=100, k=4, ids=P, vals=P, rest=None, temp=1.0, teacher=True, tok=P, w=P, hard=0.5, kl=P, logp=P,
             dz=P + 4096, ldd=100) | kw
    t = _ffi.RtqTeacher(a["k"], a["ids"], a["vals"], a["rest"], a["temp"])
    args = (None, a["z"], a["ty"], a["n"], a["V"], a["ld"], ctypes.byref(t) if a["teacher"] else None, a["tok"], a["w"], a["hard"], a["kl"],
            a["logp"], a["dz"], a["ldd"])
    s = _ffi.lib().rtq_distill(*args)
    assert s == _ffi.lib().rtq_distill_d(*args, None)
    return s


@pytest.mark.parametrize("kw,text", [
    ({"ty": 30, "z": P + 1}, "aligned"), ({"teacher": False}, "null teacher"), ({"k": 0}, "slots"), ({"k": 257}, "slots"),
    ({"temp": 0.0}, "temperature"), ({"hard": -0.1}, "hard"), ({"hard": 1.1}, "hard"), ({"hard": float("nan")}, "hard"),
    ({"tok": None}, "go together"), ({"logp": None}, "go together"), ({"tok": None, "logp": None}, "without labels"),
    ({"ids": None}, "null ids"), ({"vals": None}, "null ids"), ({"kl": None}, "kl"), ({"dz": None}, "without dlogits"),
    ({"ldd": 99}, "gradient row stride"), ({"dz": P + 4098}, "dlogits not aligned"), ({"dz": P + 4}, "overlaps"),
    ({"dz": P, "ldd": 101}, "overlaps"), ({"dz": P + 796}, "overlaps"), ({"n": 65536}, "row count"), ({"ld": 10}, "stride"), ({}, "null context"),
    ({"dz": P}, "null context"), ({"w": None, "dz": None}, "null context")])
def test_distill_refuses(kw, text):
    refused(distill(**kw), text)


def verify(**kw):
    a = dict(z=P, ty=0, ld=100, q=P, ldq=100, b=2, d=3, V=100, x=P, lens=None, u=P, temp=1.0, acc=P, out=P) | kw
    args = (None, a["z"], a["ty"], a["ld"], a["q"], a["ldq"], a["b"], a["d"], a["V"], a["x"], a["lens"], a["u"], a["temp"], a["acc"], a["out"])
    s = _ffi.lib().rtq_verify_draft(*args)
    assert s == _ffi.lib().rtq_verify_draft_d(*args, None)
    return s


@pytest.mark.parametrize("kw,text", [
    ({"b": -1}, "sequences"), ({"b": 65536}, "sequences"), ({"d": -1}, "sequences"), ({"b": 60000, "d": 1000}, "sequences"), ({"z": None}, "null logits"),
    ({"ty": 7}, "type"), ({"ld": 99}, "stride"), ({"ldq": 99}, "draft row stride"), ({"q": P + 2}, "draft logits not aligned"),
    ({"x": None}, "null drafted"), ({"acc": None}, "accepted"), ({"out": None}, "tokens"), ({"u": None}, "null uniforms"),
    ({"temp": -1.0}, "temperature"), ({"temp": float("nan")}, "temperature"), ({"V": 0}, "vocabulary"), ({}, "null context"),
    ({"u": None, "temp": 0.0}, "null context"), ({"d": 0, "x": None}, "null context"), ({"q": None, "ldq": 0}, "null context")])
def test_verify_draft_refuses(kw, text):
    refused(verify(**kw), text)


def test_python_shapes_are_checked_before_any_device_call():
    z = np.zeros((4, 10), np.float32)
    t = rt.Teacher(np.zeros((4, 2), np.int32), np.zeros((4, 2), np.float32))
    none = object()  # a context that is not looked at
    for call in (lambda: rt.top_logits(z[0], 2, ctx=none), lambda: rt.top_logits(z.astype(np.float64), 2, ctx=none),
                 lambda: rt.top_logits(z, 2, type=rt.TYPE_BF16, ctx=none),
                 lambda: rt.distill(z, rt.Teacher(t.ids[:3], t.vals[:3]), ctx=none),
                 lambda: rt.distill(z, rt.Teacher(t.ids, t.vals[:, :1]), ctx=none),
                 lambda: rt.distill(z, rt.Teacher(t.ids, t.vals, np.zeros(3)), ctx=none),
                 lambda: rt.distill(z, t, labels=[1, 2], ctx=none), lambda: rt.distill(z, t, weights=[1.0], ctx=none),
                 lambda: rt.verify_draft(z, np.zeros((2, 2)), ctx=none), lambda: rt.verify_draft(z, np.zeros((2, 1)), np.zeros((2, 1)), ctx=none),
                 lambda: rt.verify_draft(z, np.zeros((2, 1)), np.zeros((2, 2)), draft=z, ctx=none),
                 lambda: rt.verify_draft(z, np.zeros((2, 1)), np.zeros((2, 2)), lens=[1], ctx=none)):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.parametrize("rest", [False, True])
def test_plain_gradient_matches_differences(rest):
    """The formula's gradient against central differences of the loss (step 1e-5: the truncation is below 1e-9)."""
    rng = np.random.default_rng(3)
    n, V, k, temp, hard = 3, 11, 4, 1.5, 0.3
    z = rng.normal(0, 1, (n, V))
    ids = np.array([rng.permutation(V)[:k] for _ in range(n)])
    ids[0, 1] = ids[0, 0]  # listed twice
    ids[1, 2] = -1
    vals, r = rng.normal(0, 1, (n, k)), rng.normal(0, 1, n) if rest else None
    tok, w = np.array([2, 5, -1]), np.array([0.5, 1.0, 2.0])

    def loss(zz):
        kl, lp, _, _ = D.distill(zz, ids, vals, r, temp, tok, w, hard)
        return float(np.sum(w * (1 - hard) * temp ** 2 * kl) - np.nansum(w * hard * lp))

    g = D.distill(z, ids, vals, r, temp, tok, w, hard)[2]
    for i in range(n):
        for j in range(V):
            d = np.zeros_like(z)
            d[i, j] = 1e-5
            assert abs((loss(z + d) - loss(z - d)) / 2e-5 - g[i, j]) < 1e-8


def test_plain_verify_keeps_the_targets_distribution():
    """Over many uniform numbers the first token that comes out is distributed as the target's softmax (5 sigma)."""
    rng = np.random.default_rng(5)
    V, n = 5, 40000
    z, q = rng.normal(0, 1, (2, V)), rng.normal(0, 1, (1, V))
    pq = np.exp(q[0] - D.lse(q[0]))
    x = rng.choice(V, n, p=pq).astype(np.int32)
    acc, out = D.verify(np.tile(z, (n, 1)), np.tile(q, (n, 1)), x[:, None], None, rng.random((n, 2)), 1.0)
    p = np.exp(z[0] - D.lse(z[0]))
    got = np.bincount(out[:, 0], minlength=V) / n
    assert np.all(np.abs(got - p) < 5 * np.sqrt(p * (1 - p) / n))
