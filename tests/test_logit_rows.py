"""Rows of vocabulary logits without a GPU: the tests' plain forms against values worked out by hand, and what is refused."""
import numpy as np
import pytest

import distill_cases as D
import rust_trainer_amd as rt


def test_plain_divergence_has_one_bucket_a_token():
    """Two slots of 1/2 on a token that the student gives 0.9: log(1 / 0.9), not that less log 2; and any list with
    repeats as the list that they are merged into."""
    z = np.log([[0.9, 0.1]])
    kl = D.distill(z, np.array([[0, 0]]), np.ones((1, 2)), None, 1.0)[0]
    assert abs(kl[0] - np.log(1 / 0.9)) < 1e-15
    rng = np.random.default_rng(0)
    z, ids, vals = rng.normal(0, 2, (1, 50)), np.array([[3, 9, 3, -1, 9, 3, 20]]), rng.normal(0, 2, (1, 7))
    t = vals[0] / 1.5
    merged = 1.5 * np.array([[D.lse(t[[0, 2, 5]]), D.lse(t[[1, 4]]), t[6]]])
    for rest in (None, np.array([0.4])):
        many, one = D.distill(z, ids, vals, rest, 1.5), D.distill(z, np.array([[3, 9, 20]]), merged, rest, 1.5)
        assert one[0][0] > 0 and abs(many[0][0] - one[0][0]) < 1e-14 and np.abs(many[2] - one[2]).max() < 1e-14


@pytest.mark.parametrize("dtype,type", [(np.float16, rt.TYPE_BF16), (np.int32, rt.TYPE_F32), (np.uint32, rt.TYPE_F32), (">f4", rt.TYPE_F32),
                                        (">f2", rt.TYPE_F16), (">u2", rt.TYPE_BF16), (np.float32, rt.TYPE_F16)])
def test_logits_of_another_type_than_named_are_refused(dtype, type):
    """An array of another element type would be read as bits of the named one."""
    z = np.zeros((4, 10), dtype)
    none = object()  # a context that is not looked at
    t = rt.Teacher(np.zeros((4, 2)), np.zeros((4, 2)))
    for call in (lambda: rt.top_logits(z, 2, type=type, ctx=none), lambda: rt.distill(z, t, type=type, ctx=none),
                 lambda: rt.verify_draft(z, np.zeros((2, 1)), np.zeros((2, 2)), type=type, ctx=none)):
        with pytest.raises(AssertionError):
            call()


def test_bfloat16_rows_are_their_bits():
    """uint16 (or int16) arrays hold bfloat16 or float16 bits where the type says so; they get as far as the context."""
    for dtype, type in ((np.uint16, rt.TYPE_BF16), (np.int16, rt.TYPE_BF16), (np.uint16, rt.TYPE_F16), (np.float16, rt.TYPE_F16), (np.float16, None)):
        with pytest.raises(AttributeError):
            rt.top_logits(np.zeros((4, 10), dtype), 2, type=type, ctx=object())
