"""Rows of vocabulary logits without a GPU: the tests' plain forms against values worked out by hand."""
import numpy as np

import distill_cases as D


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
