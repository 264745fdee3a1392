"""The 64-bit oracle of grouped_topk where the largest logit is not among the chosen (no GPU)."""
import numpy as np

from oracle import dense


def test_weights_of_chosen_far_below_the_largest_logit():
    """The bias keeps the expert with the +inf logit out; the others keep their ratio."""
    for top in (np.inf, 1e30, 800.0):
        ids, w = dense.grouped_topk([[top, 0.0, -1.0, -2.0]], 2, True, bias=[-9.0, 0.0, 0.0, -1.0])
        e = np.exp(-1.0)
        assert ids.tolist() == [[1, 2]]
        np.testing.assert_allclose(w, [[1 / (1 + e), e / (1 + e)]], rtol=1e-12)
