"""The oracle of the block-pool operators against hand-worked tables and closed forms."""
from __future__ import annotations

import numpy as np

from oracle import attention as A
from oracle import paged


def test_update_by_hand():
    # request 0 gives a block back, 1 takes two, 2 wants more than is left, 3 takes none
    table = [[5, 6, -1], [7, -1, -1], [-1, -1, -1], [8, -1, -1]]
    got = paged.update_block_tables(table, [2, 1, 0, 1], [3, 4, 0, 0, 0], 2, [4, 12, 12, 2], [3, 4, 0, 2], block_size=4,
                                    max_rows=22)
    assert got[0] == [[5, -1, -1], [7, 6, 4], [-1, -1, -1], [8, -1, -1]]
    assert got[1] == [1, 3, 0, 1] and got[2][:1] == [3] and got[3] == 1
    assert got[4] == [0, 1, 9, 21, 21]
    assert got[5] == [23, 24, 25, 26, 27, 16, 17, 18, 19] + [-1] * 13
    assert got[6] == [True, True, False, True]


def test_ancestors_and_words():
    assert paged.ancestors([-1, 0, 0, 2, 9]) == [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {4}]
    w = paged.words([{0, 63}, {64, 65}], 2)
    assert w.tolist() == [[1 - 2 ** 63, 0], [0, 3]]


def test_attend_a_chain_is_dense_causal_attention():
    rng = np.random.default_rng(0)
    H, Hk, D, T, n = 4, 2, 8, 11, 3
    k, v = rng.standard_normal((2, 1, Hk, T, D))
    q = rng.standard_normal((n, H, D))
    out, lse, mean, dots = paged.attend(q, k, v, [[0]], [T - n], [0, n], paged.ancestors([-1, 0, 1]), D ** -0.5)
    for i in range(n):
        keep = T - n + i + 1
        ref, ref_lse = A.attention_f64(q[i][None], k[:, :, :keep], v[:, :, :keep], scale=D ** -0.5)
        assert np.allclose(out[i], ref[0], atol=1e-12) and np.allclose(lse[i], ref_lse[0], atol=1e-12)
    assert (mean >= np.abs(out) - 1e-12).all()


def test_attend_holes_and_nothing():
    k = np.ones((2, 1, 2, 4))
    v = np.arange(16.0).reshape(2, 1, 2, 4)
    out, lse, _, _ = paged.attend(np.ones((2, 1, 4)), k, v, [[-1, 1], [0, 9]], [3, 0], [0, 1, 2], [set(), set()], 1.0)
    assert np.array_equal(out[0, 0], v[1, 0, 0]) and lse[0, 0] == 4.0
    assert not out[1].any() and lse[1, 0] == -np.inf
