"""The oracle of the drafted-token step against other statements of it."""

import numpy as np

from oracle import attention as oa
from oracle import drafts


def _tree(rng, n):
    return [-1] + [int(rng.integers(-1 if rng.random() < 0.2 else 0, i)) for i in range(1, n)]


def test_ancestors_are_reachability():
    rng = np.random.default_rng(1)
    for n in (1, 2, 7, 40, 70):
        parents = _tree(rng, n)
        step = np.zeros((n, n), dtype=int)
        for i, p in enumerate(parents):
            if p >= 0:
                step[i, p] = 1
        reach, power = np.eye(n, dtype=int), np.eye(n, dtype=int)
        for limit in range(n):
            np.testing.assert_array_equal(drafts.ancestors(parents, limit), reach > 0)
            power = power @ step
            reach = reach + power
        np.testing.assert_array_equal(drafts.ancestors(parents), reach > 0)
        np.testing.assert_array_equal(drafts.depths(parents), drafts.ancestors(parents).sum(1) - 1)


def test_words_hold_the_bits():
    rng = np.random.default_rng(2)
    seen = rng.random((5, 100)) < 0.5
    words = drafts.pack_bits(seen, 2)
    for i in range(5):
        for a in range(100):
            assert (int(words[i, a // 64]) >> (a % 64)) & 1 == seen[i, a]
    np.testing.assert_array_equal(drafts.pack_bits(seen, 1), words[:, :1])


def test_a_parent_that_is_no_earlier_node_is_none():
    np.testing.assert_array_equal(drafts.depths([0, 5, 1, -7, 3]), [0, 0, 1, 0, 1])
    assert drafts.ancestors([0, 5, 1, -7, 3])[2].tolist() == [False, True, True, False, False]


def test_chain_maps_are_the_decode_step():
    slots, positions = np.arange(10, 30), np.arange(20) * 2
    got = drafts.step_maps([(slots, positions)], [3], page_size=4, pages=6, window=5, capacity=5)
    assert got["slot_map"].tolist() == [27, 28, 29, -1, -1]
    # a drafted token follows its parent by one position
    assert got["positions"].tolist() == [34, 35, 36, 0, 0]
    assert got["block_tables"].tolist() == [[2, 3, 4, 5, 6, -1]]
    assert got["tree_mask"][:, 0].tolist() == [1, 3, 7, 0, 0]
    # keys at 28, 30, 32 (34 - 5 = 29: from 30 on)
    assert got["window_starts"].tolist() == [15, 15, 16, 0, 0]


def test_rotation_is_the_complex_product():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 3, 10))
    angle = rng.random((4, 3)) * 6
    rows = np.concatenate((np.cos(angle), np.sin(angle)), 1)
    for neox in (True, False):
        y, _ = drafts.qk_norm_rope(x, None, 0.0, rows, 6, neox)
        plain, _ = drafts.qk_norm_rope(x, None, 0.0, np.tile([1.0] * 3 + [0.0] * 3, (4, 1)), 6, neox)
        np.testing.assert_allclose((plain ** 2).mean(-1), 1.0)
        one = slice(0, 3) if neox else slice(0, 6, 2)
        two = slice(3, 6) if neox else slice(1, 6, 2)
        z = (plain[..., one] + 1j * plain[..., two]) * np.exp(1j * angle)[:, None]
        np.testing.assert_allclose(y[..., one] + 1j * y[..., two], z)
        np.testing.assert_array_equal(y[..., 6:], plain[..., 6:])


def test_causal_tree_is_context_attention():
    rng = np.random.default_rng(4)
    old, new, hq, hk, d = 37, 6, 4, 2, 8
    k, v = rng.standard_normal((50, hk, d)), rng.standard_normal((50, hk, d))
    q = rng.standard_normal((new, hq, d))
    slots = rng.permutation(50)[: old + new]
    seen = np.ones((new, old + new), dtype=bool)
    seen[:, old:] = np.tril(np.ones((new, new), dtype=bool))
    for sinks in (None, rng.standard_normal(hq)):
        got, size, _ = drafts.tree_attention(q, k, v, [(0, slots, seen)], 0.4, sinks)
        want = oa.context_attention(q, k[slots[old:]], v[slots[old:]], k, v, np.array([0, new]), np.array([0, old]),
                                    slots[:old], 0.4, sinks=sinks)
        np.testing.assert_allclose(got, want, rtol=1e-5, atol=1e-6)
        assert (size >= np.abs(got) - 1e-12).all()


def test_rows_without_keys_are_zero():
    q, k = np.ones((2, 1, 8)), np.ones((4, 1, 8))
    seen = np.array([[False, False], [True, False]])
    got, _, _ = drafts.tree_attention(q, k, 3 * k, [(0, [9, 1], seen)], 1.0)
    assert (got == 0).all()  # nothing seen; the only seen key lies outside the pool


def test_a_chunk_has_its_ranks_positions():
    """New ranks among kept tokens whose positions have gaps."""
    slots, positions = np.arange(10, 16), np.array([0, 2, 7, 8, 30, 31])
    got = drafts.step_maps([(slots, positions)], [4], window=6, chunk=True)
    assert got["positions"].tolist() == [7, 8, 30, 31]
    assert got["window_starts"].tolist() == [1, 1, 2, 2]  # of the ranks at 0 and 2
    assert got["tree_mask"][:, 0].tolist() == [1, 3, 7, 15]
    assert got["window_mask"][:, 0].tolist() == [1, 3, 4, 12]
    tree = drafts.step_maps([(slots, positions)], [4], window=1, parents=[[-1, 0, 0, 2]])
    assert tree["positions"].tolist() == [7, 8, 8, 9]
    assert tree["window_mask"][:, 0].tolist() == [1, 3, 5, 12]
