"""Drafted tokens and their trees, on the host."""


def test_look_up_finds_what_followed():
    from kotensor_b200.drafts import look_up
    text = [1, 2, 3, 9, 1, 2, 3, 4, 5, 7, 2, 3]
    # after "2 3" (the longest match), the latest first, then after "3" alone what is not yet there
    assert look_up(text, depth=3) == [[4, 5, 7], [9, 1, 2]]
    assert look_up(text, most=1, depth=2) == [[4, 5]]
    assert look_up([5, 6, 7]) == [] and look_up([5]) == [] and look_up([]) == []
    assert look_up([4, 4, 4], depth=2) == [[4], [4, 4]]


def test_look_up_prefers_long_matches():
    from kotensor_b200.drafts import look_up
    text = [1, 2, 3, 10, 0, 2, 3, 20, 0, 3, 30, 0, 1, 2, 3]
    assert [c[0] for c in look_up(text, depth=1)] == [10, 20, 30]


def test_grow_merges_equal_beginnings():
    from kotensor_b200.drafts import grow
    assert grow(9, [[1, 2, 3], [1, 2, 4], [5]], 16, 100) == ([9, 1, 2, 3, 4, 5], [-1, 0, 1, 2, 2, 0])
    assert grow(9, [[1, 2, 3], [1, 2, 4], [5]], 4, 100) == ([9, 1, 2, 3], [-1, 0, 1, 2])
    assert grow(9, [[1, 100, 3], [-1], [4]], 16, 100) == ([9, 1, 4], [-1, 0, 0])
    assert grow(9, [], 1, 100) == ([9], [-1]) and grow(9, [[1]], 1, 100) == ([9], [-1])
    assert grow(9, [[1]], 0, 100) == ([], [])


def test_grown_trees_are_trees():
    import numpy as np
    from kotensor_b200.drafts import grow, look_up
    from kotensor_b200.paged import draft_tree
    rng = np.random.default_rng(0)
    for n in range(2, 60):
        text = rng.integers(0, 4, n).tolist()
        tokens, parents = grow(text[-1], look_up(text), 12, 4)
        depths, visible = draft_tree(parents)
        assert len(tokens) == len(parents) <= 12 and depths.max() <= 8
        pairs = list(zip(parents, tokens))
        assert len(set(pairs)) == len(pairs)  # no two children of a node with the same token
