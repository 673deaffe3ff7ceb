"""gqa_ref against small cases worked by hand (CPU)."""
import numpy as np

import gqa_ref as ref


def test_a_row_that_sees_one_key_has_its_value():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((3, 2, 8)), rng.standard_normal((5, 1, 8)), rng.standard_normal((5, 1, 8))
    seen = np.zeros((3, 5), bool)
    seen[0, 4] = seen[1, 2] = True
    seen[2, [0, 1]] = True
    out, mass, _ = ref.attend(q, k, v, seen)
    np.testing.assert_allclose(out[0, 0], v[4, 0])
    np.testing.assert_allclose(out[1, 1], v[2, 0])
    s = q[2, 0] @ k[:2, 0].T / np.sqrt(8)
    p = np.exp(s) / np.exp(s).sum()
    np.testing.assert_allclose(out[2, 0], p @ v[:2, 0])
    np.testing.assert_allclose(mass[2, 0], p @ np.abs(v[:2, 0]).max(axis=1))


def test_rotation_keeps_lengths_and_turns_by_the_distance():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, 1, 16)).repeat(2, axis=0)
    for neox in (True, False):
        y = ref.rotate(x, [3, 10], 16, 10000.0, neox)
        np.testing.assert_allclose((y**2).sum(-1), (x**2).sum(-1))
        z = ref.rotate(x, [103, 110], 16, 10000.0, neox)
        np.testing.assert_allclose((y[0] * y[1]).sum(), (z[0] * z[1]).sum(), rtol=1e-5)
    y = ref.rotate(x, [3, 10], 4, 10000.0, True)
    np.testing.assert_array_equal(y[..., 4:], x[..., 4:])


def test_paths_and_what_is_accepted():
    parent = [-1, 0, 0, 1, 7, 2]
    assert ref.path(parent, 3) == [0, 1, 3] and ref.path(parent, 4) == [4] and ref.path(parent, 5) == [0, 2, 5]
    tokens, chosen = [9, 5, 5, 6, 6, 7], [5, 6, 7, 1, 1, 1]
    assert ref.accept(parent, tokens, chosen) == [0, 1, 3]
    assert ref.accept(parent, tokens, [8, 6, 7, 1, 1, 1]) == [0]
    assert ref.accept([], [], []) == []


def test_edits_in_their_order():
    x = ref.edit([2.0, -2.0, 1.0, 0.5], [0, 0, 1, 9], repetition=2.0, frequency=0.25, presence=0.5,
                 biases=[(2, 5.0), (2, 1.0), (7, 3.0)], allowed=np.array([True, True, True, False]))
    np.testing.assert_allclose(x, [2 / 2 - 0.5 - 0.5, -4 - 0.25 - 0.5, 2.0, -np.inf])
