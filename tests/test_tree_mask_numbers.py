"""Masks of drafted tokens: parents that are no whole numbers of 32 bits are refused, not cut down to some that are."""
import numpy as np
import pytest

from logismos_amd import kernels


@pytest.mark.parametrize("parents", [np.array([-1, 1 << 32]), np.array([-1, -1 + (1 << 32)]), np.array([-1, 0.5]),
                                     np.array([-1.0, np.nan]), np.array([[-1, 0]])])
def test_parents_that_are_no_tokens(parents):
    with pytest.raises(kernels.UnsupportedShape), np.errstate(invalid="ignore"):
        kernels.tree_mask(parents)


@pytest.mark.parametrize("kind", [np.int8, np.int64, np.float64, list])
def test_parents_of_any_kind(kind):
    parents = [-1, 0, 0, 2, -1]
    given = parents if kind is list else np.array(parents, kind)
    assert kernels.tree_mask(given).ravel().tolist() == [1, 3, 5, 13, 16]
