"""The bounds of the batch attention tell two terms of 11 bits from one."""
import numpy as np
import pytest

import kv4_cases as kc
from kv4_close import attend_in_terms, close, rounded


def random_rows(dim, n, seed):
    """keys and values like those of the cases' caches"""
    rng = np.random.default_rng(seed)
    pair = lambda: (np.repeat(x, 64, -1) for x in ((-2 + 0.5 * rng.standard_normal((n, dim // 64))).astype(np.float16).astype(np.float64),  # noqa: E731
                                                   (0.2 + 0.2 * rng.random((n, dim // 64))).astype(np.float16).astype(np.float64)))
    return [(*pair(), rng.integers(0, 16, (n, dim))) for _ in range(2)]


SIZES = [(2, 1.0), (30, 3.0), (1000, 3.0), (1000, 8.0)]  # rows, size of the queries: as in the GPU's test


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bounds_tell_two_terms_from_one(dim):
    rng, missed = np.random.default_rng(4), {(1, 2): 0, (2, 1): 0}
    for length, size in SIZES:
        key, value = random_rows(dim, length, dim + length)
        for _ in range(6):
            q = size * rng.standard_normal(dim)
            want, tol = close(q, key, value, length - 1)
            tol = rounded(want, tol)
            off = lambda *way: (np.abs(attend_in_terms(q, key, value, length - 1, *way).astype(np.float16) - want) > tol).any()  # noqa: B023,E731
            assert not off(2, 2)
            for way in missed:
                missed[way] += off(*way)
    assert min(missed.values()) > 0, missed


def test_cases_agree():
    """the loose bounds and the close ones are about the same numbers"""
    key, value = random_rows(64, 100, 1)
    q = np.random.default_rng(5).standard_normal(64)
    a, b = kc.attend(q, key, value, 99), close(q, key, value, 99)
    assert np.array_equal(a[0], b[0]) and (b[1] < a[1]).all()
