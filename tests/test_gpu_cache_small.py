"""The cache operators at capacities and prefixes of fewer than eight keys: rows
shorter than one 16-byte piece.  References and bounds are test_gpu_cache's."""
import pytest

from tests.test_gpu_cache import TYPES, append_check, check, evict_check, lh  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("S", [1, 2, 3, 5, 7])
def test_decode(lh, S, e):  # noqa: F811
    for B, G, H, D, P in ((1, 1, 1, 8, 0), (3, 2, 5, 64, 0), (2, 1, 33, 136, 1), (2, 1, 71, 24, 3),
                          (70, 1, 2, 8, 7), (3, 2, 40, 256, S)):
        for weights in (False, True):
            check(lh, "small", B, G, H, D, P, S, [(S - b) % (S + 1) for b in range(B)], TYPES[e],
                  weights)


@pytest.mark.parametrize("S", [1, 2, 3, 5, 7])
def test_evict_and_append(lh, S):  # noqa: F811
    for e in TYPES.values():
        for D in (8, 64, 136):
            for keep in {1, (S + 1) // 2, S}:
                evict_check(lh, 3, 2, D, S, S, [S, S - 1, 0], keep, min(1, keep - 1), 0, e=e)
            for T in (1, 3, 4, 9):
                for seed in (0, 1):
                    append_check(lh, 3, 2, D, S, T, [S, S - 1, 0], [T, 1, T - 1], e=e, seed=seed)
