"""cache_decode at head dims between the built ones and past 128 at every tile:
rows of own keys on tiles of 32, 64 and 128, prefix tiles of the same, whole
16-byte K rows and rows off their boundaries.  References and bounds are
test_gpu_cache's."""
import pytest

from tests.test_gpu_cache import TYPES, check, lh  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = {
    # own tiles of 128, 64 and 32 rows past D 128, even and odd capacities
    "own128": (2, 1, 71, 256, 0, 520, [520, 77]),
    "own128-odd": (2, 1, 71, 256, 0, 521, [521, 77]),
    "own128-two": (1, 2, 129, 256, 0, 333, [333]),
    "own64": (3, 1, 40, 256, 0, 264, [264, 0, 100]),
    "own64-odd": (3, 1, 40, 256, 0, 267, [267, 0, 100]),
    "own32-odd": (2, 2, 5, 256, 0, 267, [267, 100]),
    # prefix tiles of 32, 64 and 128 rows
    "prefix32": (2, 1, 16, 256, 512, 72, [72, 9]),
    "prefix32-odd": (2, 1, 16, 256, 515, 71, [71, 9]),
    "prefix64": (3, 1, 16, 256, 512, 72, [72, 9, 0]),
    "prefix64-odd": (3, 1, 16, 256, 515, 71, [71, 9, 0]),
    "prefix128": (18, 4, 29, 256, 4096, 40, [2 * b for b in range(18)]),
    "prefix128-odd": (18, 4, 29, 256, 4099, 41, [2 * b for b in range(18)]),
    "prefix128-own128": (9, 2, 100, 256, 8200, 72, [8 * b for b in range(9)]),
    # head dims between the built ones: join groups that do not divide 256
    **{f"d{D}": (3, 2, 7, D, 130, 200, [200, 0, 65]) for D in (8, 24, 48, 72, 112, 136, 192, 248)},
    **{f"d{D}-odd": (2, 1, 40, D, 131, 201, [201, 65]) for D in (24, 72, 112, 136, 192, 248)},
    **{f"d{D}-wide": (2, 1, 71, D, 129, 205, [205, 64]) for D in (40, 88, 136, 200)},
    # several rows to a joining workgroup at dims that do not divide it
    **{f"d{D}-joined": (130, 2, 8, D, 33, 72, [(7 * b) % 73 for b in range(130)])
       for D in (24, 136, 192)},
}


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_head_dims(lh, case, e):  # noqa: F811
    for weights in (False, True):
        check(lh, case, *CASES[case], TYPES[e], weights)
