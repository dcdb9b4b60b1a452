"""Rows whose scores are all -inf are zeros whatever their keys' v holds; rows beside them
in a tile, which see other keys too, are what they are without them."""
import math

import pytest
import torch

from tests.test_gpu_window import TYPES, attend, lh, make, near, reference  # noqa: F401

pytestmark = pytest.mark.gpu

# B, G, H, D, T, S, lens, window, sinks: tiles of 32 rows in one piece and split, of 64, of
# 128 and 256; head dims on and off the built ones; K's rows on and off 16-byte boundaries
SHAPES = [
    (2, 2, 8, 128, 1, 136, [136, 100], 40, 2), (1, 1, 8, 64, 1, 3000, [3000], 2500, 4),
    (2, 1, 3, 80, 40, 205, [205, 150], 60, 0), (1, 1, 2, 256, 30, 200, [200], 50, 3),
    (8, 8, 1, 128, 260, 264, [264 - b for b in range(8)], 70, 3),
    (8, 8, 2, 64, 260, 264, [264 - b for b in range(8)], 70, 3),
    (8, 8, 4, 96, 260, 261, [261 - b for b in range(8)], 70, 3),
    (8, 8, 2, 256, 256, 264, [264 - b for b in range(8)], 70, 0),
]


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s[:6])) for s in SHAPES])
def test_rows_of_nothing_but_masked_keys(lh, shape, e):  # noqa: F811
    B, G, H, D, T, S, lens, W, sinks = shape
    print("-inf rows", shape, e, flush=True)
    t = make(B, G, H, D, T, S, lens, None, W, sinks, TYPES[e], seed=D)
    t["q"] = t["q"].abs() + 0.1
    # the first sequence: every score -inf, v anything; the last: a stretch of keys so, with
    # ordinary v, whose rows (if it is as long as their window) are zeros
    t["k"][0] = -math.inf
    t["v"][0] = torch.tensor([math.inf, -math.inf, math.nan, 1.0]).repeat(S * D // 4 + 1)[:S * D] \
        .view(S, D).to(TYPES[e])
    if B > 1:
        t["k"][-1, :, :, 100:100 + W // 2] = -math.inf
    want, tol = reference(t, lens, None, W, sinks)
    want[0], tol[0] = 0.0, 0.0
    near(attend(lh, t, lens, None, W, sinks), want, tol, f"-inf rows {shape[:6]} {e}")
