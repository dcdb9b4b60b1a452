"""Every tile of windowed attention in both of its forms: whole (one workgroup to a tile,
which stores its rows itself) and split (partial sums, joined by a second launch), told by
the workspace that the call asks for.  Padded batches, ends inside tiles, infinities that
some rows see, K's rows on and off 16-byte boundaries."""
import math

import pytest
import torch

from tests.test_gpu_window import NAN, attend, lh, make, near, reference  # noqa: F401

pytestmark = pytest.mark.gpu

# D, rows of a tile, H, T: with 64 (b, g)s the largest tile that leaves 256 of them (of
# 32 rows: fewer), and more than 256
WHOLE = [(128, 32, 3, 50), (96, 32, 3, 50), (64, 32, 3, 50), (256, 32, 1, 100),
         (128, 64, 1, 313), (88, 64, 1, 313), (96, 64, 1, 300), (64, 64, 1, 313), (40, 64, 1, 300),
         (128, 128, 2, 300), (104, 128, 2, 300), (96, 128, 2, 300), (64, 128, 2, 300),
         (128, 256, 4, 300), (120, 256, 4, 260), (80, 256, 4, 300), (64, 256, 4, 300),
         (56, 256, 4, 260), (256, 128, 2, 300), (200, 128, 2, 260)]
# D, rows of a tile, H, T, window: fewer tiles than fit, or 256 under a long window
SPLIT = [(128, 32, 3, 20, 70), (72, 32, 3, 20, 70), (64, 32, 3, 20, 70), (256, 32, 1, 60, 300),
         (64, 64, 4, 62, 4700), (32, 64, 4, 62, 4700), (96, 64, 4, 62, 4700), (72, 64, 4, 62, 4700),
         (64, 128, 4, 125, 4700)]


def check(lh, D, rows, H, T, W, odd, e, split):  # noqa: F811
    B, G, sinks = 8, 8, 3
    S = T + W + 8 - (T + W) % 8 - odd
    lens = [S - b for b in range(B)]
    # (under a long window most of the batch is padding: the reference takes long)
    counts = [T - 2 * b - (b == 3) * T // 2 if W < 1000 or b in (0, 3) else b == 1 for b in range(B)]
    print("split" if split else "whole", D, rows, H, T, W, S, e, flush=True)
    need = lh.window_attention_workspace_bytes(B, G, H, D, T, S, W, sinks)
    assert bool(need) == split, need
    t = make(B, G, H, D, T, S, lens, counts, W, sinks, e, D)
    t["v"][3, 3, S - T // 2, 5] = math.inf
    t["v"][1, 7, 1, 6] = NAN
    want, tol = reference(t, lens, counts, W, sinks)
    got = attend(lh, t, lens, counts, W, sinks).double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and not fine.all()
    zero = torch.zeros_like(want)
    near(torch.where(fine, got, zero), torch.where(fine, want, zero), torch.where(fine, tol, zero),
         f"{'split' if split else 'whole'} tile of {rows} D{D} S{S}")


@pytest.mark.parametrize("odd", [0, 3])
@pytest.mark.parametrize("D,rows,H,T", WHOLE)
def test_whole(lh, D, rows, H, T, odd):  # noqa: F811
    assert rows == 32 or 64 * -(-T * H // rows) > 256
    check(lh, D, rows, H, T, 70, odd, torch.bfloat16 if (D + odd) % 16 else torch.float16, False)


@pytest.mark.parametrize("odd", [0, 3])
@pytest.mark.parametrize("D,rows,H,T,W", SPLIT)
def test_split(lh, D, rows, H, T, W, odd):  # noqa: F811
    assert rows == 32 or 64 * -(-T * H // rows) == 256
    check(lh, D, rows, H, T, W, odd, torch.float16 if (D + odd) % 16 else torch.bfloat16, True)
