"""f16: keys far lighter than one beside them still count.

Scores in the log2 domain are set exactly: q and the keys hold one nonzero
element, scale is ln 2, so a key x below the heaviest has p = 2^-x of it.  The
heavy key's values are zero where the light ones' are not, so those columns of
the output are the light keys' sum alone, n 2^-x / (1 + n 2^-x).

Tolerance: the output is rounded once (u |out|, or half of f16's smallest step,
2^-25); each p is held in f16 as 2^7 to 2^15 times its share of the largest, so
to 2^-25 2^-7 of it at worst where it is below f16's normal range and to u of
it otherwise, which powers of two do not need; scale log2 e is 1 to 2^-23, so a
score of 32 is off by at most 2^-18 and p by as much of itself."""
import math

import pytest
import torch

from tests.test_gpu_cache import lh  # noqa: F401

pytestmark = pytest.mark.gpu

# B, G, H, D, P, S: one part of 128 keys; the longest parts (a chunk to each of
# many sequences) on tiles of 32, 64 and 128 rows; prefix splits on all three
SHAPES = [(1, 1, 1, 64, 0, 128), (300, 2, 4, 16, 0, 1024), (600, 1, 33, 8, 0, 1024),
          (260, 1, 71, 8, 0, 1000), (1, 64, 5, 24, 2048, 8), (20, 64, 3, 16, 1001, 8),
          (40, 16, 20, 136, 4096, 8)]


@pytest.mark.parametrize("x", [24, 26, 30])
@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_light_keys(lh, shape, where, x):  # noqa: F811
    B, G, H, D, P, S = shape
    print(shape, where, x, flush=True)
    e, n = torch.float16, P or S
    K = torch.zeros(D, n, dtype=e, device="cuda")
    V = torch.ones(n, D, dtype=e, device="cuda")
    at = 0 if where == "first" else n - 1
    K[0, at] = x
    V[at, 1::2] = 0.0                # odd columns: the light keys alone
    q = torch.zeros(B, G, H, D, dtype=e, device="cuda")
    q[..., 0] = 1.0
    if P:
        k, v = torch.zeros(B, G, D, S, dtype=e, device="cuda"), torch.zeros(B, G, S, D, dtype=e,
                                                                           device="cuda")
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        pre = {"prefix_k": K.expand(G, D, n).contiguous(), "prefix_v": V.expand(G, n, D).contiguous()}
    else:
        k, v = K.expand(B, G, D, n).contiguous(), V.expand(B, G, n, D).contiguous()
        lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
        pre = {}
    out = lh.cache_decode(k, v, q, lens, scale=math.log(2.0), **pre).double()
    light = (n - 1) * 2.0 ** -x
    want = light / (1 + light)
    u = 2.0 ** -11
    tol = u * want + 2.0 ** -25 + n * 2.0 ** -32 + 2.0 ** -18 * want
    err = (out[..., 1::2] - want).abs().max().item()
    assert err <= tol, (err, tol, want)
    assert (out[..., 0::2] - 1.0).abs().max().item() <= 2 * u
