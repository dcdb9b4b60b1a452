"""How a step cuts its sequences: without a prefix, and with at most half as many
sequences as workgroups run at once, all chunks fit in one round of them.  The
cut is read from the start of the workspace, where the step leaves each
sequence's first chunk and their number; results against 64 bits beside it."""
import math

import pytest
import torch

from tests.test_gpu_cache import lh  # noqa: F401

pytestmark = pytest.mark.gpu

# B, G, H, D, shortest and longest length; sums of rounded-up chunks that
# passed a round when the chunk size came from the mean alone
CASES = [(5, 8, 4, 128, 7808, 7808), (57, 1, 32, 128, 8000, 8000), (22, 4, 16, 128, 2904, 2904),
         (47, 4, 2, 80, 3056, 3056), (11, 8, 5, 256, 4032, 4032), (1, 8, 4, 128, 7777, 7777),
         # more than 64 sequences: the lengths are summed by the whole workgroup
         (65, 1, 32, 64, 897, 897), (134, 1, 40, 128, 586, 586), (173, 1, 8, 64, 287, 287),
         (107, 1, 128, 64, 4900, 4900), (128, 1, 3, 256, 2000, 2000),
         # lengths apart, some sequences empty
         (32, 1, 32, 128, 0, 8192), (70, 2, 8, 64, 100, 3000)]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("case", CASES, ids=["x".join(map(str, c)) for c in CASES])
def test_chunks_fit_one_round(lh, case, weights):  # noqa: F811
    B, G, H, D, lo, hi = case
    print(case, weights, flush=True)
    g = torch.Generator(device="cuda").manual_seed(B + hi)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    S = (hi + 7) // 8 * 8
    k, v, q = rnd(B, G, D, S), rnd(B, G, S, D), rnd(B, G, H, D)
    n = [lo + (hi - lo) * b // max(1, B - 1) for b in range(B)]
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    w = torch.zeros(B, G, S, device="cuda") if weights else None
    ws = lh.cache_decode_workspace(B, G, H, D, 0, S, weights, "cuda:0")
    out = lh.cache_decode(k, v, q, lens, None, ws, weights=w)
    plan = ws[:8 * B].view(torch.int32).view(B, 2).tolist()
    at, tiles = 0, G * (1 if H <= 32 else -(-H // 128))
    for b in range(B):                       # consecutive, none without keys
        if n[b]:
            assert plan[b][0] == at and plan[b][1] >= 1, (b, plan[b], at)
            at += plan[b][1]
    assert at * tiles <= (256 if D > 128 else 512), (at, tiles)
    # bounds as in test_gpu_cache: a rounding of out, two of p (bf16: 2^-8), fp32 beside them
    for b in {0, B // 2, B - 1}:
        if n[b] == 0:
            assert not out[b].any()
            continue
        for h in range(G):
            p = torch.softmax(q[b, h].double() @ k[b, h, :, :n[b]].double() / math.sqrt(D), -1)
            vals = v[b, h, :n[b]].double()
            o, A = p @ vals, p @ vals.abs()
            assert ((out[b, h].double() - o).abs() <= 2.0 ** -8 * o.abs() + 2.1 * 2.0 ** -8 * A).all()
            if weights:
                s = p.sum(0)
                assert ((w[b, h, :n[b]].double() - s).abs() <= 1e-4 * s + 1e-30).all()
