"""How exact the states of linear attention are, and states of wide keys and narrow values
in segments.

A state keeps fp32's accuracy (u = 2^-24 is half a step):
 * One token's a^n k v.  a^n is rounded to fp32 once, its product with v once, the 16-bit
   numbers that the product is split into (three bf16, or two f16) hold it to 2^-24, and up
   to three of them are added in fp32, each sum off by a step (2 u) at most if it truncates:
   under 8 u = 2^-21 in all.  Two bf16 numbers would be off by up to 2^-18.
 * A value that decays over n chunks.  Every chunk rounds it once, by at most u; n roundings
   of either sign, spread evenly over +-u at most, have a standard deviation of sqrt(n / 3) u,
   of which six are allowed, and the 8 u from above.  A chunk's factor rounded by itself
   would be off by up to u / 2 in the same direction every time, n u / 2."""
import math

import numpy as np
import pytest
import torch

from tests.conftest import _record
from tests.test_gpu_linear import TYPES, ints, lh, make, near, on_gpu, reference  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def worst(got, want, bound, what):
    err = (got.double().cpu() / want - 1).abs()
    _record(what, want.numel(), float(err.max()), float(err.max()), float(err.max()) / bound)
    assert float(err.max()) <= bound, (what, float(err.max()), bound)


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("T", [32, 40, 700])
def test_one_token(lh, e, T):  # noqa: F811
    """Sequence b's only token with a value is token b of the last 32; (700: in segments)."""
    B, G, D, E = 32, 1, 16, 128
    g = torch.Generator().manual_seed(T)
    k, v = torch.zeros(B, T, G, D, dtype=TYPES[e]), torch.zeros(B, T, G, E, dtype=TYPES[e])
    at = torch.arange(B)
    value = (1 + torch.rand((B, G, E), generator=g)).to(TYPES[e])
    k[at, T - 32 + at] = 1.0
    v[at, T - 32 + at] = value
    ld = torch.tensor([[-0.0371]])
    _, end = lh.linear_attention(torch.zeros(B, T, G, 1, D, dtype=TYPES[e]).cuda(), k.cuda(),
                                 v.cuda(), ld.cuda())
    weight = torch.exp(ld.double()[0, 0] * (31 - at))
    want = (weight[:, None, None] * value.double()).view(B, G, 1, 1, E).expand(B, G, 1, D, E)
    worst(end, want, 8 * U, f"one token T{T} {e}")


def steep_factors(n, T):
    """n log decays near -3e-5 whose factor over 32 tokens lies near the middle between two
    fp32 numbers, always on the same side."""
    g = (-3e-5 - np.arange(200000) * 1e-11).astype(np.float32)
    x = np.exp(32.0 * g.astype(np.float64))
    off = x.astype(np.float32) / x - 1
    picked = g[off > 0.8 * U / 2][:n]
    assert len(picked) == n
    return torch.from_numpy(picked.copy())


@pytest.mark.parametrize("heads", [512, 4])
def test_long_memory(lh, heads):  # noqa: F811
    """One value over 60000 tokens: 512 heads, one after the other's chunks (no workspace),
    and 4, whose prompts are cut into segments."""
    T, D, E = 60000, 8, 8
    ld = steep_factors(heads, T)
    k = torch.zeros(1, T, heads, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, T, heads, E, dtype=torch.bfloat16, device="cuda")
    k[:, 0] = 1.0
    value = 1 + torch.arange(E) / 8
    v[:, 0] = value.to(torch.bfloat16).cuda()
    assert bool(lh.linear_attention_workspace_bytes(1, heads, 1, D, E, T)) == (heads < 512)
    _, end = lh.linear_attention(torch.zeros_like(k).unsqueeze(3), k, v, ld[:, None].cuda())
    n = -(-T // 32)
    want = torch.exp(ld.double() * (T - 1))[:, None, None] * value.double()
    want = want.expand(heads, D, E).reshape(1, heads, 1, D, E)
    worst(end, want, 6 * math.sqrt(n / 3) * U + 8 * U, f"{heads} heads T{T}")


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("D,E", [(256, 64), (136, 32), (256, 128)])
def test_wide_keys_in_segments(lh, D, E, e):  # noqa: F811
    """Ends at, before and behind the ends of chunks and stretches; states in place."""
    counts = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 639, 640]
    B, T = len(counts), 640
    print("wide", D, E, e, flush=True)
    t = make(B, 1, 1, D, E, T, counts, TYPES[e], seed=D + E)
    assert lh.linear_attention_workspace_bytes(B, 1, 1, D, E, T)
    want, tol, end, etol = reference(t, counts)
    d = on_gpu(t)
    out = torch.full((B, T, 1, 1, E), 7.0, dtype=TYPES[e], device="cuda")
    _, s = lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out, d["state"],
                               counts=ints(counts))
    assert s is d["state"]
    near(out, want, tol, f"wide D{D} E{E} {e}")
    near(s, end, etol, f"wide D{D} E{E} {e} state")
