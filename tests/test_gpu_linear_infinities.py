"""Infinities and NaN in linear attention: states and outputs are what the recurrence
S_t = a S_(t-1) + k_t v_t^T, out_t = scale S_t^T q_t gives in IEEE arithmetic, value by
value: +inf, -inf and NaN where it gives them, the ordinary results beside them.

The recurrence runs here token by token in 64 bits with a = exp(log_decay) as fp32 holds
it (0 below the smallest subnormal, where 0 inf is NaN).  A finite result is held to
test_gpu_linear.py's bounds, whose absolute sums are taken the same way over the
magnitudes of what is finite."""
import math

import pytest
import torch

from tests.test_gpu_linear import NAN, TYPES, ints, lh, make, near, on_gpu, step_inputs  # noqa: F401

pytestmark = pytest.mark.gpu

INF = math.inf


def recurrence(t, counts, scale=None):
    """out (7 behind a sequence), the last states, and the bounds where they are finite."""
    q, k, v = (t[x].double() for x in "qkv")
    B, T, G, H, D = q.shape
    E = v.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    e = t["q"].dtype
    u, fine = torch.finfo(e).eps / 2, (T + 2 * D + 64) * 2.0 ** -23
    a = torch.exp(t["log_decay"].double()).float().double()[..., None, None]       # G H 1 1
    S = torch.zeros(B, G, H, D, E, dtype=torch.float64) if t["state"] is None \
        else t["state"].double().clone()
    mag = lambda x: torch.where(torch.isfinite(x), x.abs(), 0.0)  # noqa: E731
    M = mag(S)
    out, tol = torch.full((B, T, G, H, E), 7.0, dtype=torch.float64), \
        torch.zeros(B, T, G, H, E, dtype=torch.float64)
    for b in range(B):
        c = T if counts is None else min(max(counts[b], 0), T)
        for i in range(c):
            kk, vv, qq = k[b, i][:, None, :, None], v[b, i][:, None, None], q[b, i][..., None]
            S[b] = a * S[b] + kk * vv
            M[b] = a * M[b] + mag(kk) * mag(vv)
            out[b, i] = scale * (S[b] * qq).sum(-2)
            A = scale * (M[b] * mag(qq)).sum(-2)
            tol[b, i] = u * mag(out[b, i]) + (u * (1 + 2 * u) + fine) * A + 1e-30 \
                + (64 * 2.0 ** -25 * mag(v[b, :c]).max() + 2.0 ** -25 if e == torch.float16 else 0)
    return out, tol, S, (2.0 ** -16 + fine) * M + 1e-30


def alike(got, want, tol, what):
    """The same infinities and NaN, and near where the recurrence is finite."""
    got = got.double().cpu()
    for name, x, y in (("nan", torch.isnan(got), torch.isnan(want)),
                       ("+inf", got == INF, want == INF), ("-inf", got == -INF, want == -INF)):
        wrong = (x != y).nonzero()
        assert not len(wrong), (what, name, len(wrong), [(i, float(got[tuple(i)]),
                                                          float(want[tuple(i)]))
                                                         for i in wrong[:4].tolist()])
    there = torch.isfinite(want)
    zero = torch.zeros_like(want)
    near(torch.where(there, got, zero), torch.where(there, want, zero),
         torch.where(there, tol, zero), what)


# heads that forget nothing, something, all but nothing (a subnormal a), all (a = 0)
DECAYS = [0.0, -0.1, -30.0, -100.0, -200.0, -INF]


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("decay", DECAYS)
def test_step(lh, decay, e):  # noqa: F811
    """Infinite states, keys, values and queries of one token."""
    for B, G, H, D, E in ((3, 2, 2, 64, 64), (2, 1, 1, 256, 200), (2, 1, 3, 8, 16)):
        print("step", B, G, H, D, E, decay, e, flush=True)
        t = step_inputs(B, G, H, D, E, TYPES[e], seed=D)
        t["log_decay"][:] = decay
        t["q"] = t["q"].abs() + 0.25              # (so that infinities of one sign stay such)
        s = t["state"]
        s[0, 0, 0, 3, 5], s[0, 0, 0, 4, 5] = INF, INF
        s[0, 0, H - 1, 2, 7], s[0, G - 1, 0, 1, 9] = -INF, NAN
        s[0, 0, 0, 6, 11], s[0, 0, 0, 7, 11] = INF, -INF
        t["v"][1, 0, 1], t["v"][1, 0, 3], t["k"][1, G - 1, 2] = INF, -INF, INF
        t["k"][1, 0, 5] = 0.0
        if G > 1:
            t["q"][0, 1, 1, 4] = -INF
        full = {**t, **{x: t[x].unsqueeze(1) for x in "qkv"}}
        want, tol, end, etol = recurrence(full, None)
        d = on_gpu(t)
        o = lh.linear_attention_step(d["q"], d["k"], d["v"], d["log_decay"], d["state"])
        alike(d["state"], end, etol, f"infinite step {decay} {e} state")
        alike(o, want[:, 0], tol[:, 0], f"infinite step {decay} {e} out")
