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


# B, G, H, D, E, T, counts: every key dim's kernel on 64 and 128 columns, prompts in one
# piece (more heads than run at once) and in segments
PROMPTS = [
    (2, 2, 2, 64, 64, 100, [100, 77]), (2, 1, 3, 40, 72, 130, None), (1, 2, 1, 128, 128, 97, None),
    (2, 1, 2, 128, 48, 70, [70, 33]), (1, 1, 2, 256, 64, 66, None), (2, 1, 1, 136, 136, 95, [95, 64]),
    (2, 1, 1, 64, 64, 700, [700, 515]), (1, 2, 1, 128, 128, 650, None), (1, 1, 1, 200, 40, 600, None),
    (1, 1, 1, 256, 256, 520, None), (1, 1, 2, 72, 64, 640, None), (1, 1, 1, 16, 160, 610, None),
]


def spoiled(shape, e, decay, seed):
    """Inputs with infinities and NaN of q, k, v and the states, in columns, rows and tokens
    of their own (early, at a chunk's ends, late) beside untouched ones."""
    B, G, H, D, E, T, counts = shape
    t = make(B, G, H, D, E, T, counts, e, True, seed)
    t["log_decay"][:] = decay
    t["q"][..., 0, :] = t["q"][..., 0, :].abs() + 0.25        # (heads 0: infinities keep their sign)
    k, v, q, s = t["k"], t["v"], t["q"], t["state"]
    k[:, :, 0, 1:3] = k[:, :, 0, 1:3].abs() + 0.1
    k[0, 20, 0] = k[0, 20, 0].abs() + 0.1                      # (one that makes a column all +inf)
    v[0, 20, 0, 3], v[0, 31, 0, 4], v[0, 32, 0, 6] = INF, -INF, INF
    v[0, 40, 0, 7], v[0, T - 3, 0, E - 1] = NAN, INF
    v[0, 20, 0, 9], v[0, 50, 0, 9] = INF, -INF
    v[0, 45, 0, 10], k[0, 45, 0, 5] = INF, 0.0
    s[0, 0, 0, 3, 12], s[0, 0, H - 1, 4, 13], s[0, 0, 0, 2, 14] = INF, -INF, NAN
    if B > 1:                                                  # a sequence with an infinite key
        k[1, 12, 0, 1] = INF
        k[1, 39, 0, 2], v[1, 39, 0, 8] = -INF, INF
    if G > 1:                                                  # heads with infinite queries only
        q[0, 35, 1, 0, 3], q[0, 64, 1, H - 1, 2], q[0, 5, 1, 0, 1] = INF, -INF, NAN
    return t


def run(lh, t, counts):  # noqa: F811
    d = on_gpu(t)
    B, T, G, H, _ = t["q"].shape
    out = torch.full((B, T, G, H, t["v"].shape[-1]), 7.0, dtype=t["q"].dtype, device="cuda")
    return lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out,
                               counts=ints(counts))


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", PROMPTS, ids=["x".join(map(str, s[:6])) for s in PROMPTS])
def test_prompt(lh, shape, e):  # noqa: F811
    for decay in (0.0, -0.05, -30.0, -200.0):
        print("prompt", shape, decay, e, flush=True)
        t = spoiled(shape, TYPES[e], decay, shape[3])
        want, tol, end, etol = recurrence(t, shape[6])
        o, s = run(lh, t, shape[6])
        alike(s, end, etol, f"infinite prompt {shape[3:6]} {decay} {e} state")
        alike(o, want, tol, f"infinite prompt {shape[3:6]} {decay} {e} out")


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("decay", [-0.5, -INF])
def test_decays_of_many_heads(lh, decay, e):  # noqa: F811
    """More heads than run at once: prompts in one piece."""
    shape = (4, 33, 2, 64, 72, 90, [90, 0, 31, 64])
    assert not lh.linear_attention_workspace_bytes(*shape[:6])
    t = spoiled((4, 33, 2, 64, 72, 90, None), TYPES[e], decay, 5)
    for b, c in enumerate(shape[6]):
        for x in "qkv":
            t[x][b, c:] = NAN
    want, tol, end, etol = recurrence(t, shape[6])
    o, s = run(lh, t, shape[6])
    alike(s, end, etol, f"infinite prompt, many heads {decay} {e} state")
    alike(o, want, tol, f"infinite prompt, many heads {decay} {e} out")


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("x", "vkq")
def test_earlier_rows_keep_their_bits(lh, x, e):  # noqa: F811
    """Rows ahead of an infinity, in its chunk and before, are what they are without it."""
    for B, G, H, D, E, T, at in ((1, 2, 1, 64, 64, 100, 50), (1, 1, 2, 128, 128, 640, 333),
                                 (1, 1, 1, 40, 72, 70, 69)):
        t = make(B, G, H, D, E, T, None, TYPES[e], True, 3)
        a, _ = run(lh, t, None)
        t[x][0, at, 0, ..., 5] = INF
        b, _ = run(lh, t, None)
        assert torch.equal(a[:, :at], b[:, :at])
        assert not torch.isfinite(b[0, at, 0]).all()
        assert torch.equal(a[:, :, 1:], b[:, :, 1:])          # other heads' rows


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("T", [220, 700])
@pytest.mark.parametrize("D,E", [(64, 64), (128, 136), (40, 72)])
def test_what_follows_lost_columns(lh, D, E, T, e):  # noqa: F811
    """Infinities and NaN that meet columns of NaN, beside live ones, in chunks apart from
    each other with ordinary ones between (T220: one piece, 700: segments)."""
    for decay in (-0.01, -20.0):
        print("lost columns", D, E, T, decay, e, flush=True)
        t = make(3, 1, 2, D, E, T, None, TYPES[e], True, D + T)
        t["log_decay"][:] = decay
        t["q"][..., 0, :] = t["q"][..., 0, :].abs() + 0.25
        k, v = t["k"], t["v"]
        v[0, 40:, 0, :] = NAN                  # a sequence lost from token 40 on, in all columns
        k[0, 100, 0, 3], v[0, 130, 0, 5] = INF, INF
        v[1, 10:, 0, :16] = NAN                # a wave's columns, then infinities there and beside
        v[1, 70, 0, 3], v[1, 100, 0, 20], v[1, 101, 0, 20], v[1, T - 1, 0, 30] = INF, INF, -INF, INF
        k[1, 165, 0], v[1, 165, 0, E - 1] = 0.5, -INF
        v[2, 33, 0, 1:E:2] = NAN               # every other column; then an infinite key
        t["q"][2, 150, 0, 1, 2] = -INF
        k[2, 190, 0, 4] = -INF
        want, tol, end, etol = recurrence(t, None)
        o, s = run(lh, t, None)
        alike(s, end, etol, f"lost columns D{D} E{E} T{T} {decay} {e} state")
        alike(o, want, tol, f"lost columns D{D} E{E} T{T} {decay} {e} out")


def test_finite_values_that_look_like_infinities(lh):  # noqa: F811
    """bf16 values past 2^121 have the bits of f16's infinities and NaN: finite all the same."""
    for T in (70, 700):
        t = make(2, 1, 2, 64, 64, T, None, torch.bfloat16, True, T)
        t["v"][0, 20, 0, 5], t["v"][1, T - 2, 0, 6] = 2.0 ** 121, -2.0 ** 123
        t["k"][0, 33, 0, 7] = 2.0 ** 121
        t["v"][0, 33, 0] = 2.0 ** -8
        want, tol, end, etol = recurrence(t, None)
        assert torch.isfinite(want).all() and float(want.abs().max()) < 2.0 ** 127
        o, s = run(lh, t, None)
        alike(s, end, etol, f"huge T{T} state")
        alike(o, want, tol, f"huge T{T} out")
