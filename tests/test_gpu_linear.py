"""Linear attention with a decay for each head (linear_attention,
linear_attention_step) against a plain implementation in 64 bits.

Tolerances (derived, not fitted).  With u = finfo(e).eps / 2, a = exp(log_decay):
  A_t = scale (sum_j a^(t-j) (|q_t|.|k_j|) |v_j| + a^(t+1) |q_t|^T |S_-1|)
bounds the sum of the absolute terms of out_t, and R = sum_j a^(c-1-j) |k_j| |v_j|^T +
a^c |S_-1| that of the state.  A kernel may round to 16 bits, on the way to the output,
each term's factor once (a state as a product's operand, or q_t.k_j a^(t-j)): u A; and
the output itself: u |out|.  A state keeps fp32: its terms may pass a product as a sum
of two 16-bit numbers (each half a step of the one before: 2^-16 covers bf16, f16's is
finer), and fp32 sums of T tokens, D products and a few factors err by at most (T + 2 D +
64) 2^-23 of the absolute sum, accumulations that truncate included.  f16 holds nothing
below 2^-25: 64 factors of at most that beside |v| <= max, and the output's own."""
import math

import pytest
import torch

from tests.conftest import _record

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
NAN = float("nan")


@pytest.fixture(scope="module")
def lh():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import loom_hip
    return loom_hip


def clamp(x, lo, hi):
    return min(max(x, lo), hi)


def make(B, G, H, D, E, T, counts, e, state=True, seed=0, decay=None, std=1.0):
    """Inputs on the CPU; NaN in all tokens behind a sequence's."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    t = {"q": (rnd(B, T, G, H, D) * std).to(e), "k": (rnd(B, T, G, D) / math.sqrt(D)).to(e),
         "v": rnd(B, T, G, E).to(e),
         "log_decay": -torch.exp2(-9 * torch.rand((G, H), generator=g) - 1) if decay is None
         else torch.full((G, H), decay),
         "state": rnd(B, G, H, D, E) if state else None}
    for b in range(B):
        c = T if counts is None else clamp(counts[b], 0, T)
        for x in "qkv":
            t[x][b, c:] = NAN
    return t


def reference(t, counts, scale=None):
    """out (7 behind a sequence), the last states, and their bounds, in 64 bits."""
    q, k, v = (t[x].double() for x in "qkv")
    B, T, G, H, D = q.shape
    E = v.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    e = t["q"].dtype
    u = torch.finfo(e).eps / 2
    fine = (T + 2 * D + 64) * 2.0 ** -23
    out, tol = torch.full((B, T, G, H, E), 7.0, dtype=torch.float64), \
        torch.zeros(B, T, G, H, E, dtype=torch.float64)
    end = torch.zeros(B, G, H, D, E, dtype=torch.float64)
    etol = torch.zeros_like(end)
    ld = t["log_decay"].double().clamp(min=-1e30)
    for b in range(B):
        c = T if counts is None else clamp(counts[b], 0, T)
        i = torch.arange(c)
        lag = i[:, None] - i
        for g in range(G):
            for h in range(H):
                a = float(ld[g, h])
                S = torch.zeros(D, E, dtype=torch.float64) if t["state"] is None \
                    else t["state"][b, g, h].double()
                m = torch.where(lag >= 0, torch.exp(a * lag.clamp(min=0)), 0.0)
                x, y, z = q[b, :c, g, h], k[b, :c, g], v[b, :c, g]
                s = x @ y.t()
                rise = torch.exp(a * (i + 1.0))[:, None]
                o = scale * (torch.where(lag >= 0, s * m, 0.0) @ z + rise * (x @ S))
                A = scale * ((x.abs() @ y.abs().t() * m) @ z.abs() + rise * (x.abs() @ S.abs()))
                out[b, :c, g, h] = o
                top = z.abs().max() if c else 0.0
                tol[b, :c, g, h] = u * o.abs() + (u * (1 + 2 * u) + fine) * A + 1e-30 \
                    + (64 * 2.0 ** -25 * top + 2.0 ** -25 if e == torch.float16 else 0)
                w = torch.exp(a * (c - 1.0 - i))[:, None]
                end[b, g, h] = math.exp(a * c) * S + (y * w).t() @ z
                etol[b, g, h] = (2.0 ** -16 + fine) * ((y.abs() * w).t() @ z.abs()
                                                       + math.exp(a * c) * S.abs()) + 1e-30
                if c == 0:
                    etol[b, g, h] = 0
    return out, tol, end, etol


def near(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(),
                           float(err[bad].max()), float((err / tol)[bad].max()))
    _record(what, want.numel(), float(err.max()), 0.0, float((err / tol.clamp(min=1e-30)).max()))


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def on_gpu(t):
    return {x: None if y is None else y.cuda() for x, y in t.items()}


def attend(lh, t, counts, scale=None, **kw):
    d = on_gpu(t)
    B, T, G, H, D = t["q"].shape
    out = torch.full((B, T, G, H, t["v"].shape[-1]), 7.0, dtype=t["q"].dtype, device="cuda")
    got, end = lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out,
                                   counts=ints(counts), scale=scale, **kw)
    assert got is out
    return out, end


def check(lh, what, B, G, H, D, E, T, counts, e, state=True, seed=0, decay=None, std=1.0,
          scale=None):
    print(what, B, G, H, D, E, T, counts and counts[:6], e, state, decay, flush=True)
    t = make(B, G, H, D, E, T, counts, e, state, seed, decay, std)
    want, tol, end, etol = reference(t, counts, scale)
    o, s = attend(lh, t, counts, scale)
    name = f"{what} B{B} G{G} H{H} D{D} E{E} T{T} {e}"
    near(o, want, tol, name + " out")
    near(s, end, etol, name + " state")


SHAPES = [
    # B, G, H, D, E, T, counts
    (1, 1, 1, 64, 64, 1, None), (1, 1, 1, 8, 8, 3, None), (2, 2, 1, 128, 128, 16, None),
    (1, 2, 2, 64, 32, 31, None), (2, 1, 3, 128, 64, 32, [32, 5]), (1, 1, 1, 128, 128, 33, None),
    (2, 2, 1, 64, 128, 63, None), (1, 3, 1, 128, 128, 64, None), (2, 1, 2, 80, 96, 65, None),
    (3, 2, 1, 128, 128, 130, [130, 0, 64]), (2, 2, 2, 40, 72, 200, [200, 129]),
    (1, 1, 1, 256, 256, 100, None), (2, 1, 1, 256, 64, 70, [70, 1]), (1, 1, 4, 64, 256, 77, None),
    (1, 4, 1, 128, 128, 700, None), (4, 1, 1, 16, 248, 150, [-3, 1000, 128, 96]),
    (2, 1, 1, 200, 136, 300, None), (17, 2, 1, 64, 64, 40, [(5 * i) % 41 for i in range(17)]),
]


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s[:6])) for s in SHAPES])
def test_linear(lh, shape, e):
    check(lh, "linear", *shape, TYPES[e])
    check(lh, "linear, no state", *shape, TYPES[e], state=False, seed=1)


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("decay", [0.0, -1e-4, -0.7, -30.0, -1e4, -math.inf, 0.02])
def test_decays(lh, decay, e):
    """From heads that forget nothing to heads without memory (and one that grows)."""
    check(lh, "decay", 2, 1, 2, 64, 64, 200, [200, 77], TYPES[e], decay=decay)


@pytest.mark.parametrize("e", TYPES)
def test_long_prompts(lh, e):
    """Few heads over a long axis, which is split and joined; ends inside and at
    the splits."""
    t = TYPES[e]
    check(lh, "long", 1, 2, 1, 128, 128, 2500, None, t, decay=-1e-3)
    check(lh, "long, ragged", 3, 1, 1, 64, 64, 2049, [2049, 1024, 700], t)
    check(lh, "long, no state", 1, 1, 2, 128, 64, 1984, None, t, state=False, decay=0.0)


@pytest.mark.parametrize("e", TYPES)
def test_ends_of_chunks_and_stretches(lh, e):
    """Sequences that end at, before and behind the ends of chunks of 32 tokens and of
    the stretches that a long prompt is split into; states in place."""
    counts = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 639, 640]
    B, T = len(counts), 640
    for D, E in ((64, 64), (128, 96), (32, 200)):
        print("ends", D, E, e, flush=True)
        t = make(B, 1, 1, D, E, T, counts, TYPES[e], seed=D)
        assert lh.linear_attention_workspace_bytes(B, 1, 1, D, E, T)      # (it is split)
        want, tol, end, etol = reference(t, counts)
        d = on_gpu(t)
        out = torch.full((B, T, 1, 1, E), 7.0, dtype=TYPES[e], device="cuda")
        _, s = lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out,
                                   d["state"], counts=ints(counts))
        assert s is d["state"]
        near(out, want, tol, f"ends D{D} E{E} {e}")
        near(s, end, etol, f"ends D{D} E{E} {e} state")


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("D,E", [(128, 128), (64, 64), (256, 128), (48, 72)])
def test_many_heads(lh, D, E, e):
    """More heads than run at once: every prompt in one piece, over many chunks."""
    B, G, H, T = 5, 40, 3, 190
    counts = [190, 1, 100, 160, 31]
    check(lh, "many heads", B, G, H, D, E, T, counts, TYPES[e], seed=D)
    assert not lh.linear_attention_workspace_bytes(B, G, H, D, E, T)


def test_decay_of_a_long_memory(lh):
    """A slow decay over many tokens: the rounding of one factor near 1 would be off by
    the tokens that it is applied to.  The last state of ones, exactly (64 bits), to
    1e-6: 16 tokens' worth of fp32 steps of the sum, far below T 2^-24."""
    T, g = 20000, -2.0 ** -13 * 1.0000001
    k = torch.zeros(1, T, 1, 8, dtype=torch.bfloat16, device="cuda")
    k[..., 0] = 1.0
    v = torch.ones(1, T, 1, 8, dtype=torch.bfloat16, device="cuda")
    ld = torch.full((1, 1), g, device="cuda")
    _, end = lh.linear_attention(k.unsqueeze(3), k, v, ld)
    x = float(ld)
    want = (1 - math.exp(x * T)) / (1 - math.exp(x))
    assert abs(float(end[0, 0, 0, 0, 0]) / want - 1) < 4e-6
    assert not end[0, 0, 0, 1:].any()


@pytest.mark.parametrize("e", TYPES)
def test_scales(lh, e):
    check(lh, "scaled", 2, 1, 2, 64, 64, 100, None, TYPES[e], scale=3.0)
    check(lh, "large q", 2, 1, 2, 64, 64, 100, None, TYPES[e], std=30.0)
    check(lh, "small q", 2, 1, 2, 64, 64, 100, None, TYPES[e], std=2e-3)


def test_f16_beyond_its_range(lh):
    """States and scores past 65504, and tiny ones, where the outputs are ordinary: f16
    holds neither, the formula does."""
    T = 150
    for up in (2.0 ** 9, 2.0 ** -9):
        t = make(1, 1, 2, 64, 64, T, None, torch.float16, seed=4, decay=-1e-3)
        # k and v 2^9 (2^-9) times larger, q 2^18 times smaller (larger) in turn
        t["k"] = (t["k"].float() * up * 8).half()
        t["v"] = (t["v"].float() * up).half()
        t["state"] = t["state"] * up * up * 8
        t["q"] = (t["q"].float() / up ** 1.5).half()
        want, tol, end, etol = reference(t, None)
        assert up < 1 or float(end.abs().max()) > 65504
        o, s = attend(lh, t, None)
        near(o, want, tol, f"f16 x {up}")
        near(s, end, etol, f"f16 x {up} state")


def test_f16_scores_beyond_its_range(lh):
    """q.k past 65504 beside small values: the products of the two fit."""
    t = make(1, 1, 1, 64, 64, 90, None, torch.float16, seed=5, state=False, decay=-0.1)
    t["q"] = (t["q"].float() * 800).half()
    t["k"] = (t["k"].float() * 8 * 200).half()
    t["v"] = (t["v"].float() * 2.0 ** -10).half()
    want, tol, end, etol = reference(t, None)
    assert float((t["q"].double()[0, :, 0, 0] @ t["k"].double()[0, :, 0].t()).abs().max()) / 8 > 65504
    o, s = attend(lh, t, None)
    near(o, want, tol, "f16 scores")
    near(s, end, etol, "f16 scores' state")


@pytest.mark.parametrize("e", TYPES)
def test_what_comes_later_does_not_reach_a_row(lh, e):
    """NaN and infinities of a token reach its own and later rows, in its columns,
    and no earlier ones."""
    T, at = 140, 100
    for x, value in (("v", math.inf), ("v", NAN), ("k", NAN), ("q", NAN)):
        t = make(1, 2, 2, 64, 64, T, None, TYPES[e], seed=6)
        where = {"v": (0, at, 1, 5), "k": (0, at, 1, 5), "q": (0, at, 1, 1, 5)}[x]
        bad = torch.zeros(1, T, 2, 2, 64, dtype=torch.bool)
        lost = torch.zeros(1, 2, 2, 64, 64, dtype=torch.bool)
        if x == "v":
            bad[0, at:, 1, :, 5] = lost[0, 1, :, :, 5] = True
        elif x == "k":
            bad[0, at:, 1] = lost[0, 1, :, 5] = True
        else:
            bad[0, at, 1, 1] = True
        t[x][where] = 0.0           # what else there is does not depend on it
        want, tol, end, etol = reference(t, None)
        t[x][where] = value
        o, s = attend(lh, t, None)
        assert torch.equal(~torch.isfinite(o.float().cpu()), bad), x
        assert torch.equal(~torch.isfinite(s.cpu()), lost), x
        near(torch.where(bad, want, o.double().cpu()), want, tol, f"beside {x} {value}")
        near(torch.where(lost, end, s.double().cpu()), end, etol, f"beside {x} {value}, state")


def step_inputs(B, G, H, D, E, e, seed=0):
    t = make(B, G, H, D, E, 1, None, e, True, seed)
    return {**t, "q": t["q"][:, 0].contiguous(), "k": t["k"][:, 0].contiguous(),
            "v": t["v"][:, 0].contiguous()}


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (1, 2, 1, 64, 64), (3, 2, 3, 80, 96),
                                   (2, 4, 1, 128, 128), (1, 1, 4, 256, 256), (5, 1, 2, 128, 32),
                                   (2, 3, 1, 40, 200), (40, 8, 1, 64, 128), (1, 1, 1, 256, 8),
                                   (1, 1, 1, 8, 256), (130, 16, 1, 128, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_step(lh, shape, e):
    print("step", shape, e, flush=True)
    t = step_inputs(*shape, TYPES[e])
    counts = [1 - (b % 5 == 3) for b in range(shape[0])]
    full = {**t, **{x: t[x].unsqueeze(1) for x in "qkv"}}
    want, tol, end, etol = reference(full, counts)
    d = on_gpu(t)
    out = torch.full((*shape[:3], shape[4]), 7.0, dtype=TYPES[e], device="cuda")
    got = lh.linear_attention_step(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out,
                                   counts=ints(counts))
    assert got is out
    near(out, want[:, 0], tol[:, 0], f"step {shape} {e} out")
    near(d["state"], end, etol, f"step {shape} {e} state")


def test_arguments(lh):
    """State in place, outputs and workspaces given; zero tokens."""
    t = make(2, 2, 1, 128, 128, 1000, [1000, 300], torch.bfloat16, seed=7)
    ref, end = attend(lh, t, [1000, 300])
    d = on_gpu(t)
    assert torch.equal(d["state"].cpu(), t["state"])
    need = lh.linear_attention_workspace_bytes(2, 2, 1, 128, 128, 1000)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    o, s = lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"],
                               state_out=d["state"], workspace=ws, counts=ints([1000, 300]))
    assert s is d["state"] and torch.equal(s, end)
    for b, c in enumerate([1000, 300]):
        assert torch.equal(o[b, :c], ref[b, :c])
    if need:
        with pytest.raises(ValueError, match="workspace needs"):
            lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], workspace=ws[:need - 1])
    before = s.clone()
    out = torch.full_like(ref, 3.0)
    lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], s, out, s, counts=ints([0, -1]))
    assert torch.equal(s, before) and (out == 3.0).all()
    _, z = lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], counts=ints([0, 0]))
    assert not z.any()


def test_prompt_and_steps_agree(lh):
    """A ragged prompt in two pieces, then steps, against the whole."""
    B, G, H, D, E, T, steps = 3, 2, 2, 64, 96, 200, 8
    counts = [200, 65, 131]
    t = make(B, G, H, D, E, T + steps, None, torch.bfloat16, seed=8)
    total = [c + steps for c in counts]
    want, tol, end, etol = reference(t, total)
    d = on_gpu(t)
    state = d["state"]
    at = torch.arange(B)
    cut = 64
    first = {x: d[x][:, :cut].contiguous() for x in "qkv"}
    o, state = lh.linear_attention(first["q"], first["k"], first["v"], d["log_decay"], state)
    near(o, want[:, :cut], tol[:, :cut], "first piece")
    rest = {x: d[x][:, cut:T].contiguous() for x in "qkv"}
    left = [c - cut for c in counts]
    o, state = lh.linear_attention(rest["q"], rest["k"], rest["v"], d["log_decay"], state,
                                   counts=ints(left))
    for b in range(B):
        near(o[b, :left[b]], want[b, cut:counts[b]], tol[b, cut:counts[b]], "second piece")
    for i in range(steps):
        x = torch.tensor(counts) + i
        new = {y: d[y][at, x].contiguous() for y in "qkv"}
        o = lh.linear_attention_step(new["q"], new["k"], new["v"], d["log_decay"], state)
        near(o, want[at, x], tol[at, x], f"step {i}")
    near(state, end, etol, "last state")


def test_a_layer_of_each(lh):
    """A hybrid stack's two layers over a prompt and steps: window attention's output is
    linear attention's value, as a program runs them, against 64 bits.  The second
    layer's v is the first's rounded output, so each is held to its own bound."""
    from tests import test_gpu_window as tw
    B, G, H, D, S, W, sinks, T = 2, 2, 1, 64, 128, 30, 2, 90
    lens = [90, 70]
    a = tw.make(B, G, H, D, T, S, lens, lens, W, sinks, torch.bfloat16, seed=11)
    a["q"][:] = torch.nan_to_num(a["q"])
    want, tol = tw.reference(a, lens, lens, W, sinks)
    x = lh.window_attention(a["k"].cuda(), a["v"].cuda(), a["q"].cuda(), tw.ints(lens), W,
                            torch.full_like(a["q"].cuda(), 7.0), sinks=sinks, counts=tw.ints(lens))
    tw.near(x, want, tol, "first layer")
    t = make(B, G, H, D, D, T, lens, torch.bfloat16, seed=12)
    t["v"] = x[:, :, :, 0].cpu().contiguous()
    for b in range(B):
        t["v"][b, lens[b]:] = NAN
    want, tol, end, etol = reference(t, lens)
    o, s = attend(lh, t, lens)
    near(o, want, tol, "second layer")
    near(s, end, etol, "second layer's state")


def test_repeats_bit_for_bit(lh):
    t = make(2, 2, 1, 128, 128, 900, [900, 500], torch.bfloat16, seed=9)
    a, sa = attend(lh, t, [900, 500])
    for _ in range(3):
        b, sb = attend(lh, t, [900, 500])
        assert torch.equal(a, b) and torch.equal(sa, sb)


def test_graph_replays_follow_the_counts(lh):
    """A captured prompt and step: replays read the counts, states and tokens as they are
    then; eager work runs between them."""
    t = make(2, 2, 1, 128, 128, 800, None, torch.bfloat16, seed=21)
    d = on_gpu(t)
    one = on_gpu(step_inputs(2, 2, 1, 128, 128, torch.bfloat16, seed=22))
    counts = ints([800, 800])
    out = torch.zeros(2, 800, 2, 1, 128, dtype=torch.bfloat16, device="cuda")
    end, o1 = torch.zeros(2, 2, 1, 128, 128, device="cuda"), \
        torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(max(16, lh.linear_attention_workspace_bytes(2, 2, 1, 128, 128, 800)),
                     dtype=torch.uint8, device="cuda")

    def run():
        lh.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], out, end, ws,
                            counts=counts)
        lh.linear_attention_step(one["q"], one["k"], one["v"], one["log_decay"], end, o1)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    side = torch.randn(1 << 18, device="cuda")
    for cs in ([800, 0], [1, 64], [799, 333], [800, 800]):
        counts.copy_(torch.tensor(cs, dtype=torch.int32))
        d["state"].mul_(0.5)
        for o in (out, end, o1):
            o.zero_()
        run()
        torch.cuda.synchronize()
        ref = [o.clone() for o in (out, end, o1)]
        for o in (out, end, o1):
            o.zero_()
        side.mul_(1.0001)
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip((out, end, o1), ref):
            assert torch.equal(o, r), cs


def test_streams_at_once(lh):
    """Prompts and steps of different extents side by side, each on its own stream."""
    ts = [make(2, 2, 1, 128, 128, 900, None, torch.bfloat16, seed=31),
          make(3, 1, 2, 64, 96, 333, [333, 5, 100], torch.float16, seed=32)]
    counts = [None, [333, 5, 100]]
    want = [attend(lh, t, c) for t, c in zip(ts, counts)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(attend(lh, ts[i], counts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, s in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(s, want[i][1])


def test_past_four_gib(lh):
    """A state and tokens behind 4 GiB."""
    B, G, D = 66, 256, 256
    state = torch.zeros(B, G, 1, D, D, device="cuda")           # 4.4 GB
    state[-1, -1, 0] = 2.0
    q = torch.ones(B, G, 1, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(B, G, D, dtype=torch.bfloat16, device="cuda")
    k[-1, -1] = 1.0
    v = torch.ones(B, G, D, dtype=torch.bfloat16, device="cuda")
    ld = torch.full((G, 1), math.log(0.5), device="cuda")
    o = lh.linear_attention_step(q, k, v, ld, state, scale=0.25)
    # 0.5 * 2 + 1 = 2 within fp32's log of a half, 256 of them times a quarter
    assert torch.equal(o[-1, -1].float(), torch.full((1, D), 128.0, device="cuda"))
    assert not o[0].any() and abs(float(state[-1, -1, 0, -1, -1]) - 2.0) < 1e-6
    del state
    B, T, G = 1, 2100, 4200                                     # q, out 4.5 GB each
    q = torch.zeros(B, T, G, 1, D, dtype=torch.bfloat16, device="cuda")
    q[:, -1] = 1.0
    k = torch.zeros(B, T, G, 8 * 32, dtype=torch.bfloat16, device="cuda")
    k[:, -1, -1, 0] = 1.0
    v = torch.ones(B, T, G, D, dtype=torch.bfloat16, device="cuda")
    ld = torch.zeros(G, 1, device="cuda")
    o, end = lh.linear_attention(q, k, v, ld, scale=1.0)
    assert torch.equal(o[0, -1, -1, 0].float(), torch.ones(D, device="cuda"))
    assert not o[0, -1, 0].any() and not o[0, :-1].any()
    assert (end[0, -1, 0, 0] == 1).all() and not end[0, :-1].any()
