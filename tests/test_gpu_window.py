"""Attention over a sliding window and sinks (window_attention, window_decode)
against a plain implementation in 64 bits.

Tolerances (derived, not fitted).  With u = finfo(e).eps / 2, the largest relative
error of one rounding to the 16-bit type, and A = sum_j p_j |v_j|: the output is
rounded once (u |out|), and a kernel may round every p_j to 16 bits before its
product with v and divide by the sum of the rounded ones (2 u A to first order).  In
fp32 (eps/2 = 2^-24) a score of D products carries at most (D + 4) 2^-24 c sum |q k|
in the log2 domain (c = scale log2 e), doubled for MFMA accumulations that truncate;
twice that in a difference of scores, times ln 2, is the relative error E of every
p_j, to which sums of N positive terms add N 2^-24 at the very most and the
exponentials a few 2^-24.  f16 holds nothing below 2^-25, and the base of a running
maximum may lie up to 2^8 from the largest score: N 2^-25 max |v| more."""
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


def visible(p, window, sinks):
    """The keys that position p sees."""
    low = max(0, p - window + 1)
    return list(range(min(sinks, low, p + 1))) + list(range(low, p + 1))


def make(B, G, H, D, T, S, lens, counts, window, sinks, e, seed=0, std=1.0):
    """Inputs on the CPU; NaN in every slot that no row sees."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g).to(e)  # noqa: E731
    t = {"k": rnd(B, G, D, S), "v": rnd(B, G, S, D),
         "q": (torch.randn((B, T, G, H, D), generator=g) * std).to(e)}
    for b in range(B):
        n, c = clamp(lens[b], 0, S), T if counts is None else clamp(counts[b], 0, T)
        seen = set()
        for i in range(c):
            seen.update(visible(n - c + i, window, sinks))
        hidden = torch.tensor([j not in seen for j in range(S)])
        t["k"][b, :, :, hidden] = NAN
        t["v"][b, :, hidden] = NAN
        t["q"][b, c:] = NAN
    return t


def reference(t, lens, counts, window, sinks, scale=None):
    """out (7 in the rows behind a sequence) and its bound, in 64 bits."""
    q = t["q"].double()
    B, T, G, H, D = q.shape
    S = t["k"].shape[3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    e = t["q"].dtype
    u = torch.finfo(e).eps / 2
    out, tol = torch.full(q.shape, 7.0, dtype=torch.float64), torch.zeros_like(q)
    for b in range(B):
        n, c = clamp(lens[b], 0, S), T if counts is None else clamp(counts[b], 0, T)
        for i in range(c):
            at = torch.tensor(visible(n - c + i, window, sinks), dtype=torch.long)
            N = len(at)
            if N == 0:
                out[b, i] = 0
                continue
            k, v = t["k"][b][:, :, at].double(), t["v"][b][:, at].double()
            s = q[b, i] @ k * scale                              # G H N
            p = torch.softmax(s, -1)
            p = torch.where(torch.isnan(p) & (s.amax(-1, keepdim=True) == -math.inf), 0.0, p)
            qk = (q[b, i].abs() @ k.abs()).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
            E = 4 * math.log(2) * (D + 4) * 2.0 ** -24 * qk * scale * math.log2(math.e) \
                + (N + 16) * 2.0 ** -24
            A = p @ v.abs()
            out[b, i] = p @ v
            tol[b, i] = u * out[b, i].abs() + (2 * u * (1 + 4 * u) + 2 * E) * A \
                + (N * 2.0 ** -25 * v.abs().amax(1, keepdim=True) if e == torch.float16 else 0) \
                + 1e-30
    return out, tol


def near(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(),
                           float(err[bad].max()), float((err / tol)[bad].max()))
    _record(what, want.numel(), float(err.max()), 0.0, float((err / tol.clamp(min=1e-30)).max()))


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def attend(lh, t, lens, counts, window, sinks, scale=None, out=None, **kw):
    q = t["q"].cuda()
    out = torch.full_like(q, 7.0) if out is None else out
    got = lh.window_attention(t["k"].cuda(), t["v"].cuda(), q, ints(lens), window, out,
                              sinks=sinks, counts=ints(counts), scale=scale, **kw)
    assert got is out
    return got


def check(lh, what, B, G, H, D, T, S, lens, counts, window, sinks, e, seed=0, std=1.0, scale=None):
    print(what, B, G, H, D, T, S, lens[:6], counts and counts[:6], window, sinks, e, flush=True)
    t = make(B, G, H, D, T, S, lens, counts, window, sinks, e, seed, std)
    want, tol = reference(t, lens, counts, window, sinks, scale)
    got = attend(lh, t, lens, counts, window, sinks, scale)
    near(got, want, tol, f"{what} B{B} G{G} H{H} D{D} T{T} S{S} W{window}+{sinks} {e}")
    return t, got


SHAPES = [
    # B, G, H, D, T, S, lens, counts, window, sinks
    (1, 1, 1, 64, 1, 8, [1], None, 1, 0),
    (1, 1, 1, 8, 1, 8, [8], None, 3, 1),
    (1, 1, 32, 128, 1, 64, [64], None, 16, 4),
    (3, 2, 4, 128, 1, 136, [0, 64, 136], None, 40, 2),
    (3, 2, 4, 64, 1, 200, [200, 77, 130], [1, 0, 1], 64, 0),
    (2, 1, 71, 64, 1, 256, [128, 255], None, 100, 70),
    (1, 1, 16, 64, 5, 40, [40], None, 7, 2),
    (2, 2, 5, 80, 33, 200, [33, 200], None, 64, 1),
    (2, 1, 8, 128, 64, 192, [64, 150], [64, 1], 30, 0),
    (3, 2, 3, 96, 100, 333, [0, 50, 333], [0, 50, 100], 65, 4),
    (2, 1, 4, 256, 40, 264, [264, 100], None, 128, 8),
    (2, 4, 8, 128, 17, 1000, [1000, 600], None, 500, 4),
    (1, 2, 2, 40, 129, 301, [301], None, 1, 3),
    (2, 1, 12, 64, 70, 520, [520, 71], [70, 70], 1000, 5),
    (1, 1, 1, 128, 300, 300, [300], None, 128, 4),
    (4, 1, 2, 72, 9, 96, [-3, 1000, 5, 9], [9, 9, 9, 30], 20, 3),
    (2, 1, 129, 64, 3, 80, [9, 80], None, 33, 40),
    (17, 2, 7, 128, 2, 512, [30 * i for i in range(17)], None, 100, 4),
]


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s[:6])) for s in SHAPES])
def test_window(lh, shape, e):
    check(lh, "window", *shape, TYPES[e])


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (64, 64), (63, 65), (65, 63),
                                          (128, 200), (500, 0), (10 ** 9, 10 ** 9), (3, 500)])
def test_windows_and_sinks(lh, window, sinks, e):
    """Windows and sinks that begin and end at, before and behind the tiles' edges."""
    check(lh, "edges", 2, 2, 3, 64, 70, 328, [328, 131], [70, 66], window, sinks, TYPES[e])
    check(lh, "edges, one token", 3, 2, 8, 128, 1, 328, [328, 64, 65], None, window, sinks, TYPES[e])


@pytest.mark.parametrize("D", [8, 24, 64, 72, 96, 104, 128, 136, 200, 256])
@pytest.mark.parametrize("S", [256, 255, 250, 252])
def test_head_dims_and_odd_rows(lh, D, S):
    """Every head dim's tiles; K rows off 16-byte boundaries; the last slot decides."""
    e = torch.bfloat16 if S % 2 else torch.float16
    check(lh, "rows", 2, 1, 3, D, 40, S, [S, S - 30], None, 70, 5, e)
    check(lh, "rows, one token", 2, 1, 9, D, 1, S, [S, S - 30], None, 70, 5, e)


@pytest.mark.parametrize("e", TYPES)
def test_larger_tiles(lh, e):
    """As many rows as take the larger tiles and several of them, one head and many."""
    t = TYPES[e]
    check(lh, "one head", 2, 2, 1, 128, 600, 640, [640, 610], [600, 555], 200, 4, t)
    check(lh, "heads of 4", 2, 4, 4, 128, 260, 300, [300, 260], None, 100, 4, t)
    check(lh, "heads of 40", 1, 1, 40, 64, 50, 300, [300], None, 90, 0, t)
    check(lh, "many", 30, 2, 4, 64, 70, 136, [70 + 2 * i for i in range(30)],
          [70 - i for i in range(30)], 50, 2, t)
    check(lh, "wide", 1, 2, 4, 256, 200, 299, [299], None, 100, 4, t)


@pytest.mark.parametrize("e", TYPES)
def test_long_windows(lh, e):
    """Few rows over many keys: a row's keys are split and joined."""
    t = TYPES[e]
    check(lh, "long", 2, 1, 32, 128, 1, 9000, [9000, 4321], None, 8000, 4, t)
    check(lh, "long, few", 1, 2, 2, 64, 3, 20000, [19999], None, 20000, 0, t)
    check(lh, "long, odd", 1, 1, 5, 80, 4, 5001, [5001], None, 4000, 100, t)
    check(lh, "long beside short", 3, 1, 8, 256, 1, 5000, [5000, 0, 70], None, 3000, 16, t)


@pytest.mark.parametrize("e", TYPES)
def test_steep_scores(lh, e):
    """Scores far apart: the largest among the sinks, early and late in the window."""
    check(lh, "steep", 3, 2, 4, 128, 70, 300, [300, 100, 200], None, 150, 20, TYPES[e], std=12.0)
    check(lh, "flat", 3, 2, 4, 128, 70, 300, [300, 100, 200], None, 150, 20, TYPES[e], std=1e-3)
    check(lh, "scaled", 2, 1, 8, 64, 5, 200, [100, 200], None, 90, 3, TYPES[e], scale=0.7)


def test_infinite_scores(lh):
    """Keys of -inf score take no part; a row of nothing else is zero."""
    lens, W, sinks = [96, 50], 30, 4
    t = make(2, 1, 4, 64, 20, 96, lens, None, W, sinks, torch.bfloat16, seed=5)
    t["q"] = t["q"].abs() + 0.1
    t["k"][0, 0, :, 60:80] = -math.inf      # all that a few rows see beside the sinks
    t["k"][0, 0, :, :2] = -math.inf
    want, tol = reference(t, lens, None, W, sinks)
    near(attend(lh, t, lens, None, W, sinks), want, tol, "-inf keys")
    t["k"][0] = -math.inf
    got = attend(lh, t, lens, None, W, sinks)
    assert torch.equal(got[0].float().cpu(), torch.zeros(20, 1, 4, 64))
    assert torch.isfinite(got[1].float()).all()


@pytest.mark.parametrize("T,H", [(50, 1), (50, 3), (130, 4), (7, 8), (300, 1)])
def test_what_a_row_does_not_see_does_not_reach_it(lh, T, H):
    """NaN and infinities in K and V of single keys reach the rows that see them and
    no others, whatever tile these share."""
    S, W, sinks, D, c = 400, 60, 3, 64, T
    lens = [S - 5]
    t = make(1, 2, H, D, T, S, lens, None, W, sinks, torch.bfloat16, seed=T)
    n, first = S - 5, S - 5 - T
    for at, which, value, col in ((n - c // 2, "v", math.inf, 5), (n - c // 3, "v", NAN, 9),
                                  (max(0, first - W // 2), "v", -math.inf, 20),
                                  (1, "v", NAN, 33)):
        t[which][0, 1, at, col] = value
    t["k"][0, 0, 7, n - c // 4] = NAN
    t["k"][0, 0, 9, max(0, first - W // 3)] = NAN
    want, tol = reference(t, lens, None, W, sinks)
    got = attend(lh, t, lens, None, W, sinks).double().cpu()
    # finite where the formula is, within the bound; not finite where it is not
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    zero = torch.zeros_like(want)
    near(torch.where(fine, got, zero), torch.where(fine, want, zero),
         torch.where(fine, tol, zero), "beside infinities")


def test_arguments(lh):
    """Outputs and workspaces given, out on q, a step as both calls make it."""
    lens, W, sinks = [500, 333], 300, 4
    t = make(2, 2, 4, 64, 1, 504, lens, None, W, sinks, torch.bfloat16, seed=7)
    ref = attend(lh, t, lens, None, W, sinks)
    k, v, q = (t[x].cuda() for x in "kvq")
    need = lh.window_attention_workspace_bytes(2, 2, 4, 64, 1, 504, W, sinks)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    got = lh.window_decode(k, v, q[:, 0].contiguous(), ints(lens), W, workspace=ws, sinks=sinks)
    assert torch.equal(got, ref[:, 0])
    if need:
        with pytest.raises(ValueError, match="workspace needs"):
            lh.window_attention(k, v, q, ints(lens), W, workspace=ws[:need - 1], sinks=sinks)
    lh.window_attention(k, v, q, ints(lens), W, q, sinks=sinks)      # out on q
    assert torch.equal(q, ref)


@pytest.mark.parametrize("T,W", [(200, 100), (2, 600)])
def test_out_on_q(lh, T, W):
    lens = [700, 650]
    t = make(2, 1, 3, 128, T, 704, lens, None, W, 4, torch.float16, seed=8)
    ref = attend(lh, t, lens, None, W, 4)
    q = t["q"].cuda()
    lh.window_attention(t["k"].cuda(), t["v"].cuda(), q, ints(lens), W, q, sinks=4)
    assert torch.equal(q, ref)


def test_matches_the_framework_s_other_attention(lh):
    """A window of all keys is causal attention; one token's is a decoding step."""
    B, G, H, D, T = 2, 2, 1, 64, 192
    t = make(B, G, H, D, T, T, [T, T], None, T, 0, torch.bfloat16, seed=9)
    got = attend(lh, t, [T, T], None, T, 0)
    k, v = t["k"].cuda(), t["v"].cuda()
    q = t["q"].cuda()
    full = lh.attention(k.view(B * G, D, T), v.view(B * G, T, D),
                        q[:, :, :, 0].permute(0, 2, 1, 3).reshape(B * G, T, D).contiguous(),
                        causal=True)
    want, tol = reference(t, [T, T], None, T, 0)
    near(got, want, tol, "window of all keys")
    # (attention rounds the scaled q to 16 bits too: u times the largest score)
    u, top = 2.0 ** -8, 8.0
    near(full.view(B, G, T, D).permute(0, 2, 1, 3).unsqueeze(3), want,
         tol + 2 * u * top * t["v"].double().abs().max(), "attention")
    last = lh.cache_decode(k, v, q[:, -1].contiguous(), ints([T, T]))
    near(last.unsqueeze(1), want[:, -1:], tol[:, -1:], "cache_decode")


def test_repeats_bit_for_bit(lh):
    lens = [640, 100, 333]
    t = make(3, 2, 4, 128, 50, 640, lens, None, 300, 4, torch.bfloat16, seed=9)
    a = attend(lh, t, lens, None, 300, 4)
    for _ in range(3):
        assert torch.equal(torch.nan_to_num(attend(lh, t, lens, None, 300, 4)), torch.nan_to_num(a))


@pytest.mark.parametrize("T", [1, 40])
def test_past_four_gib(lh, T):
    """Keys whose K and V lie behind 4 GiB decide the rows that see them."""
    B, D, S, W = 2, 256, 5 << 20, 100
    k = torch.zeros(B, 1, D, S, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(B, 1, S, D, dtype=torch.bfloat16, device="cuda")
    n = [S, S - 67]
    q = torch.ones(B, T, 1, 2, D, dtype=torch.bfloat16, device="cuda")
    for b in range(B):
        k[b, 0, :, n[b] - T - 3] = 2.0      # score 32 above the others
        v[b, 0, n[b] - T - 3] = float(b + 1)
        if n[b] < S:
            v[b, 0, n[b]:] = NAN
        v[b, 0, 10:n[b] - T - W] = 100.0
    out = lh.window_attention(k, v, q, ints(n), W, sinks=3)
    for b in range(B):
        # the others' share: at most 103 exp(-32)
        assert torch.equal(out[b].float(), torch.full_like(out[b].float(), float(b + 1)))


# ---- together, and where programs run them ---------------------------------------

def test_prompt_and_steps_agree(lh):
    """A ragged prompt and steps, appended and attended to, against the whole; then
    on caches cut to what the window sees."""
    B, G, H, D, S, W, sinks, steps, T = 3, 2, 4, 64, 160, 40, 4, 12, 90
    g = torch.Generator().manual_seed(3)
    counts = [90, 31, 77]
    total = [c + steps for c in counts]
    rnd = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16)  # noqa: E731
    ks, vs, qs = rnd(B, T + steps, G, D), rnd(B, T + steps, G, D), rnd(B, T + steps, G, H, D)
    whole = {"k": torch.zeros(B, G, D, S, dtype=torch.bfloat16),
             "v": torch.zeros(B, G, S, D, dtype=torch.bfloat16), "q": qs}
    for b in range(B):
        whole["k"][b, :, :, :total[b]] = ks[b, :total[b]].permute(1, 2, 0)
        whole["v"][b, :, :total[b]] = vs[b, :total[b]].permute(1, 0, 2)
    want, tol = reference(whole, total, total, W, sinks)
    k = torch.full((B, G, D, S), NAN, dtype=torch.bfloat16, device="cuda")
    v = torch.full((B, G, S, D), NAN, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(B, G, S, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    cut = lambda x: x[:, :T].cuda()  # noqa: E731
    lens = lh.cache_append(k, v, lens, cut(ks), cut(vs), counts=ints(counts))
    out = lh.window_attention(k, v, cut(qs), lens, W, sinks=sinks, counts=ints(counts))
    for b in range(B):
        near(out[b, :counts[b]], want[b, :counts[b]], tol[b, :counts[b]], "prompt")
    at = torch.arange(B)
    for i in range(steps):
        x = torch.tensor(counts) + i
        lens = lh.cache_append(k, v, lens, ks[at, x].unsqueeze(1).cuda(),
                               vs[at, x].unsqueeze(1).cuda())
        out = lh.window_decode(k, v, qs[at, x].cuda(), lens, W, sinks=sinks)
        near(out, want[at, x], tol[at, x], f"step {i}")
        if i == 5:     # what lies before the window is let go: the slots move, the keys stay
            k, v, w, lens, _ = lh.cache_evict(k, v, w, lens, W + sinks, recent=W, sinks=sinks,
                                              capacity=S)


def test_graph_replays_follow_the_lengths(lh):
    """Captured calls, with and without splits: replays read the lengths, counts and
    caches as they are then; eager work runs between them."""
    B, G, H, D, S, T = 3, 2, 4, 128, 1000, 20
    t = make(B, G, H, D, T, S, [S] * B, None, S, 0, torch.bfloat16, seed=31)
    k, v, q = (t[x].cuda() for x in "kvq")
    lens, counts = ints([S] * B), ints([T] * B)
    one = q[:, 0].contiguous()
    o1, o2 = torch.zeros_like(one), torch.zeros_like(q)
    ws = [torch.empty(max(16, lh.window_attention_workspace_bytes(B, G, H, D, x, S, 900, 4)),
                      dtype=torch.uint8, device="cuda") for x in (1, T)]

    def run():
        lh.window_decode(k, v, one, lens, 900, o1, ws[0], sinks=4)
        lh.window_attention(k, v, q, lens, 900, o2, ws[1], sinks=4, counts=counts)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    side = torch.randn(1 << 18, device="cuda")
    for ls, cs in (([1000, 0, 37], [20, 0, 20]), ([999, 64, 500], [1, 2, 3]), ([S] * B, [T] * B)):
        lens.copy_(torch.tensor(ls, dtype=torch.int32))
        counts.copy_(torch.tensor(cs, dtype=torch.int32))
        for o in (o1, o2):
            o.zero_()
        run()
        torch.cuda.synchronize()
        ref = [o1.clone(), o2.clone()]
        for o in (o1, o2):
            o.zero_()
        side.mul_(1.0001)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, ref[0]) and torch.equal(o2, ref[1]), ls


def test_threads_on_their_own_streams(lh):
    """Host threads, each with its stream, caches and sizes: the results of calls
    made alone, bit for bit."""
    import threading
    cases = [(2, 2, 8, 128, 1, 4000, [4000, 1234], 3000), (1, 2, 4, 64, 300, 512, [512], 100),
             (3, 1, 5, 80, 30, 333, [333, 30, 200], 90)]
    d = []
    for i, (B, G, H, D, T, S, lens, W) in enumerate(cases):
        t = make(B, G, H, D, T, S, lens, None, W, 4, torch.bfloat16, seed=60 + i)
        d.append(({x: t[x].cuda() for x in "kvq"}, ints(lens), W))

    def work(i):
        t, lens, W = d[i]
        return lh.window_attention(t["k"], t["v"], t["q"], lens, W, sinks=4)

    want = [work(i) for i in range(len(d))]
    torch.cuda.synchronize()
    got, errors = [[] for _ in d], []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(8):
                    got[i].append(work(i))
            s.synchronize()
        except Exception as e:      # noqa: BLE001  (reported by the test)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(d))]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not errors, errors
    for i in range(len(d)):
        for r in got[i]:
            assert torch.equal(r, want[i])


@pytest.mark.parametrize("H,T", [(40, 9), (64, 5), (130, 3)])
def test_infinities_between_waves_of_one_tile(lh, H, T):
    """Rows of a wave that all are one token's, beside waves of others in the tile: an
    infinity that only these see stays with them."""
    S, W, D = 300, 50, 64
    t = make(1, 1, H, D, T, S, [S], None, W, 2, torch.bfloat16, seed=H)
    t["v"][0, 0, S - 1, 5] = math.inf              # the last token sees it
    t["v"][0, 0, S - T - W + 1, 9] = -math.inf     # the first does
    want, tol = reference(t, [S], None, W, 2)
    got = attend(lh, t, [S], None, W, 2).double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and not fine.all()
    zero = torch.zeros_like(want)
    near(torch.where(fine, got, zero), torch.where(fine, want, zero),
         torch.where(fine, tol, zero), "beside infinities of other waves")


@pytest.mark.parametrize("S", [264, 261])
@pytest.mark.parametrize("D,H,rows", [(128, 4, 256), (64, 4, 256), (96, 4, 256), (256, 2, 128),
                                      (128, 2, 128), (64, 2, 128), (80, 2, 128), (128, 1, 64),
                                      (56, 1, 64), (88, 1, 64), (200, 1, 32)])
def test_every_tile(lh, D, H, rows, S):
    """64 (b, g)s: as many rows as the tiles of 64, 128 and 256 are taken for, K's rows on
    and off 16-byte boundaries, padded batches, infinities that some rows see."""
    B, G, T, W, sinks = 8, 8, 256, 70, 3
    e = torch.bfloat16 if D % 64 else torch.float16
    assert H * T >= 4 * rows
    lens = [S - b for b in range(B)]
    counts = [T - 5 * b - (b == 3) * 200 for b in range(B)]
    print("tile", D, H, rows, S, flush=True)
    t = make(B, G, H, D, T, S, lens, counts, W, sinks, e, D)
    t["v"][2, 3, 150, 5] = math.inf
    t["v"][1, 7, 1, 9] = NAN
    want, tol = reference(t, lens, counts, W, sinks)
    got = attend(lh, t, lens, counts, W, sinks).double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and not fine.all()
    zero = torch.zeros_like(want)
    near(torch.where(fine, got, zero), torch.where(fine, want, zero),
         torch.where(fine, tol, zero), f"tile of {rows} D{D} S{S}")


def test_many_heads_in_large_tiles(lh):
    """71 heads: tokens that begin and end inside a tile and inside a wave's rows."""
    check(lh, "71 heads", 64, 1, 71, 64, 15, 100, [100 - b for b in range(64)],
          [15 - b % 7 for b in range(64)], 40, 2, torch.bfloat16)
