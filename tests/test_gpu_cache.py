"""The cache operators (append, decode with a shared prefix and gathered weights,
evict) against plain implementations: moves bit for bit, a decoding step against
64 bits.

Tolerances of a step (derived, not fitted).  With u = finfo(e).eps / 2, the
largest relative error of one rounding to the 16-bit type, and A = sum_j p_j
|v_j|: the output is rounded once (u |out|), and a kernel may round every p_j to
16 bits before its product with v, and sum the rounded ones (2 u A to first
order).  In fp32 (eps/2 = 2^-24) a score of D products carries at most
(D + 4) 2^-24 c sum |q k| in the log2 domain (c = scale log2 e), doubled for
MFMA accumulations that truncate; twice that in a difference of scores, times
ln 2, is the relative error E of every p_j, to which sums of N positive terms add
N 2^-24 at the very most and the exponentials a few 2^-24.
f16 holds nothing below 2^-25, and the base of a running maximum may lie up to
2^8 from the largest score: N 2^-25 max |v| more."""
import math

import pytest
import torch

from tests.conftest import assert_close_gpu  # noqa: F401  (its error list is printed)

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def lh():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import loom_hip
    return loom_hip


def make(B, G, H, D, P, S, lens, e, seed=0, std=1.0):
    """Inputs of a step on the CPU; NaN in every slot behind a length."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g).to(e)  # noqa: E731
    t = {"k": rnd(B, G, D, S), "v": rnd(B, G, S, D), "q": (torch.randn((B, G, H, D), generator=g)
                                                           * std).to(e),
         "lens": torch.tensor(lens, dtype=torch.int32),
         "weights": torch.rand((B, G, S), generator=g),
         "prefix_k": rnd(G, D, P) if P else None, "prefix_v": rnd(G, P, D) if P else None}
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        t["k"][b, :, :, n:] = float("nan")
        t["v"][b, :, n:] = float("nan")
    return t


def reference(t, scale=None):
    """out, weights added, and the bounds of both, in 64 bits."""
    k, v, q = (t[x].double() for x in ("k", "v", "q"))
    B, G, H, D = q.shape
    S = k.shape[3]
    P = 0 if t["prefix_k"] is None else t["prefix_k"].shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    e = t["q"].dtype
    u = torch.finfo(e).eps / 2
    out, otol = torch.zeros(B, G, H, D, dtype=torch.float64), torch.zeros(B, G, H, D,
                                                                         dtype=torch.float64)
    w, wtol = torch.zeros(B, G, S, dtype=torch.float64), torch.zeros(B, G, S, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(t["lens"][b]), 0), S)
        for g in range(G):
            keys, vals = k[b, g, :, :n], v[b, g, :n]
            if P:
                keys = torch.cat([t["prefix_k"][g].double(), keys], 1)
                vals = torch.cat([t["prefix_v"][g].double(), vals], 0)
            N = keys.shape[1]
            if N == 0:
                continue
            s = q[b, g] @ keys * scale
            p = torch.softmax(s, -1)
            p = torch.where(torch.isnan(p) & (s.amax(-1, keepdim=True) == -math.inf), 0.0, p)
            absqk = (q[b, g].abs() @ keys.abs()).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
            E = 4 * math.log(2) * (D + 4) * 2.0 ** -24 * absqk * scale * math.log2(math.e) \
                + (N + 16) * 2.0 ** -24
            o = p @ vals
            A = p @ vals.abs()
            out[b, g] = o
            otol[b, g] = u * o.abs() + (2 * u * (1 + 4 * u) + 2 * E) * A \
                + (N * 2.0 ** -25 * vals.abs().amax(0) if e == torch.float16 else 0) + 1e-30
            pn = p[:, P:]
            w[b, g, :n] = pn.sum(0)
            wtol[b, g, :n] = (2 * E * pn).sum(0) + H * 2.0 ** -24 * pn.sum(0)
    return out, otol, w, wtol


def near(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float((err / tol)[bad].max()))
    from tests.conftest import _record
    _record(what, want.numel(), float(err.max()), 0.0, float((err / tol.clamp(min=1e-30)).max()))


def step(lh, t, weights=True, into=None, scale=None, **kw):
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    w = d["weights"].clone() if weights else None
    o = lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], prefix_k=d["prefix_k"],
                        prefix_v=d["prefix_v"], weights=w, weights_out=into, scale=scale, **kw)
    return o, w


def check(lh, what, B, G, H, D, P, S, lens, e, weights=True, seed=0, std=1.0, scale=None):
    print(what, B, G, H, D, P, S, lens[:6], e, weights, flush=True)
    t = make(B, G, H, D, P, S, lens, e, seed, std)
    out, otol, w, wtol = reference(t, scale)
    o, wo = step(lh, t, weights, scale=scale)
    near(o, out, otol, f"{what} out B{B} G{G} H{H} D{D} P{P} S{S} {e}")
    if weights:
        total = t["weights"].double() + w
        near(wo, total, wtol + 2.0 ** -23 * total.abs(), f"{what} weights B{B} G{G} H{H} D{D} P{P}")
        for b, n in enumerate(lens):         # behind a length: untouched
            n = min(max(n, 0), S)
            assert torch.equal(wo[b, :, n:].cpu(), t["weights"][b, :, n:])


SHAPES = [
    # B, G, H, D, P, S, lens: from one key to several tiles, odd sizes
    (1, 1, 1, 64, 0, 8, [1]),
    (1, 1, 32, 128, 0, 64, [64]),
    (2, 1, 32, 128, 0, 192, [65, 191]),
    (3, 1, 8, 64, 1, 40, [0, 1, 40]),
    (3, 2, 4, 128, 64, 136, [0, 64, 136]),
    (2, 2, 5, 80, 63, 200, [7, 200]),
    (2, 1, 71, 64, 129, 256, [128, 255]),
    (5, 1, 32, 128, 333, 264, [0, 8, 63, 64, 264]),
    (2, 1, 48, 96, 1000, 72, [3, 72]),
    (4, 4, 8, 128, 2048, 64, [1, 2, 33, 64]),
    (40, 1, 16, 64, 520, 16, list(range(0, 17)) + [16] * 23),
    (2, 2, 12, 256, 100, 320, [100, 319]),
    (1, 1, 40, 256, 0, 1024, [1000]),
    (2, 1, 129, 64, 24, 80, [9, 80]),
    (1, 1, 200, 128, 100, 160, [159]),
    (17, 2, 7, 128, 700, 512, [30 * i for i in range(17)]),
    (1, 8, 4, 8, 16, 48, [48]),
    (2, 1, 3, 40, 17, 24, [20, 24]),
]


@pytest.mark.parametrize("e", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s[:6])) for s in SHAPES])
def test_decode(lh, shape, e):
    for weights in (False, True):
        check(lh, "step", *shape, TYPES[e], weights)


@pytest.mark.parametrize("e", TYPES)
def test_decode_shapes_of_a_launch(lh, e):
    """The larger ways a step is laid out: prefix tiles of 128 rows, own tiles of
    64 and 128, several rows to a joining workgroup, weights in parts of 256
    keys, heads past 256, more than 256 sequences."""
    t = TYPES[e]
    check(lh, "128-row tiles", 33, 1, 31, 64, 16500, 72, [2 * b for b in range(33)], t)
    check(lh, "128-row tiles, odd", 18, 4, 29, 64, 4099, 40, [2 * b for b in range(18)], t,
          weights=False)
    check(lh, "joined rows", 70, 4, 8, 80, 33, 40, [(7 * b) % 41 for b in range(70)], t)
    check(lh, "joined rows, one part", 129, 2, 8, 128, 0, 64, [(7 * b) % 65 for b in range(129)], t)
    check(lh, "parts of 256", 16, 2, 33, 64, 5, 2100, [131 * b for b in range(16)], t)
    check(lh, "wide heads", 2, 1, 300, 64, 70, 520, [519, 64], t)
    check(lh, "heads of 64", 5, 1, 64, 128, 130, 1001, [0, 250, 500, 750, 1001], t)
    check(lh, "heads of 71", 3, 1, 71, 128, 131, 501, [0, 250, 501], t)


@pytest.mark.parametrize("e", TYPES)
def test_decode_weights_of_many_keys(lh, e):
    """512 and 1024 keys to a workgroup that gathers weights: several of them to a
    sequence, lengths at their ends, one to many heads."""
    t = TYPES[e]
    lens = [0, 1, 511, 512, 513, 1023, 1024, 1025, 1100, 256, 255, 257]
    check(lh, "parts of 512", 24, 4, 5, 16, 0, 1100, [lens[b % 12] for b in range(24)], t)
    check(lh, "parts of 512, heads", 100, 1, 33, 16, 9, 1540, [lens[b % 12] + 436 for b in range(100)], t)
    check(lh, "parts of 1024", 64, 8, 1, 8, 0, 1101, [lens[b % 12] for b in range(64)], t)
    check(lh, "parts of 1024, heads", 173, 3, 19, 8, 7, 1025, [lens[b % 12] for b in range(173)], t)
    check(lh, "parts of 1024, many heads", 520, 1, 257, 8, 0, 1032, [lens[b % 12] for b in range(520)], t)


def test_decode_caches_past_the_last_level_cache(lh):
    check(lh, "large caches", 2, 1, 8, 128, 100, 300000, [300000, 123457], torch.bfloat16)
    check(lh, "large caches, odd", 2, 1, 8, 128, 0, 300001, [300001, 64], torch.float16)


@pytest.mark.parametrize("S", [2047, 2044, 2046])
@pytest.mark.parametrize("P", [0, 515, 1021])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_odd_rows(lh, S, P, D):
    """K rows off 16-byte boundaries; lengths that reach the last slot."""
    check(lh, "odd rows", 2, 1, 9, D, P, S, [S, S - 700], torch.bfloat16)


def test_decode_long_rows(lh):
    """Sequences that take many splits beside ones that take none."""
    check(lh, "long", 3, 1, 32, 128, 0, 30000, [30000, 0, 77], torch.bfloat16)
    check(lh, "long prefix", 2, 1, 32, 128, 40000, 64, [0, 64], torch.bfloat16)
    check(lh, "many", 300, 1, 4, 64, 65, 136, [(37 * i) % 137 for i in range(300)], torch.float16)


@pytest.mark.parametrize("e", TYPES)
def test_decode_steep_scores(lh, e):
    """Scores far apart: the largest anywhere, in the prefix or the cache."""
    check(lh, "steep", 3, 2, 8, 128, 300, 200, [0, 100, 200], TYPES[e], std=12.0)
    check(lh, "flat", 3, 2, 8, 128, 300, 200, [0, 100, 200], TYPES[e], std=1e-3)
    check(lh, "scaled", 2, 1, 8, 64, 70, 200, [100, 200], TYPES[e], scale=0.7)


def test_decode_lengths_out_of_range(lh):
    """Lengths below 0 and above S count as 0 and S."""
    check(lh, "clamped", 3, 1, 4, 64, 20, 96, [-5, 1000, 2 ** 31 - 1], torch.bfloat16)


def test_decode_no_keys(lh):
    check(lh, "empty", 3, 2, 4, 64, 0, 64, [0, 5, 0], torch.bfloat16)
    check(lh, "all empty", 2, 1, 33, 128, 0, 64, [0, 0], torch.float16)


def test_decode_infinite_scores(lh):
    """Keys of -inf score take no part; a row of nothing else is zero."""
    t = make(2, 1, 4, 64, 40, 96, [96, 50], torch.bfloat16, seed=5)
    t["q"] = t["q"].abs() + 0.1
    t["k"][0, 0, :, :70] = -math.inf        # the first keys of a cache
    t["prefix_k"][0, :, 8:] = -math.inf     # the last of the prefix
    out, otol, w, wtol = reference(t)
    o, wo = step(lh, t)
    near(o, out, otol, "-inf keys")
    near(wo, t["weights"].double() + w, wtol + 2.0 ** -22, "-inf weights")
    t["prefix_k"][:] = -math.inf
    t["k"][0] = -math.inf
    o, wo = step(lh, t)
    assert torch.equal(o[0].float().cpu(), torch.zeros(1, 4, 64))
    assert torch.equal(wo[0].cpu(), t["weights"][0])
    assert torch.isfinite(o[1].float()).all()


def test_decode_nan_and_inf_values_reach_their_rows_only(lh):
    t = make(2, 2, 4, 64, 16, 40, [40, 33], torch.bfloat16, seed=6)
    t["v"][0, 1, 3, 7] = math.nan
    t["k"][1, 0, 5, 8] = math.nan
    o, wo = step(lh, t)
    bad = torch.isnan(o.float().cpu())
    want = torch.zeros_like(bad)
    want[0, 1, :, 7] = True                 # one column of one head
    want[1, 0] = True                       # a NaN score: the whole row
    assert torch.equal(bad, want)
    bad = torch.isnan(wo.cpu())
    assert bad[1, 0, :33].all() and not bad[0].any() and not bad[1, 1].any()
    assert not bad[1, 0, 33:].any()


def test_decode_infinite_values(lh):
    """An infinity in the last key's V: the masked keys behind it add nothing."""
    for n, H in ((33, 4), (5, 40), (97, 71)):
        t = make(1, 1, H, 64, 0, 104, [n], torch.bfloat16, seed=n)
        t["v"][0, 0, n - 1, 3] = math.inf
        t["v"][0, 0, n - 1, 9] = -math.inf
        o, _ = step(lh, t)
        o = o.float().cpu()
        assert (o[..., 3] == math.inf).all() and (o[..., 9] == -math.inf).all()
        o[..., 3] = o[..., 9] = 0
        assert torch.isfinite(o).all()


def test_decode_arguments(lh):
    """Outputs and workspace given, an empty prefix tensor, weights elsewhere."""
    t = make(2, 2, 4, 64, 0, 40, [40, 33], torch.bfloat16, seed=7)
    ref, wref = step(lh, t)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    out = torch.full((2, 2, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    into = torch.full((2, 2, 40), 9.0, device="cuda")
    ws = lh.cache_decode_workspace(2, 2, 4, 64, 0, 40, True, "cuda:0")
    ws.fill_(255)
    got = lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], out, ws, weights=d["weights"],
                          weights_out=into,
                          prefix_k=torch.empty(2, 64, 0, dtype=torch.bfloat16, device="cuda"),
                          prefix_v=torch.empty(2, 0, 64, dtype=torch.bfloat16, device="cuda"))
    assert got is out and torch.equal(out, ref)
    for b, n in enumerate([40, 33]):
        assert torch.equal(into[b, :, :n], wref[b, :, :n])
        assert (into[b, :, n:] == 9.0).all()
    assert torch.equal(d["weights"].cpu(), t["weights"])     # only read
    with pytest.raises(ValueError, match="workspace needs"):
        lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], out, ws[:16])
    with pytest.raises(RuntimeError, match="scale"):
        lh.cache_decode(d["k"], d["v"], d["q"], d["lens"], scale=0.0)


def test_decode_matches_flash_decode(lh):
    """One KV head, full caches: the framework's other decoding step."""
    t = make(4, 1, 32, 128, 0, 1024, [1024] * 4, torch.bfloat16, seed=8)
    o, _ = step(lh, t, weights=False)
    f = lh.flash_decode(t["k"][:, 0].cuda(), t["v"][:, 0].cuda(), t["q"][:, 0].cuda())
    out, otol, _, _ = reference(t)
    near(o, out, otol, "step")
    near(f.unsqueeze(1), out, otol, "flash_decode")


def test_decode_repeats_bit_for_bit(lh):
    t = make(6, 2, 8, 128, 777, 640, [640, 0, 100, 333, 64, 1], torch.bfloat16, seed=9)
    a, wa = step(lh, t)
    for _ in range(3):
        b, wb = step(lh, t)
        assert torch.equal(a, b) and torch.equal(wa, wb)


def test_decode_past_four_gib(lh):
    """A key whose K and V lie behind 4 GiB decides the row."""
    B, D, S = 3, 256, 4 << 20
    k = torch.zeros(B, 1, D, S, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(B, 1, S, D, dtype=torch.bfloat16, device="cuda")
    n = [S, 5, S - 3]
    q = torch.ones(B, 1, 2, D, dtype=torch.bfloat16, device="cuda")
    for b in range(B):
        k[b, 0, :, n[b] - 1] = 2.0          # score 32 above the others
        v[b, 0, n[b] - 1] = float(b + 1)
        if n[b] < S:
            v[b, 0, n[b]:] = math.nan
    w = torch.zeros(B, 1, S, device="cuda")
    o = lh.cache_decode(k, v, q, torch.tensor(n, dtype=torch.int32, device="cuda"), weights=w)
    for b in range(B):
        # the others' share: at most S exp(-32) = 5.4e-8
        assert torch.equal(o[b].float(), torch.full_like(o[b].float(), float(b + 1)))
        assert abs(float(w[b, 0, n[b] - 1]) - 2.0) < 1e-5


# ---- eviction -----------------------------------------------------------------

def order(x):
    return [(-math.inf, 0) if math.isnan(v) else (v, 1) for v in x]


def kept(w, n, keep, recent, sinks):
    if n <= keep:
        return list(range(n))
    o = order(w[:n].tolist())
    middle = sorted(range(sinks, n - recent), key=lambda i: (o[i], -i), reverse=True)
    return sorted(list(range(sinks)) + list(range(n - recent, n))
                  + middle[:keep - sinks - recent])


def evict_check(lh, B, G, D, S, So, lens, keep, recent, sinks, e=torch.bfloat16, w=None, seed=0):
    print("evict", B, G, D, S, So, lens[:6], keep, recent, sinks, e, flush=True)
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((B, G, D, S), generator=g).to(e)
    v = torch.randn((B, G, S, D), generator=g).to(e)
    if w is None:
        w = torch.exp(2 * torch.randn((B, G, S), generator=g))
    for b, n in enumerate(lens):
        w[b, :, max(n, 0):] = math.nan
    ko, vo = torch.full((B, G, D, So), 7.0, dtype=e), torch.full((B, G, So, D), 7.0, dtype=e)
    wo = torch.full((B, G, So), 7.0)
    got = lh.cache_evict(k.cuda(), v.cuda(), w.cuda(),
                         torch.tensor(lens, dtype=torch.int32).cuda(), keep, recent=recent,
                         sinks=sinks, k_out=ko.cuda(), v_out=vo.cuda(), weights_out=wo.cuda())
    index = torch.full((B, G, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        for h in range(G):
            at = kept(w[b, h], n, keep, recent, sinks)
            i, m = torch.tensor(at, dtype=torch.long), len(at)
            index[b, h, :m] = i.int()
            ko[b, h, :, :m] = k[b, h][:, i]
            vo[b, h, :m] = v[b, h][i]
            wo[b, h, :m] = w[b, h][i]
    assert torch.equal(got[4].cpu(), index)
    assert torch.equal(got[3].cpu(), torch.tensor([min(max(n, 0), S, keep) if n >= 0 else 0
                                                   for n in lens], dtype=torch.int32))
    bits = lambda x: x.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(got[0].cpu()), bits(ko))
    assert torch.equal(bits(got[1].cpu()), bits(vo))
    assert torch.equal(got[2].cpu().view(torch.int32), wo.view(torch.int32))


@pytest.mark.parametrize("case", [
    # B, G, D, S, So, lens, keep, recent, sinks
    (1, 1, 64, 8, 8, [8], 1, 0, 0), (1, 1, 64, 8, 8, [8], 1, 1, 0),
    (1, 1, 64, 8, 8, [8], 1, 0, 1), (2, 1, 64, 64, 16, [64, 17], 16, 4, 2),
    (3, 2, 128, 200, 100, [0, 100, 101], 100, 10, 4), (2, 2, 80, 333, 129, [333, 129], 128, 60, 4),
    (2, 1, 256, 1000, 501, [999, 3], 500, 0, 0), (1, 3, 96, 4097, 1024, [4097], 1024, 1000, 24),
    (1, 1, 128, 9001, 9000, [9001], 9000, 1, 1), (2, 1, 64, 5000, 3001, [4999, 5000], 2999, 7, 3),
    (4, 1, 8, 77, 30, [-3, 1000, 31, 30], 30, 3, 3), (1, 1, 64, 70000, 30000, [69999], 30000, 9, 0),
    (65, 2, 16, 150, 60, [(11 * i) % 151 for i in range(65)], 50, 5, 1),
    # kept slots far apart (several windows of a row), and ever closer
    (1, 1, 64, 70000, 704, [69999], 600, 9, 0), (1, 1, 40, 70001, 701, [70001], 600, 9, 0),
    (1, 2, 64, 16384, 2049, [16383], 2048, 0, 0), (1, 2, 64, 16377, 3000, [16377], 2999, 0, 0),
    (1, 1, 72, 8192, 6000, [8192], 5555, 100, 4),
    (3, 1, 64, 12288, 600, [12288, 700, 4097], 599, 5, 4), (2, 1, 24, 9000, 90, [9000, 8999], 77, 0, 0),
    # weights in registers up to 32768 slots, read again past them
    (2, 1, 16, 20001, 5000, [20001, 16385], 4999, 100, 4),
    (2, 1, 8, 32768, 32000, [32768, 32767], 31999, 0, 3),
    (2, 1, 8, 32769, 40, [32769, 1500], 40, 9, 9), (1, 1, 8, 263000, 100, [262145], 99, 0, 0),
], ids=lambda c: "x".join(map(str, c[:5])) + f"-{c[6]}")
def test_evict(lh, case):
    for e in TYPES.values():
        evict_check(lh, *case, e=e)


def test_evict_ties_and_odd_weights(lh):
    """Equal weights (the lowest slots stay), zeros of both signs, negative
    weights, infinities, NaN."""
    S = 700
    evict_check(lh, 1, 1, 64, S, S, [S], 300, 10, 5, w=torch.zeros(1, 1, S))
    g = torch.Generator().manual_seed(3)
    w = torch.randint(-2, 3, (2, 2, S), generator=g).float()
    w[0, 0, ::3] = -0.0
    evict_check(lh, 2, 2, 64, S, 400, [S, 600], 299, 10, 5, w=w.clone())
    w[0, 1, 50:90] = math.inf
    w[1, 0, 20:300] = -math.inf
    w[1, 1, 7:500] = math.nan
    w[0, 0] = math.nan
    for keep in (20, 299, 400):
        evict_check(lh, 2, 2, 64, S, 400, [S, 600], keep, 10, 5, w=w.clone())
    for S2 in (30000, 40000):     # ties over all of a long cache
        w2 = torch.randint(0, 2, (1, 1, S2), generator=g).float()
        evict_check(lh, 1, 1, 8, S2, 20000, [S2], 20000, 10, 5, w=w2)
    # values that differ in their last bit only
    w = (torch.full((1, 1, S), 1.0).view(torch.int32)
         + torch.randperm(S, generator=g).int()).view(torch.float32)
    evict_check(lh, 1, 1, 64, S, 512, [S], 333, 0, 0, w=w)


def test_evict_allocates_what_is_left_out(lh):
    t = make(2, 1, 1, 64, 0, 64, [64, 20], torch.bfloat16)
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    r = lh.cache_evict(d["k"], d["v"], d["weights"], d["lens"], 32, recent=4, capacity=40)
    assert [tuple(x.shape) for x in r] == [(2, 1, 64, 40), (2, 1, 40, 64), (2, 1, 40), (2,),
                                           (2, 1, 32)]
    assert r[3].tolist() == [32, 20] and r[4][1, 0, 20:].tolist() == [-1] * 12
    assert tuple(lh.cache_evict(d["k"], d["v"], d["weights"], d["lens"], 32)[0].shape)[3] == 64
    with pytest.raises(RuntimeError, match="overlap"):
        lh.cache_evict(d["k"], d["v"], d["weights"], d["lens"], 32, k_out=d["k"])
    with pytest.raises(RuntimeError, match="keep"):
        lh.cache_evict(d["k"], d["v"], d["weights"], d["lens"], 32, recent=33)


# ---- appending ------------------------------------------------------------------

def append_check(lh, B, G, D, S, T, lens, counts, e=torch.bfloat16, seed=0):
    print("append", B, G, D, S, T, lens[:6], counts and counts[:6], e, flush=True)
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((B, G, D, S), generator=g).to(e)
    v = torch.randn((B, G, S, D), generator=g).to(e)
    nk = torch.randn((B, T, G, D), generator=g).to(e)
    nv = torch.randn((B, T, G, D), generator=g).to(e)
    w = torch.full((B, G, S), 3.0)
    kg, vg, wg = k.cuda(), v.cuda(), w.cuda()
    after = lh.cache_append(kg, vg, torch.tensor(lens, dtype=torch.int32).cuda(), nk.cuda(),
                            nv.cuda(), counts=None if counts is None else
                            torch.tensor(counts, dtype=torch.int32).cuda(),
                            weights=wg if seed else None)
    want = []
    for b in range(B):
        n = min(max(lens[b], 0), S)
        c = T if counts is None else min(max(counts[b], 0), T)
        m = min(c, S - n)
        for h in range(G):
            k[b, h, :, n:n + m] = nk[b, :m, h].t()
            v[b, h, n:n + m] = nv[b, :m, h]
            w[b, h, n:n + m] = 0.0 if seed else 3.0
        want.append(n + m)
    assert torch.equal(wg.cpu(), w)
    assert after.tolist() == want
    assert torch.equal(kg.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(vg.cpu().view(torch.int16), v.view(torch.int16))


@pytest.mark.parametrize("case", [
    # B, G, D, S, T, lens, counts
    (1, 1, 64, 8, 1, [0], None), (1, 1, 64, 8, 1, [8], None), (3, 2, 128, 65, 1, [0, 64, 65], None),
    (2, 1, 80, 100, 7, [95, 3], None), (2, 2, 256, 264, 100, [164, 7], None),
    (3, 8, 128, 512, 200, [0, 311, 312], [200, 0, 200]), (2, 1, 96, 77, 64, [13, 14], [64, 63]),
    (4, 1, 8, 33, 9, [-4, 1000, 30, 5], [3, 3, 9, 1000]), (1, 3, 64, 3001, 1500, [777], [1499]),
    (2, 1, 128, 2048, 2048, [0, 1], [2048, -1]), (66, 1, 64, 40, 3, [i % 41 for i in range(66)], None),
    (1, 1, 128, 4096, 1025, [1024], None), (2, 2, 40, 130, 129, [1, 0], [129, 128]),
], ids=lambda c: "x".join(map(str, c[:5])))
def test_append(lh, case):
    for seed, e in enumerate(TYPES.values()):      # the second with weights
        append_check(lh, *case, e=e, seed=seed)


def test_append_past_four_gib(lh):
    B, D, S = 2, 256, 5 << 20
    k = torch.zeros(B, 1, D, S, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(B, 1, S, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([S - 2, S - 70], dtype=torch.int32, device="cuda")
    nk = torch.randn(B, 100, 1, D, device="cuda").to(torch.bfloat16)
    nv = torch.randn(B, 100, 1, D, device="cuda").to(torch.bfloat16)
    assert lh.cache_append(k, v, lens, nk, nv).tolist() == [S, S]
    for b, m in enumerate((2, 70)):
        assert torch.equal(k[b, 0, :, S - m:], nk[b, :m, 0].t())
        assert torch.equal(v[b, 0, S - m:], nv[b, :m, 0])
        assert not k[b, 0, :, :S - m].any() and not v[b, 0, :S - m].any()


# ---- together, and where programs run them ---------------------------------------

def plain_loop(steps, B, G, H, D, P, S, keep, t, news):
    """The loop below on the CPU in 64 bits, with lists for caches."""
    K = [[[] for _ in range(G)] for _ in range(B)]
    V = [[[] for _ in range(G)] for _ in range(B)]
    W = [[[] for _ in range(G)] for _ in range(B)]
    outs = []
    for i in range(steps):
        nk, nv, counts, q = news[i]
        out = torch.zeros(B, G, H, D, dtype=torch.float64)
        for b in range(B):
            for g in range(G):
                for x in range(counts[b]):
                    K[b][g].append(nk[b, x, g].double())
                    V[b][g].append(nv[b, x, g].double())
                    W[b][g].append(0.0)
                keys = torch.stack([*t["prefix_k"][g].double().t(), *K[b][g]])
                vals = torch.stack([*t["prefix_v"][g].double(), *V[b][g]])
                p = torch.softmax(q[b, g].double() @ keys.t() / math.sqrt(D), -1)
                out[b, g] = p @ vals
                for j in range(len(W[b][g])):
                    W[b][g][j] += float(p[:, P + j].sum())
        outs.append(out)
        if i % 4 == 3:
            for b in range(B):
                for g in range(G):
                    at = kept(torch.tensor(W[b][g], dtype=torch.float64), len(W[b][g]), keep, 4, 2)
                    K[b][g] = [K[b][g][j] for j in at]
                    V[b][g] = [V[b][g][j] for j in at]
                    W[b][g] = [W[b][g][j] for j in at]
    return outs, W


def test_serving_loop(lh):
    """A ragged prompt, then steps: append, decode over prefix and cache with
    weights gathered, cut to the heaviest keys every fourth step."""
    B, G, H, D, P, S, keep, steps = 3, 2, 4, 64, 37, 96, 24, 12
    t = make(B, G, H, D, P, S, [0] * B, torch.bfloat16, seed=21)
    g = torch.Generator().manual_seed(22)
    news = []
    for i in range(steps):
        T = 40 if i == 0 else 1
        counts = [40, 13, 26] if i == 0 else [1] * B
        news.append((torch.randn((B, T, G, D), generator=g).to(torch.bfloat16),
                     torch.randn((B, T, G, D), generator=g).to(torch.bfloat16), counts,
                     (2 * torch.randn((B, G, H, D), generator=g)).to(torch.bfloat16)))
    want, W = plain_loop(steps, B, G, H, D, P, S, keep, t, news)
    k = torch.full((B, G, D, S), math.nan, dtype=torch.bfloat16, device="cuda")
    v = torch.full((B, G, S, D), math.nan, dtype=torch.bfloat16, device="cuda")
    w = torch.full((B, G, S), math.nan, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    pk, pv = t["prefix_k"].cuda(), t["prefix_v"].cuda()
    u = 2.0 ** -8
    for i, (nk, nv, counts, q) in enumerate(news):
        lens = lh.cache_append(k, v, lens, nk.cuda(), nv.cuda(),
                               counts=torch.tensor(counts, dtype=torch.int32).cuda(), weights=w)
        out = lh.cache_decode(k, v, q.cuda(), lens, prefix_k=pk, prefix_v=pv, weights=w)
        # |v| < 5 in every draw: 3 roundings of at most u (A <= 5), fp32 beside them
        near(out, want[i], torch.full_like(want[i], 3 * u * 5), f"loop step {i}")
        if i % 4 == 3:
            k, v, w, lens, _ = lh.cache_evict(k, v, w, lens, keep, recent=4, sinks=2)
    for b in range(B):
        for h in range(G):
            n = int(lens[b])
            assert n == len(W[b][h])
            # steps x H weights of fp32 accuracy (E < 1e-4 at these sizes)
            near(w[b, h, :n], torch.tensor(W[b][h], dtype=torch.float64),
                 torch.full((n,), steps * H * 1e-4, dtype=torch.float64), "loop weights")


def _captured(run, outs):
    run()
    torch.cuda.synchronize()
    ref = [o.clone() for o in outs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    side = torch.randn(1 << 18, device="cuda")
    return g, ref, side


def test_graph_replays_follow_the_lengths(lh):
    """A captured step and eviction: replays read the lengths, caches and
    weights as they are then; eager calls run between them."""
    B, G, H, D, P, S = 4, 2, 8, 128, 200, 320
    t = make(B, G, H, D, P, S, [S] * B, torch.bfloat16, seed=31)
    d = {n: x.cuda() for n, x in t.items()}
    into = torch.zeros(B, G, S, device="cuda")
    out = torch.empty(B, G, H, D, dtype=torch.bfloat16, device="cuda")
    ws = lh.cache_decode_workspace(B, G, H, D, P, S, True, "cuda:0")
    ko = torch.zeros(B, G, D, 128, dtype=torch.bfloat16, device="cuda")
    vo = torch.zeros(B, G, 128, D, dtype=torch.bfloat16, device="cuda")
    wo, lo = torch.zeros(B, G, 128, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    ix = torch.zeros(B, G, 100, dtype=torch.int32, device="cuda")
    nk = torch.randn(B, 1, G, D, device="cuda").to(torch.bfloat16)
    la = torch.zeros(B, dtype=torch.int32, device="cuda")

    def run():
        lh.cache_append(d["k"], d["v"], d["lens"], nk, nk, la)
        lh.cache_decode(d["k"], d["v"], d["q"], la, out, ws, prefix_k=d["prefix_k"],
                        prefix_v=d["prefix_v"], weights=d["weights"], weights_out=into)
        lh.cache_evict(d["k"], d["v"], into, la, 100, recent=8, sinks=2, k_out=ko, v_out=vo,
                       weights_out=wo, lens_out=lo, index=ix)

    outs = [out, into, ko, vo, wo, lo, ix, la]
    g, _, side = _captured(run, outs)
    for lens in ([0, 1, 64, 319], [320, 200, 100, 99], [S] * B, [7, 8, 9, 10]):
        d["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        for o in outs:
            o.zero_()
        run()
        torch.cuda.synchronize()
        ref = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        side.mul_(1.0001)
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, ref):
            assert torch.equal(o, r), lens


def test_threads_on_their_own_streams(lh):
    """Four host threads, each with its stream, caches and sizes: the results of
    calls made alone, bit for bit."""
    import threading
    ts = [make(2 + i, 2, 8, 64 + 64 * (i % 2), 100 * i, 256 + 64 * i,
               [(50 * b + 7 * i) % 257 for b in range(2 + i)], torch.bfloat16, seed=50 + i)
          for i in range(4)]
    d = [{n: None if x is None else x.cuda() for n, x in t.items()} for t in ts]

    def work(x):
        w = x["weights"].clone()
        o = lh.cache_decode(x["k"], x["v"], x["q"], x["lens"], prefix_k=x["prefix_k"],
                            prefix_v=x["prefix_v"], weights=w)
        r = lh.cache_evict(x["k"], x["v"], w, x["lens"], 40, recent=4, sinks=1,
                           k_out=torch.zeros_like(x["k"]), v_out=torch.zeros_like(x["v"]),
                           weights_out=torch.zeros_like(w))
        return (o, w, *r)

    want = [work(x) for x in d]
    torch.cuda.synchronize()
    got, errors = [[] for _ in d], []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(8):
                    got[i].append(work(d[i]))
            s.synchronize()
        except Exception as e:      # noqa: BLE001  (reported by the test)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not errors, errors
    for i in range(4):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_two_streams_at_once(lh):
    """Two steps of different extents side by side, each on its own stream."""
    ts = [make(4, 2, 8, 128, 500, 640, [640, 0, 100, 333], torch.bfloat16, seed=41),
          make(8, 1, 32, 64, 0, 1024, [1024] * 8, torch.float16, seed=42)]
    want = [step(lh, t) for t in ts]
    torch.cuda.synchronize()
    d = [{n: None if x is None else x.cuda() for n, x in t.items()} for t in ts]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, x in enumerate(d):
            with torch.cuda.stream(streams[i]):
                w = x["weights"].clone()
                o = lh.cache_decode(x["k"], x["v"], x["q"], x["lens"], prefix_k=x["prefix_k"],
                                    prefix_v=x["prefix_v"], weights=w)
                got[i].append((o, w))
    torch.cuda.synchronize()
    for i in range(2):
        for o, w in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(w, want[i][1])
