"""The work of a serving loop's cache whose speed matters: appending new tokens
to the sequences' caches (``append``), one decoding step over them with an
optional shared prefix and accumulated attention weights (``decode``), and
cutting them to their heaviest keys (``evict``).

``listed()`` names twelve calls, ``draw()`` gives more of the same ranges;
``prepare`` makes what a serving program holds before the call, ``run`` makes
the call -- the framework's own where ``own`` is true, else the same
mathematics in elementary torch operations -- ``work`` counts the bytes and
operations the call cannot do without, and ``exact`` computes its outputs in 64
bits.

Every case is a dict of plain values.  B sequences of G KV heads, H query heads
to each, head dim D; S is the caches' capacity and ``lo`` spreads the lengths:
evenly between lo * S and S, in an order of the seed's.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a step of one sequence that goes on from a cached system prompt: the
        # smallest call, where launches and the host's way to them count
        {"name": "prefix_one", "op": "decode", "dtype": "bf16", "B": 1, "G": 1, "H": 32, "D": 128,
         "P": 1000, "S": 256, "lo": 1.0, "weights": False},
        # a batch of conversations under one long instruction, one KV head
        {"name": "prefix_batch", "op": "decode", "dtype": "bf16", "B": 32, "G": 1, "H": 32,
         "D": 128, "P": 8192, "S": 1024, "lo": 0.25, "weights": False},
        # grouped heads, a prefix of odd length (rows off 16-byte boundaries)
        {"name": "prefix_groups_f16", "op": "decode", "dtype": "f16", "B": 16, "G": 8, "H": 4,
         "D": 128, "P": 4095, "S": 2048, "lo": 0.25, "weights": False},
        # the largest: a full server, grouped heads, long prefix and long caches
        {"name": "prefix_server", "op": "decode", "dtype": "bf16", "B": 48, "G": 8, "H": 8,
         "D": 128, "P": 16384, "S": 4096, "lo": 0.25, "weights": False},
        # one sequence whose keys' weights are gathered
        {"name": "weights_one", "op": "decode", "dtype": "bf16", "B": 1, "G": 1, "H": 32,
         "D": 128, "P": 0, "S": 4096, "lo": 1.0, "weights": True},
        # a serving batch with long caches, weights gathered
        {"name": "weights_batch", "op": "decode", "dtype": "bf16", "B": 32, "G": 1, "H": 32,
         "D": 128, "P": 0, "S": 8192, "lo": 0.5, "weights": True},
        # many query heads of a narrow head dim over an odd capacity, prefix and weights
        {"name": "weights_prefix_71", "op": "decode", "dtype": "bf16", "B": 16, "G": 1, "H": 71,
         "D": 64, "P": 515, "S": 2047, "lo": 0.0, "weights": True},
        # a long prompt's cache cut to a quarter
        {"name": "evict_one", "op": "evict", "dtype": "bf16", "B": 1, "G": 1, "D": 128, "S": 4096,
         "lo": 1.0, "keep": 1024, "recent": 128, "sinks": 4, "cap": 2048},
        # a batch of full caches cut to a quarter
        {"name": "evict_batch", "op": "evict", "dtype": "bf16", "B": 32, "G": 1, "D": 128,
         "S": 8192, "lo": 0.5, "keep": 2048, "recent": 256, "sinks": 4, "cap": 4096},
        # grouped heads at odd sizes, most keys kept
        {"name": "evict_groups_odd", "op": "evict", "dtype": "f16", "B": 8, "G": 8, "D": 64,
         "S": 16383, "lo": 0.75, "keep": 9001, "recent": 500, "sinks": 0, "cap": 10001},
        # every decoding step: one token to each sequence
        {"name": "append_step", "op": "append", "dtype": "bf16", "B": 32, "G": 1, "D": 128,
         "S": 8192, "T": 1, "lo": 0.25},
        # a padded batch of prompts of different lengths
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "B": 8, "G": 8, "D": 128,
         "S": 8192, "T": 4096, "lo": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """An extent between lo and hi, spread over its logarithm: half of them a
    multiple of 64, a quarter a multiple of 8, a quarter as data gives them."""
    v, k = _log(rng, lo, hi), rng.random()
    step = 64 if k < 0.5 else 8 if k < 0.75 else 1
    return max(lo, min(hi, max(step, (v + step // 2) // step * step)))


def _draw_once(rng):
    op = rng.choice(["decode", "decode", "decode", "decode", "evict", "evict", "append"])
    c = {"op": op, "dtype": "bf16" if rng.random() < 0.65 else "f16", "B": _log(rng, 1, 64),
         "G": rng.choice([1, 1, 1, 2, 4, 8]), "D": rng.choice([64, 64, 80, 96, 128, 128, 128, 256]),
         "lo": rng.choice([0.0, 0.25, 0.5, 1.0])}
    if op == "decode":
        h = [1, 2, 4, 5, 7, 8, 12, 16] if c["G"] > 1 else [8, 16, 32, 32, 40, 48, 64, 71]
        c.update(H=rng.choice(h), P=0 if rng.random() < 0.25 else _size(rng, 16, 16384),
                 S=_size(rng, 64, 8192), weights=rng.random() < 0.5)
    elif op == "evict":
        s = _size(rng, 256, 16384)
        keep = max(8, int(s * rng.uniform(0.1, 0.8)))
        c.update(S=s, keep=keep, recent=int(keep * rng.uniform(0, 0.5)),
                 sinks=rng.choice([0, 1, 4]), cap=min(s, keep + _log(rng, 1, 256)))
    else:
        t = 1 if rng.random() < 0.4 else _size(rng, 2, 4096)
        c.update(T=t, S=t + _size(rng, 64, 8192))
    return c


def draw(rng):
    """One more case, no more costly than the largest listed one of its kind."""
    most = {}
    for c in listed():
        w, have = work(c), most.get(c["op"], (0, 0))
        most[c["op"]] = (max(have[0], w["bytes"]), max(have[1], w["flops"]))
    while True:
        c = _draw_once(rng)
        w, (b, f) = work(c), most[c["op"]]
        # the caches are made and compared whole, whatever a call touches
        whole = 4 * c["B"] * c["G"] * c["D"] * c["S"]
        if w["bytes"] <= b and w["flops"] <= f and whole <= 1 << 30:
            return c


def _lengths(case):
    """The lengths of the caches before the call, ascending."""
    B, top = case["B"], case["S"] - case.get("T", 0)
    return [int(top * (1 - (1 - case["lo"]) * i / max(1, B - 1))) for i in reversed(range(B))]


def _counts(case):
    """How many of the T new tokens each sequence brings: a single one each, or
    prompts between a quarter of T and T."""
    B, T = case["B"], case["T"]
    return [T if T == 1 else max(1, T // 4 + (T - T // 4) * (i + 1) // B) for i in range(B)]


def work(case):
    B, G, D = case["B"], case["G"], case["D"]
    if case["op"] == "append":
        return {"bytes": 2 * 4 * G * D * sum(_counts(case)) + 12 * B, "flops": 0}
    n = _lengths(case)
    if case["op"] == "evict":
        kept = sum(min(x, case["keep"]) for x in n)
        # every weight read; the kept keys' K, V and weight read and written
        return {"bytes": G * (4 * sum(n) + kept * 2 * (4 * D + 4) + 4 * B * case["keep"]) + 8 * B,
                "flops": 0}
    H, P = case["H"], case["P"]
    nbytes = 4 * G * D * (P + sum(n)) + 4 * B * G * H * D + 4 * B
    if case["weights"]:
        nbytes += 8 * G * sum(n)
    return {"bytes": nbytes, "flops": 4 * G * H * D * (B * P + sum(n))}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _keys(g, shape, axis, dtype):
    """Keys of which one in sixteen draws more attention than the rest."""
    k = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    stand = [1] * len(shape)
    stand[axis] = shape[axis]
    k *= 1.0 + 2.0 * (torch.rand(stand, generator=g, device="cuda") < 1 / 16)
    return k.to(dtype)


def prepare(case, seed):
    g, e = _gen(seed), _TYPES[case["dtype"]]
    B, G, D, S = case["B"], case["G"], case["D"], case["S"]
    order = torch.randperm(B, generator=g, device="cuda")
    t = {"k": _keys(g, (B, G, D, S), 3, e), "v": _normal(g, (B, G, S, D), e),
         "lens": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]}
    if case["op"] == "append":
        t["new_k"] = _normal(g, (B, case["T"], G, D), e)
        t["new_v"] = _normal(g, (B, case["T"], G, D), e)
        # a step brings one token each; prompts are padded to the longest
        t["counts"] = None if case["T"] == 1 else \
            torch.tensor(_counts(case), dtype=torch.int32, device="cuda")[order.flip(0)]
        return {"case": case, **t}
    if case["op"] == "decode":
        t["q"] = _normal(g, (B, G, case["H"], D), e)
        t["prefix_k"] = _keys(g, (G, D, case["P"]), 2, e) if case["P"] else None
        t["prefix_v"] = _normal(g, (G, case["P"], D), e) if case["P"] else None
        t["weights"] = t["into"] = None
        if case["weights"]:
            t["weights"] = torch.rand((B, G, S), generator=g, device="cuda")
            t["into"] = torch.zeros((B, G, S), device="cuda")
        return {"case": case, **t}
    # weights of a few heavy keys and many light ones, some of them (keys that
    # no head has looked at) exactly zero
    w = torch.exp(2.0 * torch.randn((B, G, S), generator=g, device="cuda"))
    w *= torch.rand((B, G, S), generator=g, device="cuda") > 0.2
    t["weights"] = w
    # the smaller caches that a program moves to
    t["k_out"] = torch.zeros((B, G, D, case["cap"]), dtype=e, device="cuda")
    t["v_out"] = torch.zeros((B, G, case["cap"], D), dtype=e, device="cuda")
    t["weights_out"] = torch.zeros((B, G, case["cap"]), device="cuda")
    return {"case": case, **t}


def run(state):
    case = state["case"]
    if own:
        loom_hip = _package()
        if case["op"] == "append":
            return state["k"], state["v"], loom_hip.cache_append(
                state["k"], state["v"], state["lens"], state["new_k"], state["new_v"],
                counts=state["counts"])
        if case["op"] == "evict":
            return loom_hip.cache_evict(
                state["k"], state["v"], state["weights"], state["lens"], case["keep"],
                recent=case["recent"], sinks=min(case["sinks"], case["keep"] - case["recent"]),
                k_out=state["k_out"], v_out=state["v_out"], weights_out=state["weights_out"])
        out = loom_hip.cache_decode(
            state["k"], state["v"], state["q"], state["lens"], prefix_k=state["prefix_k"],
            prefix_v=state["prefix_v"], weights=state["weights"], weights_out=state["into"])
        return (out, state["into"]) if case["weights"] else out
    return {"append": _append, "evict": _evict, "decode": _decode}[case["op"]](state)


def _package():
    p = os.path.join(_ROOT, "loom-dataflow_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import loom_hip
    return loom_hip


def _append(st):
    k, v, lens = st["k"], st["v"], st["lens"].long()
    B, T = st["new_k"].shape[:2]
    S = k.shape[3]
    n = torch.full_like(lens, T) if st["counts"] is None else st["counts"].long()
    t = torch.arange(T, device=k.device)
    at = lens[:, None] + t
    b, i = torch.nonzero((t < n[:, None]) & (at < S), as_tuple=True)
    to = at[b, i]
    k[b, :, :, to] = st["new_k"][b, i]
    v[b, :, to, :] = st["new_v"][b, i]
    return k, v, torch.clamp(lens + n, max=S).to(torch.int32)


def _decode(st):
    case, f = st["case"], torch.float32
    k, v, q = st["k"].to(f), st["v"].to(f), st["q"].to(f) / math.sqrt(case["D"])
    B, G, H, D = q.shape
    S, P = k.shape[3], case["P"]
    there = torch.arange(S, device=k.device) < st["lens"][:, None]
    s = torch.matmul(q, k).masked_fill(~there[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    if P:
        rows = q.transpose(0, 1).reshape(G, B * H, D)
        sp = torch.matmul(rows, st["prefix_k"].to(f))
        top = torch.maximum(top, sp.amax(-1).view(G, B, H, 1).transpose(0, 1))
    top = top.clamp(min=torch.finfo(f).min)       # a row without keys
    e = torch.exp(s - top)
    den, out = e.sum(-1, keepdim=True), torch.matmul(e, v)
    if P:
        ep = torch.exp(sp - top.transpose(0, 1).reshape(G, B * H, 1))
        den = den + ep.sum(-1).view(G, B, H, 1).transpose(0, 1)
        out = out + torch.matmul(ep, st["prefix_v"].to(f)).view(G, B, H, D).transpose(0, 1)
    den = torch.where(den > 0, den, torch.ones_like(den))
    out = (out / den).to(st["q"].dtype)
    if not case["weights"]:
        return out
    w = (e / den).sum(2)
    st["into"].copy_(torch.where(there[:, None], st["weights"] + w, st["into"]))
    return out, st["into"]


def _evict(st):
    case, lens = st["case"], st["lens"].long()
    k, v, w = st["k"], st["v"], st["weights"]
    B, G, S = w.shape
    keep, recent = case["keep"], case["recent"]
    sinks = min(case["sinks"], keep - recent)
    at = torch.arange(S, device=w.device)
    n = lens[:, None, None]
    there = at < n
    must = (at < sinks) | (at >= n - recent)
    rank = torch.where(must, torch.full_like(w, float("inf")), w)
    rank = torch.where(there, rank, torch.full_like(w, float("-inf")))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    # what is kept, in the order of the slots; slots behind a short cache last
    slot = torch.where(torch.gather(there.expand(B, G, S), 2, best), best, S)
    slot = torch.sort(slot, dim=-1).values
    b, g, j = torch.nonzero(slot < S, as_tuple=True)
    s = slot[b, g, j]
    st["k_out"][b, g, :, j] = k[b, g, :, s]
    st["v_out"][b, g, j] = v[b, g, s]
    st["weights_out"][b, g, j] = w[b, g, s]
    index = torch.where(slot < S, slot, -1).to(torch.int32)
    return (st["k_out"], st["v_out"], st["weights_out"],
            torch.clamp(lens, max=keep).to(torch.int32), index)


def exact(case, seed):
    st, f = prepare(case, seed), torch.float64
    k, v, lens = st["k"], st["v"], st["lens"].tolist()
    B, G, D, S = case["B"], case["G"], case["D"], case["S"]
    if case["op"] == "append":
        n = [case["T"]] * B if st["counts"] is None else st["counts"].tolist()
        for b in range(B):
            m = min(n[b], S - lens[b])
            for g in range(G):
                k[b, g, :, lens[b]:lens[b] + m] = st["new_k"][b, :m, g].t()
                v[b, g, lens[b]:lens[b] + m] = st["new_v"][b, :m, g]
        return k.to(f), v.to(f), None
    if case["op"] == "evict":
        ko, vo, wo = st["k_out"].to(f), st["v_out"].to(f), st["weights_out"].to(f)
        keep, recent = case["keep"], case["recent"]
        sinks = min(case["sinks"], keep - recent)
        w = st["weights"].cpu()
        for b in range(B):
            for g in range(G):
                slots = list(range(lens[b]))
                if lens[b] > keep:
                    x = w[b, g].tolist()
                    middle = sorted(slots[sinks:lens[b] - recent], key=lambda i: (-x[i], i))
                    slots = slots[:sinks] + sorted(middle[:keep - sinks - recent]) \
                        + slots[lens[b] - recent:]
                at = torch.tensor(slots, dtype=torch.long, device=k.device)
                m = len(slots)
                ko[b, g, :, :m] = k[b, g].index_select(1, at).to(f)
                vo[b, g, :m] = v[b, g].index_select(0, at).to(f)
                wo[b, g, :m] = st["weights"][b, g].index_select(0, at).to(f)
        return ko, vo, wo, None, None
    out = torch.zeros((B, G, case["H"], D), dtype=f, device=k.device)
    into = None if st["into"] is None else st["into"].to(f)
    for g in range(G):
        pk = pv = None
        if case["P"]:
            pk, pv = st["prefix_k"][g].to(f), st["prefix_v"][g].to(f)
        for b in range(B):
            n = lens[b]
            x = st["q"][b, g].to(f)
            keys, vals = k[b, g, :, :n].to(f), v[b, g, :n].to(f)
            own_scores = torch.matmul(x, keys) / math.sqrt(D)
            scores = own_scores if pk is None else \
                torch.cat([torch.matmul(x, pk) / math.sqrt(D), own_scores], -1)
            if scores.shape[-1] == 0:
                continue
            p = torch.softmax(scores, -1)
            own_p = p[:, p.shape[1] - n:]
            out[b, g] = torch.matmul(own_p, vals)
            if pk is not None:
                out[b, g] += torch.matmul(p[:, :p.shape[1] - n], pv)
            if into is not None:
                into[b, g, :n] = st["weights"][b, g, :n].to(f) + own_p.sum(0)
    return out if into is None else (out, into)
