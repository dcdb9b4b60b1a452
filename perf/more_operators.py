"""The work of decoders whose memory does not grow with the sequence: attention
over a sliding window of the cache and its first tokens (``window``: new tokens of
a prompt or of one step), and linear attention with a decay for each head, over
whole prompts (``linear``) and one token at a time (``step``).

``listed()`` names twelve calls, ``draw()`` gives more of the same ranges;
``prepare`` makes what a serving program holds before the call, ``run`` makes the
call -- the framework's own where ``own`` is true, else the same mathematics in
elementary torch operations -- ``work`` counts the bytes and operations the call
cannot do without, and ``exact`` computes its outputs in 64 bits.

Every case is a dict of plain values.  B sequences of G KV heads, H query heads to
each.  window: head dim D, caches of capacity S of which T new tokens have just
been appended, ``lo`` spreads what the caches held before them: evenly between
lo * (S - T) and S - T, in an order of the seed's.  linear, step: key dim D, value
dim E.  ``ragged``: the batch is padded, its sequences bring between a quarter of T
and T tokens.
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
        # one step of one sequence over a short window: the smallest call, where
        # launches and the host's way to them count
        {"name": "window_step_one", "op": "window", "dtype": "bf16", "B": 1, "G": 1, "H": 32,
         "D": 128, "S": 4096, "T": 1, "W": 512, "sinks": 4, "lo": 1.0, "ragged": False},
        # a serving batch's step, grouped heads, a long window
        {"name": "window_step_batch", "op": "window", "dtype": "f16", "B": 32, "G": 8, "H": 4,
         "D": 128, "S": 8192, "T": 1, "W": 4096, "sinks": 4, "lo": 0.25, "ragged": False},
        # many conversations, a usual window, more query heads to a KV head
        {"name": "window_step_server", "op": "window", "dtype": "bf16", "B": 64, "G": 8, "H": 8,
         "D": 128, "S": 4096, "T": 1, "W": 1024, "sinks": 0, "lo": 0.0, "ragged": False},
        # whole prompts from the first token on
        {"name": "window_prompt", "op": "window", "dtype": "bf16", "B": 4, "G": 8, "H": 4,
         "D": 128, "S": 4096, "T": 4096, "W": 1024, "sinks": 4, "lo": 1.0, "ragged": False},
        # the largest: a long prompt's next chunk behind what its cache holds
        {"name": "window_chunk", "op": "window", "dtype": "bf16", "B": 1, "G": 8, "H": 8,
         "D": 128, "S": 32768, "T": 8192, "W": 4096, "sinks": 16, "lo": 1.0, "ragged": False},
        # a padded batch at odd sizes (K rows off 16-byte boundaries), narrow heads
        {"name": "window_odd", "op": "window", "dtype": "f16", "B": 3, "G": 2, "H": 5, "D": 80,
         "S": 2047, "T": 1001, "W": 333, "sinks": 1, "lo": 0.0, "ragged": True},
        # one short prompt, a state to begin with
        {"name": "linear_one", "op": "linear", "dtype": "bf16", "B": 1, "G": 16, "H": 1, "D": 128,
         "E": 128, "T": 512, "state": True, "ragged": False},
        # one long prompt: few heads, a long axis
        {"name": "linear_long", "op": "linear", "dtype": "bf16", "B": 1, "G": 32, "H": 1,
         "D": 128, "E": 128, "T": 32768, "state": False, "ragged": False},
        # a padded batch of prompts
        {"name": "linear_prompts", "op": "linear", "dtype": "bf16", "B": 8, "G": 32, "H": 1,
         "D": 128, "E": 128, "T": 4096, "state": False, "ragged": True},
        # grouped heads, key and value dims that differ, an odd length
        {"name": "linear_odd", "op": "linear", "dtype": "f16", "B": 3, "G": 4, "H": 3, "D": 64,
         "E": 96, "T": 1777, "state": True, "ragged": True},
        # one token of one sequence
        {"name": "step_one", "op": "step", "dtype": "bf16", "B": 1, "G": 32, "H": 1, "D": 128,
         "E": 128},
        # one token of a serving batch: the states' stream
        {"name": "step_batch", "op": "step", "dtype": "bf16", "B": 64, "G": 32, "H": 1, "D": 128,
         "E": 128},
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
    op = rng.choice(["window", "window", "window", "linear", "linear", "step"])
    c = {"op": op, "dtype": "bf16" if rng.random() < 0.65 else "f16", "B": _log(rng, 1, 64)}
    if op == "window":
        t = 1 if rng.random() < 0.5 else _size(rng, 2, 8192)
        g = rng.choice([1, 1, 2, 4, 8])
        c.update(G=g, H=rng.choice([1, 2, 4, 5, 7, 8, 12] if g > 1 else [1, 8, 16, 32, 32, 40, 71]),
                 D=rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), T=t,
                 S=t + _size(rng, 64, 16384), W=_size(rng, 32, 8192),
                 sinks=rng.choice([0, 1, 4, 4, 16, 100]), lo=rng.choice([0.0, 0.25, 0.5, 1.0]),
                 ragged=t > 1 and rng.random() < 0.5)
        return c
    h = rng.choice([1, 1, 1, 2, 3, 4])
    d = rng.choice([64, 64, 80, 128, 128, 128, 256])
    c.update(G=max(1, _log(rng, 2, 48) // h), H=h, D=d,
             E=d if rng.random() < 0.6 else rng.choice([32, 64, 96, 128, 192, 256]))
    if op == "linear":
        t = _size(rng, 2, 32768)
        c.update(T=t, state=rng.random() < 0.5, ragged=rng.random() < 0.5)
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
        # caches are made whole, and the plain form holds a state for every chunk
        whole = 4 * c["B"] * c["G"] * c["D"] * c["S"] if c["op"] == "window" else 0
        if w["bytes"] <= b and w["flops"] <= f and whole <= 1 << 30:
            return c


def _counts(case):
    """How many of the T new tokens each sequence brings."""
    B, T = case["B"], case.get("T", 1)
    if not case.get("ragged"):
        return [T] * B
    return [max(1, T // 4 + (T - T // 4) * (i + 1) // B) for i in range(B)]


def _before(case):
    """What the caches held before the new tokens, ascending."""
    B, top = case["B"], case["S"] - case["T"]
    return [int(top * (1 - (1 - case["lo"]) * i / max(1, B - 1))) for i in reversed(range(B))]


def work(case):
    B, G, H, D = case["B"], case["G"], case["H"], case["D"]
    n = _counts(case)
    if case["op"] != "window":
        E, tokens = case["E"], sum(n)
        states = 4 * B * G * H * D * E * (2 if case["op"] == "step" or case["state"] else 1)
        return {"bytes": tokens * G * 2 * (H * D + D + E + H * E) + states + 4 * G * H,
                "flops": 4 * tokens * G * H * D * E}
    W, sinks, keys, pairs = case["W"], case["sinks"], 0, 0
    # (prepare orders both by the same permutation)
    for m, base in zip(n, _before(case)):
        first = max(0, base - W + 1)
        keys += base + m - first + min(sinks, first)
        # the rows' keys: min(W, p + 1) of the window, min(sinks, p - W + 1) before it
        for p0, p1, top, shift in ((base, base + m, W, 1), (base, base + m, sinks, 1 - W)):
            lo, hi = p0 + shift, p1 + shift          # sum of clamp(x, 0, top), x = lo .. hi - 1
            a, b = min(max(lo, 0), top), min(max(hi, 0), top)
            pairs += (b - a) * (a + b - 1) // 2 + max(0, hi - max(lo, top)) * top
    return {"bytes": 4 * G * D * keys + 4 * sum(n) * G * H * D + 4 * B,
            "flops": 4 * G * H * D * pairs}


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
    B, G, H, D = case["B"], case["G"], case["H"], case["D"]
    order = torch.randperm(B, generator=g, device="cuda")
    n = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")[order]
    t = {"case": case, "counts": n if case.get("ragged") else None}
    if case["op"] == "window":
        S, T = case["S"], case["T"]
        t["k"] = _keys(g, (B, G, D, S), 3, e)
        t["v"] = _normal(g, (B, G, S, D), e)
        t["lens"] = torch.tensor(_before(case), dtype=torch.int32, device="cuda")[order] + n
        t["q"] = _normal(g, (B, T, G, H, D) if T > 1 else (B, G, H, D), e)
        # a padded batch's output holds something behind its sequences already
        t["out"] = torch.zeros_like(t["q"])
        return t
    E, T = case["E"], case.get("T", 1)
    lead = (B, T) if case["op"] == "linear" else (B,)
    t["q"] = _normal(g, (*lead, G, H, D), e)
    # keys of unit length, as such layers normalise them
    t["k"] = (_normal(g, (*lead, G, D), torch.float32) / math.sqrt(D)).to(e)
    t["v"] = _normal(g, (*lead, G, E), e)
    # heads that remember between 4 and 4096 tokens
    far = 2 + 10 * torch.rand((G, H), generator=g, device="cuda", dtype=torch.float64)
    t["log_decay"] = torch.log1p(-torch.exp2(-far)).to(torch.float32)
    t["state"] = None
    if case["op"] == "step" or case["state"]:
        # what as many tokens as a head remembers leave behind
        t["state"] = _normal(g, (B, G, H, D, E), torch.float32) \
            * torch.exp2(far / 2).to(torch.float32)[..., None, None] / math.sqrt(2 * D)
    t["out"] = torch.zeros((*lead, G, H, E), dtype=e, device="cuda")
    return t


def run(state):
    op = state["case"]["op"]
    if own:
        loom_hip, case = _package(), state["case"]
        if op == "window":
            if case["T"] == 1:
                return loom_hip.window_decode(
                    state["k"], state["v"], state["q"], state["lens"], case["W"], state["out"],
                    sinks=case["sinks"])
            return loom_hip.window_attention(
                state["k"], state["v"], state["q"], state["lens"], case["W"], state["out"],
                sinks=case["sinks"], counts=state["counts"])
        if op == "step":
            return loom_hip.linear_attention_step(
                state["q"], state["k"], state["v"], state["log_decay"], state["state"],
                state["out"]), state["state"]
        return loom_hip.linear_attention(
            state["q"], state["k"], state["v"], state["log_decay"], state["state"], state["out"],
            counts=state["counts"])
    return {"window": _window, "linear": _linear, "step": _step}[op](state)


def _package():
    p = os.path.join(_ROOT, "loom-dataflow_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import loom_hip
    return loom_hip


def _window(st):
    case, f = st["case"], torch.float32
    W, sinks = case["W"], case["sinks"]
    k, v, q, lens = st["k"], st["v"], st["q"], st["lens"].long()
    B, G, D, S = k.shape
    T, H, dev = case["T"], case["H"], k.device
    n = torch.full_like(lens, T) if st["counts"] is None else st["counts"].long()
    first = lens - n                                   # where the new tokens begin
    # blocks of C tokens against the C + W - 1 keys that end with their last one
    C = min(T, 256)
    N = -(-T // C)
    there = torch.arange(N * C, device=dev)
    span = torch.arange(N * C + W - 1, device=dev) - (W - 1) + first[:, None]
    at = span.clamp(0, S - 1)
    kw = torch.gather(k, 3, at[:, None, None].expand(B, G, D, -1)).unfold(3, C + W - 1, C)
    kw = kw.permute(0, 1, 3, 2, 4).to(f).contiguous()                        # B G N D C+W-1
    vw = torch.gather(v, 2, at[:, None, :, None].expand(B, G, -1, D)).unfold(2, C + W - 1, C)
    vw = vw.permute(0, 1, 2, 4, 3).to(f).contiguous()                        # B G N C+W-1 D
    x = q.view(B, T, G, H, D).to(f) / math.sqrt(D)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 0, 0, N * C - T))
    x = x.view(B, N, C, G, H, D).permute(0, 3, 1, 2, 4, 5).reshape(B, G, N, C * H, D)
    pos = (first[:, None] + there).view(B, N, C)
    key = span.unfold(1, C + W - 1, C)                                       # B N C+W-1
    seen = (key[:, :, None] <= pos[..., None]) & (key[:, :, None] > pos[..., None] - W) \
        & (key[:, :, None] >= 0)
    s = torch.matmul(x, kw).view(B, G, N, C, H, -1)
    s = s.masked_fill_(~seen[:, None, :, :, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    if sinks:
        m = min(sinks, S)
        sk = k[..., :m].to(f).unsqueeze(2).expand(B, G, N, D, m).contiguous()
        early = torch.arange(m, device=dev) <= pos[..., None] - W            # B N C m
        ss = torch.matmul(x, sk).view(B, G, N, C, H, m)
        ss = ss.masked_fill_(~early[:, None, :, :, None], float("-inf"))
        top = torch.maximum(top, ss.amax(-1, keepdim=True))
    top = top.clamp(min=torch.finfo(f).min)            # a row without keys
    p = s.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, G, N, C * H, -1), vw).view(B, G, N, C, H, D)
    if sinks:
        ps = torch.exp(ss - top)
        den = den + ps.sum(-1, keepdim=True)
        sv = v[:, :, :m].to(f).unsqueeze(2).expand(B, G, N, m, D).contiguous()
        out = out + torch.matmul(ps.view(B, G, N, C * H, m), sv).view(B, G, N, C, H, D)
    out = out / torch.where(den > 0, den, torch.ones_like(den))
    out = out.permute(0, 2, 3, 1, 4, 5).reshape(B, N * C, G, H, D)[:, :T].to(q.dtype)
    if st["counts"] is not None:                       # rows behind a sequence stay
        out = torch.where((there[:T] < n[:, None])[..., None, None, None], out, st["out"])
    return out.view(q.shape)


def _linear(st):
    case, f, d = st["case"], torch.float32, torch.float64
    B, T, G, H, D = st["q"].shape
    E, dev = case["E"], st["q"].device
    n = torch.full((B,), T, device=dev) if st["counts"] is None else st["counts"].long()
    C = min(T, 64)
    N = -(-T // C)
    pad = N * C - T
    i = torch.arange(C, device=dev)
    live = (torch.arange(N * C, device=dev) < n[:, None]).view(B, 1, N, C, 1)

    def chunks(x):                                     # B T G x -> B G N C x
        x = torch.nn.functional.pad(x.to(f), (0, 0, 0, 0, 0, pad))
        return x.view(B, N, C, G, -1).permute(0, 3, 1, 2, 4) * live

    k, v = chunks(st["k"]), chunks(st["v"])
    q = chunks(st["q"].reshape(B, T, G, H * D)).view(B, G, N, C, H, D)
    q = q.permute(0, 1, 4, 2, 3, 5) / math.sqrt(D)     # B G H N C D
    # decays of far positions in 64 bits
    g = st["log_decay"].to(d)[:, :, None]
    # a chunk's tokens that count
    m = (n[:, None] - torch.arange(N, device=dev) * C).clamp(0, C)           # B N
    # what is left of a token at the end of its chunk
    left = torch.exp(g[None, :, :, None] * (m[..., None] - 1 - i).clamp(min=0)[:, None, None]).to(f)
    kd = k[:, :, None] * left[..., None]               # B G H N C D
    own_state = torch.matmul(kd.transpose(4, 5).contiguous(), v[:, :, None])  # B G H N D E
    # the states at the chunks' starts and at the end
    to = torch.nn.functional.pad(m, (1, 0)).cumsum(1)  # tokens before a chunk: B N+1
    ends = to[:, 1:]
    far = (to[:, :, None] - ends[:, None]).clamp(min=0)                      # B N+1 N
    before = torch.arange(N + 1, device=dev)[:, None] > torch.arange(N, device=dev)
    mix = torch.where(before, torch.exp(g[None, ..., None] * far[:, None, None]), 0.0).to(f)
    states = torch.matmul(mix, own_state.view(B, G, H, N, D * E)).view(B, G, H, N + 1, D, E)
    if st["state"] is not None:
        states += torch.exp(g[None] * to[:, None, None])[..., None, None].to(f) \
            * st["state"][:, :, :, None]
    lag = i[:, None] - i
    decay = torch.where(lag >= 0, torch.exp(g[..., None] * lag.clamp(min=0)), 0.0).to(f)
    a = torch.matmul(q, k.transpose(3, 4).contiguous()[:, :, None]) * decay[None, :, :, None]
    out = torch.matmul(a, v[:, :, None])
    out += torch.matmul(q * torch.exp(g * (i + 1)).to(f)[None, :, :, None, :, None],
                        states[:, :, :, :N])
    out = out.permute(0, 3, 4, 1, 2, 5).reshape(B, N * C, G, H, E)[:, :T].to(st["q"].dtype)
    if st["counts"] is not None:                       # rows behind a sequence stay
        keep = torch.arange(T, device=dev) < n[:, None]
        out = torch.where(keep[..., None, None, None], out, st["out"])
    return out, states[:, :, :, N].contiguous()


def _step(st):
    f = torch.float32
    s = st["state"]
    s.mul_(torch.exp(st["log_decay"])[..., None, None])
    s.add_(st["k"].to(f)[:, :, None, :, None] * st["v"].to(f)[:, :, None, None, :])
    q = st["q"].to(f) / math.sqrt(st["case"]["D"])
    return torch.matmul(q[..., None, :], s)[..., 0, :].to(st["q"].dtype), s


def exact(case, seed):
    st, f = prepare(case, seed), torch.float64
    B, G, H, D = case["B"], case["G"], case["H"], case["D"]
    T = case.get("T", 1)
    n = [T] * B if st["counts"] is None else st["counts"].tolist()
    if case["op"] == "window":
        W, sinks = case["W"], case["sinks"]
        q = st["q"].view(B, T, G, H, D)
        out = st["out"].to(f).view(B, T, G, H, D)
        dev = q.device
        for b, length in enumerate(st["lens"].tolist()):
            for t0 in range(0, n[b], 512):
                t1 = min(n[b], t0 + 512)
                p = torch.arange(length - n[b] + t0, length - n[b] + t1, device=dev)
                low = max(0, int(p[0]) - W + 1)
                keys = torch.cat([torch.arange(min(sinks, low), device=dev),
                                  torch.arange(low, int(p[-1]) + 1, device=dev)])
                see = (keys <= p[:, None]) & ((keys > p[:, None] - W) | (keys < sinks))
                for h0 in range(G):
                    x = q[b, t0:t1, h0].to(f)                                # t H D
                    s = torch.matmul(x, st["k"][b, h0][:, keys].to(f)) / math.sqrt(D)
                    s = torch.where(see[:, None], s, -math.inf)
                    out[b, t0:t1, h0] = torch.matmul(torch.softmax(s, -1),
                                                     st["v"][b, h0][keys].to(f))
        return out.view(st["q"].shape)
    E = case["E"]
    q = st["q"].view(B, T, G, H, D)
    k, v = st["k"].view(B, T, G, D), st["v"].view(B, T, G, E)
    g = st["log_decay"].to(f)
    out = st["out"].to(f).view(B, T, G, H, E)
    end = torch.zeros((B, G, H, D, E), dtype=f, device=q.device)
    L = 128
    for b in range(B):
        s = end[b] if st["state"] is None else st["state"][b].to(f)
        for t0 in range(0, n[b], L):
            m = min(L, n[b] - t0)
            i = torch.arange(m, dtype=f, device=q.device)
            kb = k[b, t0:t0 + m].to(f).permute(1, 0, 2)[:, None]             # G 1 m D
            vb = v[b, t0:t0 + m].to(f).permute(1, 0, 2)[:, None]
            qb = q[b, t0:t0 + m].to(f).permute(1, 2, 0, 3) / math.sqrt(D)     # G H m D
            a = torch.matmul(qb, kb.transpose(2, 3))
            a = a * torch.exp(g[..., None, None] * (i[:, None] - i)).tril()
            o = torch.matmul(a, vb) \
                + torch.exp(g[..., None] * (i + 1))[..., None] * torch.matmul(qb, s)
            out[b, t0:t0 + m] = o.permute(2, 0, 1, 3)
            w = torch.exp(g[..., None] * (m - 1 - i))[..., None]
            s = torch.exp(g * m)[..., None, None] * s + torch.matmul((kb * w).transpose(2, 3), vb)
        end[b] = s
    return (out if case["op"] == "linear" else out[:, 0]), end
