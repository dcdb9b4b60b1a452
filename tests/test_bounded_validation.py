"""Refusals of windowed and linear attention, without a GPU: the C entry points
reject bad arguments before anything is launched, the Python calls name the tensor
that is wrong and allocate nothing for a call that is refused; fuzzed extents and
pointers get a code and a message."""
import ctypes

import pytest
import torch
from hypothesis import given
from hypothesis import strategies as st

import loom_hip as lh
from tests.test_fuzz_abi import FUZZ
from tests.test_fuzz_cache import extents, pointers

FAR = 1 << 40     # made-up addresses, far from each other and never dereferenced


def P(i, off=0):
    return ctypes.c_void_p(FAR * (i + 1) + off)


def call(name, *args):
    buf = ctypes.create_string_buffer(256)
    rc = getattr(lh._lib, name)(*args, None, buf, len(buf))
    return rc, buf.value.decode()


def entry(name, n, ptrs, rest, f16):
    a = [P(i) for i in range(n)]
    for i, v in (ptrs or {}).items():
        a[i] = v
    return call(name + ("_f16" if f16 else ""), *a, *rest)


# k, v, q, lens, counts, out, workspace
W_DIMS = (2, 2, 4, 64, 30, 128, 50, 4)


def window(ptrs=None, dims=W_DIMS, scale=0.1, ws=1 << 40, f16=False):
    return entry("loom_hip_window_attention", 7, ptrs, (ws, *dims, ctypes.c_float(scale)), f16)


# q, k, v, log_decay, state, counts, out, state_out, workspace
L_DIMS = (2, 2, 4, 64, 32, 300)


def linear(ptrs=None, dims=L_DIMS, scale=0.1, ws=1 << 40, f16=False):
    return entry("loom_hip_linear_attention", 9, ptrs, (ws, *dims, ctypes.c_float(scale)), f16)


# q, k, v, log_decay, state, counts, out
def step(ptrs=None, dims=L_DIMS[:5], scale=0.1, f16=False):
    return entry("loom_hip_linear_attention_step", 7, ptrs, (*dims, ctypes.c_float(scale)), f16)


@pytest.mark.parametrize("f16", [False, True])
def test_null(f16):
    for f, args in ((window, (0, 1, 2, 3, 5)), (linear, (0, 1, 2, 3, 6, 7)),
                    (step, (0, 1, 2, 3, 4, 6))):
        for i in args:
            rc, msg = f({i: None}, f16=f16)
            assert rc == 1 and "null" in msg, (f, i, rc, msg)


def at(dims, i, x):
    return (*dims[:i], x, *dims[i + 1:])


@pytest.mark.parametrize("dims,code,word", [
    *[(at(W_DIMS, i, x), 1, "positive") for i in range(6) for x in (0, -1)],
    (at(W_DIMS, 6, 0), 1, "window"), (at(W_DIMS, 6, -5), 1, "window"),
    (at(W_DIMS, 7, -1), 1, "sinks"),
    (at(W_DIMS, 3, 60), 2, "head_dim"), (at(W_DIMS, 3, 264), 2, "head_dim"),
    (at(W_DIMS, 0, 70000), 1, "too large"), (at(W_DIMS, 4, 1 << 40), 1, "too large"),
    (at(W_DIMS, 5, 1 << 40), 1, "too large"), (at(W_DIMS, 2, 1 << 40), 1, "too large"),
    ((1 << 62, 1 << 62, 4, 64, 30, 128, 50, 4), 1, "too large"),
    ((1, 1, 1 << 29, 64, 1, 128, 50, 4), 1, "too large"),
    ((1, 1, 1, 256, 1, (1 << 22) + 1, 50, 4), 1, "D*S"),
])
def test_window_extents(dims, code, word):
    rc, msg = window(dims=dims)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("dims,code,word", [
    *[(at(L_DIMS, i, x), 1, "positive") for i in range(6) for x in (0, -1)],
    (at(L_DIMS, 3, 60), 2, "dim 60"), (at(L_DIMS, 3, 264), 2, "dim 264"),
    (at(L_DIMS, 4, 4), 2, "dim 4"), (at(L_DIMS, 4, 512), 2, "dim 512"),
    (at(L_DIMS, 5, 1 << 40), 1, "too large"), (at(L_DIMS, 0, 1 << 20), 1, "too large"),
    (at(L_DIMS, 1, 1 << 62), 1, "too large"), (at(L_DIMS, 2, (1 << 63) - 1), 1, "too large"),
])
def test_linear_extents(dims, code, word):
    rc, msg = linear(dims=dims)
    assert rc == code and word in msg, (rc, msg)
    if dims[5] == L_DIMS[5]:
        rc, msg = step(dims=dims[:5])
        assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_scale(scale):
    for f in (window, linear, step):
        rc, msg = f(scale=scale)
        assert rc == 1 and "scale" in msg, (f, rc, msg)


def test_alignment():
    for f, some in ((window, {0: 2, 1: 2, 2: 8, 3: 2, 4: 1, 5: 8}),
                    (linear, {0: 2, 1: 8, 2: 8, 3: 2, 4: 4, 5: 2, 6: 8, 7: 4}),
                    (step, {0: 2, 1: 8, 2: 8, 3: 2, 4: 4, 5: 2, 6: 8})):
        for i, off in some.items():
            rc, msg = f({i: P(i, off)})
            assert rc == 1 and "aligned" in msg, (f, i, rc, msg)
    # K rows off 16-byte boundaries need 2 bytes: past the checks of alignment
    rc, msg = window({0: P(0, 2), 5: P(3)}, dims=at(W_DIMS, 5, 127))
    assert rc == 1 and "overlap" in msg


def spans(f):
    """The bytes of a default call's tensors."""
    if f is window:
        B, G, H, D, T, S = W_DIMS[:6]
        cache, rows = B * G * S * D * 2, B * T * G * H * D * 2
        return [cache, cache, rows, 4 * B, 4 * B, rows,
                lh.window_attention_workspace_bytes(*W_DIMS)]
    B, G, H, D, E, T = L_DIMS if f is linear else (*L_DIMS[:5], 1)
    x = B * T * G * 2
    s = [x * H * D, x * D, x * E, G * H * 4, B * G * H * D * E * 4, 4 * B, x * H * E]
    if f is linear:
        s += [s[4], lh.linear_attention_workspace_bytes(*L_DIMS)]
    return s


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("f,outs,same", [(window, (5, 6), (5, 2)), (linear, (6, 7, 8), (7, 4)),
                                         (step, (4, 6), None)])
def test_overlaps(f, outs, same, f16):
    n = spans(f)
    for o in outs:
        for i in range(len(n)):
            if i == o or not n[o] or not n[i]:
                continue
            # the output begins 16 bytes before the other's end, or ends 16 past its start
            for to in (P(i, max(0, n[i] // 16 * 16 - 16)), P(i, 16 - n[o] // 16 * 16)):
                if to.value == P(i).value and same and {o, i} == set(same):
                    continue
                rc, msg = f({o: to}, f16=f16)
                assert rc == 1 and "overlap" in msg, (f, o, i, rc, msg)
    if same:      # in place, but then nothing else lies on the two
        o, i = same
        rc, msg = f({o: P(i), (3 if f is window else 5): P(i, 64)}, f16=f16)
        assert rc == 1 and "overlap" in msg
        rc, msg = f({o: P(i, 16)}, f16=f16)
        assert rc == 1 and "overlap" in msg


def test_workspaces():
    big = (1, 1, 4, 128, 1, 100000, 100000, 0)
    need = lh.window_attention_workspace_bytes(*big)
    if need:
        for ptrs, ws in (({}, need - 1), ({6: None}, need), ({6: P(6, 8)}, need)):
            rc, msg = window(ptrs, dims=big, ws=ws)
            assert rc == 1 and "workspace needs" in msg
    big = (1, 1, 1, 128, 128, 100000)
    need = lh.linear_attention_workspace_bytes(*big)
    if need:
        for ptrs, ws in (({}, need - 1), ({8: None}, need), ({8: P(8, 8)}, need)):
            rc, msg = linear(ptrs, dims=big, ws=ws)
            assert rc == 1 and "workspace needs" in msg


# ---- fuzzed: every call carries one thing that the last check refuses -------------

def refused(name, *args):
    rc, msg = call(name, *args)
    assert rc in (1, 2) and msg, (name, args, rc, msg)


@FUZZ
@given(st.booleans(), st.lists(pointers, min_size=7, max_size=7), st.integers(0, (1 << 64) - 1),
       st.lists(extents, min_size=8, max_size=8), st.floats(width=32))
def test_fuzz_window(f16, p, ws, dims, scale):
    p[5] = p[0]                       # out on k
    refused("loom_hip_window_attention" + ("_f16" if f16 else ""), *p, ws, *dims,
            ctypes.c_float(scale))


@FUZZ
@given(st.booleans(), st.lists(pointers, min_size=9, max_size=9), st.integers(0, (1 << 64) - 1),
       st.lists(extents, min_size=6, max_size=6), st.floats(width=32))
def test_fuzz_linear(f16, p, ws, dims, scale):
    x = "_f16" if f16 else ""
    p[6] = p[1]                       # out on k
    refused("loom_hip_linear_attention" + x, *p, ws, *dims, ctypes.c_float(scale))
    refused("loom_hip_linear_attention_step" + x, *p[:7], *dims[:5], ctypes.c_float(scale))


@FUZZ
@given(st.lists(extents, min_size=8, max_size=8))
def test_fuzz_workspace_bytes(dims):
    assert lh.window_attention_workspace_bytes(*dims) >= 0
    assert lh.linear_attention_workspace_bytes(*dims[:6]) >= 0


# ---- the Python calls --------------------------------------------------------------

_empty = torch.empty


@pytest.fixture
def made_up_device(monkeypatch):
    """Calls reach the C entry points with made-up pointers, far apart; any
    allocation of theirs fails the test."""
    def enter(func, tensors, extra=(), plan_of=None):
        sig = tuple(None if t is None else (t.dtype, t.shape) for t in tensors)
        return plan_of(func, sig, extra), 0, [None if t is None else FAR * (i + 1)
                                              for i, t in enumerate(tensors)]

    def empty(*a, **kw):
        raise AssertionError(f"allocates {a}")

    monkeypatch.setattr(lh, "_cache_enter", enter)
    monkeypatch.setattr(lh, "_current_device", lambda: 0)
    monkeypatch.setattr(lh, "_raw_stream", lambda i: None)
    monkeypatch.setattr(lh.torch, "empty", empty)


def meta(*shape, dtype=torch.bfloat16):
    return _empty(shape, dtype=dtype, device="meta")


i32, f32 = torch.int32, torch.float32


@pytest.mark.parametrize("window,sinks", [(0, 0), (-1, 0), (5, -1), (1 << 64, 0), (5, 1 << 63),
                                          ((1 << 64) + 5, 0), (-(1 << 64) + 5, 0)])
def test_windows_out_of_range(made_up_device, window, sinks):
    for T, f in ((3, lh.window_attention), (None, lh.window_decode)):
        q = meta(2, 3, 1, 2, 64) if T else meta(2, 1, 2, 64)
        with pytest.raises(lh.LoomHipError, match="window") as e:
            f(meta(2, 1, 64, 40), meta(2, 1, 40, 64), q, meta(2, dtype=i32), window, sinks=sinks)
        assert e.value.code == 1


def test_calls_too_large_say_so(made_up_device):
    B, S = 70000, 8
    with pytest.raises(lh.LoomHipError, match="too large"):
        lh.window_decode(meta(B, 1, 8, S), meta(B, 1, S, 8), meta(B, 1, 1, 8), meta(B, dtype=i32),
                         4, meta(B, 1, 1, 8))
    B = (1 << 20) + 1
    for f, T in ((lh.linear_attention, (2,)), (lh.linear_attention_step, ())):
        a = [meta(B, *T, 1, 1, 8), meta(B, *T, 1, 8), meta(B, *T, 1, 8), meta(1, 1, dtype=f32),
             meta(B, 1, 1, 8, 8, dtype=f32), meta(B, *T, 1, 1, 8)]
        with pytest.raises(lh.LoomHipError, match="too large"):
            f(*a, *([a[4]] if T else []))


def cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def window_args(T=3):
    q = cpu(2, T, 1, 2, 64) if T else cpu(2, 1, 2, 64)
    return [cpu(2, 1, 64, 40), cpu(2, 1, 40, 64), q, cpu(2, dtype=i32)]


def linear_args(T=3):
    t = (T,) if T else ()
    return [cpu(2, *t, 1, 2, 64), cpu(2, *t, 1, 64), cpu(2, *t, 1, 32), cpu(1, 2, dtype=f32),
            cpu(2, 1, 2, 64, 32, dtype=f32)]


@pytest.mark.parametrize("call,args,names", [
    (lambda *a: lh.window_attention(*a, 5), window_args(), ["k", "v", "q", "lens"]),
    (lambda *a: lh.window_decode(*a, 5), window_args(None), ["k", "v", "q", "lens"]),
    (lh.linear_attention, linear_args(), ["q", "k", "v", "log_decay", "state"]),
    (lh.linear_attention_step, linear_args(None), ["q", "k", "v", "log_decay", "state"]),
], ids=["window_attention", "window_decode", "linear_attention", "linear_attention_step"])
def test_python_names_what_is_wrong(call, args, names):
    with pytest.raises(ValueError, match="ROCm device"):          # all of them well-formed
        call(*args)
    for i, name in enumerate(names):
        for bad, error in ((args[i].double(), TypeError), (args[i].unsqueeze(0), ValueError),
                           (torch.cat([args[i], args[i]], 0), ValueError), (3, TypeError)):
            with pytest.raises(error) as e:
                call(*args[:i], bad, *args[i + 1:])
            assert isinstance(bad, int) or any(n in str(e.value) for n in names), (name, e.value)
        if args[i].dim() > 1:
            t = args[i].transpose(-1, -2).contiguous().transpose(-1, -2)
            if not t.is_contiguous():
                with pytest.raises(ValueError, match=f"{name}: must be contiguous"):
                    call(*args[:i], t, *args[i + 1:])


def test_python_optional_tensors():
    for kw, error in (({"counts": cpu(3, dtype=i32)}, ValueError),
                      ({"counts": cpu(2, dtype=torch.int64)}, TypeError),
                      ({"out": cpu(2, 3, 1, 2, 64, dtype=torch.float16)}, TypeError),
                      ({"out": cpu(2, 1, 1, 2, 64)}, ValueError)):
        with pytest.raises(error, match=next(iter(kw))):
            lh.window_attention(*window_args(), 5, **kw)
    for kw, error in (({"counts": cpu(3, dtype=i32)}, ValueError),
                      ({"out": cpu(2, 3, 1, 2, 64)}, ValueError),
                      ({"state_out": cpu(2, 1, 2, 64, 32)}, TypeError),
                      ({"state_out": cpu(2, 1, 2, 32, 64, dtype=f32)}, ValueError)):
        with pytest.raises(error, match=next(iter(kw))):
            lh.linear_attention(*linear_args(), **kw)
    with pytest.raises(TypeError, match="state"):
        lh.linear_attention_step(*linear_args(None)[:4], None)
