"""Refusals of the cache operators, without a GPU: the C entry points reject bad
arguments before anything is launched, and the Python calls name the tensor
that is wrong."""
import ctypes

import pytest
import torch

import loom_hip as lh

FAR = 1 << 40     # made-up addresses, far from each other and never dereferenced


def P(i, off=0):
    return ctypes.c_void_p(FAR * (i + 1) + off)


def call(name, *args):
    buf = ctypes.create_string_buffer(256)
    rc = getattr(lh._lib, name)(*args, None, buf, len(buf))
    return rc, buf.value.decode()


def append(ptrs=None, dims=(2, 2, 64, 128, 4)):
    a = [P(i) for i in range(8)]
    for i, v in (ptrs or {}).items():
        a[i] = v
    return call("loom_hip_cache_append", *a, *dims)


def evict(ptrs=None, dims=(2, 2, 64, 128, 64, 32, 4, 2)):
    a = [P(i) for i in range(9)]
    for i, v in (ptrs or {}).items():
        a[i] = v
    return call("loom_hip_cache_evict", *a, *dims)


def decode(ptrs=None, dims=(2, 2, 4, 64, 64, 128), scale=0.1, ws=1 << 40, f16=False):
    a = [P(i) for i in range(10)]
    for i, v in (ptrs or {}).items():
        a[i] = v
    return call("loom_hip_cache_decode" + ("_f16" if f16 else ""), *a, ws, *dims,
                ctypes.c_float(scale))


@pytest.mark.parametrize("arg", [0, 1, 3, 4, 5, 7])
def test_append_null(arg):
    rc, msg = append({arg: None})
    assert rc == 1 and "null" in msg


@pytest.mark.parametrize("dims,code,word", [
    ((0, 2, 64, 128, 4), 1, "positive"), ((2, 2, 64, 128, 0), 1, "positive"),
    ((2, -1, 64, 128, 4), 1, "positive"), ((2, 2, 60, 128, 4), 2, "head_dim"),
    ((2, 2, 264, 128, 4), 2, "head_dim"), ((70000, 1, 64, 128, 4), 1, "too large"),
    ((2, 2, 64, 1 << 40, 4), 1, "too large"), ((2, 2, 64, 128, 1 << 40), 1, "too large"),
    ((1 << 62, 1 << 62, 64, 128, 4), 1, "too large"),
])
def test_append_extents(dims, code, word):
    rc, msg = append(dims=dims)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("ptrs,word", [
    ({0: P(0, 2)}, "aligned"), ({1: P(1, 2)}, "aligned"), ({4: P(4, 8)}, "aligned"),
    ({5: P(5, 2)}, "aligned"), ({3: P(3, 2)}, "aligned"), ({2: P(2, 2)}, "aligned"),
    ({7: P(3)}, "overlap"), ({7: P(3, 4)}, "overlap"), ({7: P(6)}, "overlap"),
    ({4: P(0, 4096)}, "overlap"), ({5: P(1)}, "overlap"), ({1: P(0)}, "overlap"),
    ({2: P(0, 64)}, "overlap"), ({3: P(1, 64)}, "overlap"), ({7: P(2, 4)}, "overlap"),
])
def test_append_pointers(ptrs, word):
    rc, msg = append(ptrs)
    assert rc == 1 and word in msg, (rc, msg)


@pytest.mark.parametrize("arg", range(9))
def test_evict_null(arg):
    rc, msg = evict({arg: None})
    assert rc == 1 and "null" in msg


@pytest.mark.parametrize("dims,code,word", [
    ((2, 0, 64, 128, 64, 32, 4, 2), 1, "positive"), ((2, 2, 64, 128, 0, 32, 4, 2), 1, "positive"),
    ((2, 2, 64, 128, 64, 0, 0, 0), 1, "keep"), ((2, 2, 64, 128, 64, 65, 4, 2), 1, "keep"),
    ((2, 2, 64, 128, 64, 32, 33, 0), 1, "keep"), ((2, 2, 64, 128, 64, 32, 31, 2), 1, "keep"),
    ((2, 2, 64, 128, 64, 32, -1, 2), 1, "keep"), ((2, 2, 64, 128, 64, 32, 4, -2), 1, "keep"),
    ((2, 2, 64, 128, 64, 32, 4, (1 << 63) - 1), 1, "keep"),
    ((2, 2, 4, 128, 64, 32, 4, 2), 2, "head_dim"),
    ((256, 256, 64, 128, 64, 32, 4, 2), 1, "too large"),
    ((2, 2, 64, 1 << 31, 64, 32, 4, 2), 1, "too large"),
])
def test_evict_extents(dims, code, word):
    rc, msg = evict(dims=dims)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("ptrs,word", [
    ({0: P(0, 2)}, "aligned"), ({4: P(4, 8)}, "aligned"), ({5: P(5, 2)}, "aligned"),
    ({2: P(2, 2)}, "aligned"), ({4: P(0)}, "overlap"), ({5: P(1, 64)}, "overlap"),
    ({6: P(2)}, "overlap"), ({7: P(3)}, "overlap"), ({8: P(2, 256)}, "overlap"),
    ({8: P(6)}, "overlap"), ({5: P(4, 64)}, "overlap"),
])
def test_evict_pointers(ptrs, word):
    rc, msg = evict(ptrs)
    assert rc == 1 and word in msg, (rc, msg)


@pytest.mark.parametrize("f16", [False, True])
def test_decode_pointers(f16):
    for arg in (2, 3, 4, 5, 8):
        rc, msg = decode({arg: None}, f16=f16)
        assert rc == 1 and "null" in msg
    for arg in (0, 1):
        rc, msg = decode({arg: None}, f16=f16)
        assert rc == 1 and "prefix" in msg
    rc, msg = decode(dims=(2, 2, 4, 64, 0, 128), f16=f16)     # a prefix of no keys
    assert rc == 1 and "prefix" in msg
    for arg in (6, 7):
        rc, msg = decode({arg: None}, f16=f16)
        assert rc == 1 and "together" in msg
    rc, msg = decode({7: P(6, 16)}, f16=f16)
    assert rc == 1 and "overlap" in msg
    for arg, off in ((0, 8), (1, 8), (2, 2), (3, 2), (4, 8), (5, 2), (6, 2), (8, 2)):
        rc, msg = decode({arg: P(arg, off)}, f16=f16)
        assert rc == 1 and "aligned" in msg, (arg, msg)
    rc, msg = decode({9: None}, f16=f16)
    assert rc == 1 and "workspace" in msg
    need = lh.cache_decode_workspace_bytes(2, 2, 4, 64, 64, 128, True)
    rc, msg = decode(ws=need - 1, f16=f16)
    assert rc == 1 and "workspace" in msg


@pytest.mark.parametrize("dims,code,word", [
    ((0, 2, 4, 64, 64, 128), 1, "positive"), ((2, 2, 0, 64, 64, 128), 1, "positive"),
    ((2, 2, 4, 64, -1, 128), 1, "positive"), ((2, 2, 4, 64, 64, 0), 1, "positive"),
    ((2, 2, 4, 68, 64, 128), 2, "head_dim"), ((2, 2, 4, 512, 64, 128), 2, "head_dim"),
    ((2, 2, 4, 64, 1 << 31, 128), 1, "too large"), ((65536, 1, 4, 64, 64, 128), 1, "too large"),
    ((2, 2, 1 << 40, 64, 64, 128), 1, "too large"),
    ((1, 1, 1, 256, 64, (1 << 23) + 1), 1, "multiple of 8"),
    ((1, 1, 1, 256, (1 << 23) + 1, 64), 1, "multiple of 8"),
])
def test_decode_extents(dims, code, word):
    rc, msg = decode(dims=dims)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_decode_scale(scale):
    rc, msg = decode(scale=scale)
    assert rc == 1 and "scale" in msg


def test_workspace_bytes():
    w = lh.cache_decode_workspace_bytes
    assert w(0, 1, 1, 64, 0, 64) == 0
    assert w(1, 1, 1, 64, -1, 64) == 0
    assert w(1 << 40, 1 << 40, 1, 64, 0, 64) == (1 << 64) - 1
    assert w(1, 1, 1 << 50, 64, 1 << 50, 64, True) == (1 << 64) - 1
    # gathering weights never takes less
    assert w(4, 2, 8, 128, 100, 1000, True) >= w(4, 2, 8, 128, 100, 1000) > 0


# ---- Python: what is wrong with which tensor, before a device is needed ------

def tensors(B=2, G=2, H=4, D=64, P=16, S=24, T=3, dtype=torch.bfloat16):
    t = {"k": torch.zeros(B, G, D, S, dtype=dtype), "v": torch.zeros(B, G, S, D, dtype=dtype),
         "q": torch.zeros(B, G, H, D, dtype=dtype), "lens": torch.zeros(B, dtype=torch.int32),
         "prefix_k": torch.zeros(G, D, P, dtype=dtype), "prefix_v": torch.zeros(G, P, D, dtype=dtype),
         "weights": torch.zeros(B, G, S), "new_k": torch.zeros(B, T, G, D, dtype=dtype),
         "new_v": torch.zeros(B, T, G, D, dtype=dtype), "counts": torch.zeros(B, dtype=torch.int32)}
    return t


def go(func, t, **kw):
    if func == "decode":
        return lh.cache_decode(t["k"], t["v"], t["q"], t["lens"], prefix_k=t["prefix_k"],
                               prefix_v=t["prefix_v"], weights=t["weights"], **kw)
    if func == "append":
        return lh.cache_append(t["k"], t["v"], t["lens"], t["new_k"], t["new_v"],
                               counts=t["counts"], weights=t["weights"], **kw)
    return lh.cache_evict(t["k"], t["v"], t["weights"], t["lens"], 8, **kw)


@pytest.mark.parametrize("func", ["decode", "append", "evict"])
def test_python_needs_a_device(func):
    for dtype in (torch.bfloat16, torch.float16):
        with pytest.raises(ValueError, match="k: must be on a ROCm device"):
            go(func, {**tensors(dtype=dtype), **({"prefix_k": None, "prefix_v": None})})


BAD = [
    ("decode", "k", torch.zeros(2, 2, 64, 24), TypeError, "bfloat16"),
    ("decode", "k", torch.zeros(2, 64, 24, dtype=torch.bfloat16), ValueError, "4 dims"),
    ("decode", "k", None, ValueError, "4 dims"),
    ("decode", "v", torch.zeros(2, 2, 25, 64, dtype=torch.bfloat16), ValueError, "v: expected shape"),
    ("decode", "v", torch.zeros(2, 2, 24, 64, dtype=torch.float16), TypeError, "v: expected"),
    ("decode", "q", torch.zeros(2, 2, 4, 32, dtype=torch.bfloat16), ValueError, "q: expected shape"),
    ("decode", "q", torch.zeros(2, 8, 64, dtype=torch.bfloat16), ValueError, "4 dims"),
    ("decode", "lens", torch.zeros(2, dtype=torch.int64), TypeError, "lens: expected torch.int32"),
    ("decode", "lens", torch.zeros(3, dtype=torch.int32), ValueError, "lens: expected shape"),
    ("decode", "lens", [1, 2], TypeError, "torch.Tensor"),
    ("decode", "lens", None, TypeError, "lens"),
    ("decode", "weights", torch.zeros(2, 2, 24, dtype=torch.float64), TypeError, "weights"),
    ("decode", "weights", torch.zeros(2, 24), ValueError, "weights: expected shape"),
    ("decode", "prefix_k", None, ValueError, "together"),
    ("decode", "prefix_v", None, ValueError, "together"),
    ("decode", "prefix_k", torch.zeros(2, 16, 64, dtype=torch.bfloat16), ValueError, "prefix_k"),
    ("decode", "prefix_k", torch.zeros(64, 16, dtype=torch.bfloat16), ValueError, "3 dims"),
    ("append", "new_k", torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16), ValueError, "new_k"),
    ("append", "new_k", torch.zeros(2, 2, 64, dtype=torch.bfloat16), ValueError, "4 dims"),
    ("append", "new_v", torch.zeros(2, 3, 2, 64, dtype=torch.float16), TypeError, "new_v"),
    ("append", "counts", torch.zeros(2), TypeError, "counts"),
    ("append", "weights", torch.zeros(2, 2, 25), ValueError, "weights: expected shape"),
    ("evict", "weights", torch.zeros(2, 2, 24, dtype=torch.bfloat16), TypeError, "weights"),
    ("evict", "weights", None, TypeError, "weights"),
]


@pytest.mark.parametrize("func,name,value,exc,word", BAD,
                         ids=[f"{c[0]}-{c[1]}-{i}" for i, c in enumerate(BAD)])
def test_python_names_the_tensor(func, name, value, exc, word):
    t = tensors()
    t[name] = value
    with pytest.raises(exc, match=word):
        go(func, t)


def test_python_contiguity_and_outputs():
    t = tensors(D=24)
    t["k"] = torch.zeros(2, 2, 24, 24, dtype=torch.bfloat16).transpose(2, 3)
    with pytest.raises(ValueError, match="k: must be contiguous"):
        go("evict", t)
    t = tensors()
    with pytest.raises(ValueError, match="k_out: expected shape"):
        go("evict", t, capacity=16, k_out=torch.zeros(2, 2, 64, 20, dtype=torch.bfloat16))
    # the capacity of one output given holds for the others
    with pytest.raises(ValueError, match="v_out: expected shape"):
        go("evict", t, k_out=torch.zeros(2, 2, 64, 16, dtype=torch.bfloat16),
           v_out=torch.zeros(2, 2, 20, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="index: expected shape"):
        go("evict", t, index=torch.zeros(2, 2, 9, dtype=torch.int32))
    with pytest.raises(ValueError, match="out: expected shape"):
        go("decode", t, out=torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16))
    t["weights"] = None
    with pytest.raises(ValueError, match="weights_out needs weights"):
        go("decode", t, weights_out=torch.zeros(2, 2, 24))
