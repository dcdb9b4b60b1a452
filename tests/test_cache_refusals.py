"""What the Python calls of the cache operators refuse before they allocate
anything (CPU only: tensors on the meta device stand for large ones, the device
is made up and nothing is launched)."""
import pytest
import torch

import loom_hip as lh

FAR = 1 << 40
_empty = torch.empty


@pytest.fixture
def made_up_device(monkeypatch):
    """Calls reach the C entry points with made-up pointers, far apart; any
    allocation of theirs fails the test."""
    def enter(func, tensors, extra=()):
        sig = tuple(None if t is None else (t.dtype, t.shape) for t in tensors)
        return lh._cache_plan(func, sig, extra), 0, [None if t is None else FAR * (i + 1)
                                                      for i, t in enumerate(tensors)]

    def empty(*a, **kw):
        raise AssertionError(f"allocates {a}")

    monkeypatch.setattr(lh, "_cache_enter", enter)
    monkeypatch.setattr(lh, "_current_device", lambda: 0)
    monkeypatch.setattr(lh, "_raw_stream", lambda i: None)
    monkeypatch.setattr(lh.torch, "empty", empty)


def meta(*shape, dtype=torch.bfloat16):
    return _empty(shape, dtype=dtype, device="meta")


def decode(B, G, H, D, P, S, **kw):
    return lh.cache_decode(meta(B, G, D, S), meta(B, G, S, D), meta(B, G, H, D),
                           meta(B, dtype=torch.int32), meta(B, G, H, D),
                           prefix_k=meta(G, D, P) if P else None,
                           prefix_v=meta(G, P, D) if P else None, **kw)


@pytest.mark.parametrize("dims", [(70000, 1, 1, 8, 0, 8), (256, 256, 1, 8, 0, 8),
                                  (1, 1, 1 << 24, 8, 0, 8), (1, 1, 1, 8, 0, (1 << 29) + 8),
                                  (1, 1, 1, 8, (1 << 29) + 8, 8)])
def test_a_step_too_large_says_so(made_up_device, dims):
    with pytest.raises(lh.LoomHipError, match="too large") as e:
        decode(*dims)
    assert e.value.code == 1
    # also with a workspace, which no size would suit
    with pytest.raises(lh.LoomHipError, match="too large"):
        decode(*dims, workspace=meta(64, dtype=torch.uint8))


def test_no_workspace_is_that_large():
    with pytest.raises(ValueError, match="too large"):
        lh.cache_decode_workspace(70000, 1, 1, 8, 0, 8, False, "cpu")
    assert lh.cache_decode_workspace(2, 1, 1, 8, 0, 8, False, "cpu").numel() == \
        lh.cache_decode_workspace_bytes(2, 1, 1, 8, 0, 8)


def evict(keep, S=64, **kw):
    return lh.cache_evict(meta(2, 1, 8, S), meta(2, 1, S, 8), meta(2, 1, S, dtype=torch.float32),
                          meta(2, dtype=torch.int32), keep, **kw)


@pytest.mark.parametrize("keep,kw", [
    (65, {}), (1 << 40, {}), (1 << 64, {}), (33, {"capacity": 32}), ((1 << 64) + 5, {}),
    (8, {"recent": 9}), (8, {"recent": -1}), (8, {"sinks": -1}), (8, {"recent": 4, "sinks": 5}),
    # a multiple of 2^64 more than what would fit
    (8, {"recent": 1 << 64}), (8, {"sinks": (1 << 64) + 2}), (8, {"recent": -(1 << 64)}),
])
def test_evict_keeps_at_most_the_capacity(made_up_device, keep, kw):
    with pytest.raises(lh.LoomHipError, match="keep") as e:
        evict(keep, **kw)
    assert e.value.code == 1
