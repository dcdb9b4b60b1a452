"""Fuzzing the argument checks of the cache operators' entry points (CPU only):
any extents, pointers and sizes are refused with a code and a message.  Every
call carries one thing that the last of its checks refuses (two outputs on each
other, no workspace), so nothing is ever launched.  Runs again under the
sanitizers (test_cache_sanitizers.py), where a signed overflow or an access out
of bounds ends the run."""
import ctypes

from hypothesis import given
from hypothesis import strategies as st

import loom_hip
from tests.test_fuzz_abi import FUZZ

extents = st.one_of(st.integers(-2, 300), st.integers(1, 1 << 31),
                    st.integers(-(1 << 62), 1 << 62),
                    st.sampled_from([8, 64, 128, 256, 1 << 20, 1 << 23, 1 << 29, (1 << 29) + 1,
                                     65535, 65536, (1 << 63) - 1, -(1 << 63)]))
pointers = st.one_of(st.none(), st.integers(0, 4096), st.integers(0, 1 << 60),
                     st.integers(1, 1 << 20).map(lambda x: x << 40))


def refused(name, *args):
    buf = ctypes.create_string_buffer(256)
    rc = getattr(loom_hip._lib, name)(*args, None, buf, len(buf))
    assert rc in (1, 2) and buf.value, (name, args, rc, buf.value)


@FUZZ
@given(st.lists(pointers, min_size=8, max_size=8), st.lists(extents, min_size=5, max_size=5))
def test_append(p, dims):
    p[1] = p[0]                       # k and v
    refused("loom_hip_cache_append", *p, *dims)


@FUZZ
@given(st.lists(pointers, min_size=9, max_size=9), st.lists(extents, min_size=8, max_size=8))
def test_evict(p, dims):
    p[5] = p[4]                       # k_out and v_out
    refused("loom_hip_cache_evict", *p, *dims)


@FUZZ
@given(st.booleans(), st.lists(pointers, min_size=9, max_size=9), st.integers(0, (1 << 64) - 1),
       st.lists(extents, min_size=6, max_size=6), st.floats(width=32))
def test_decode(f16, p, ws, dims, scale):
    # no workspace, then one that out lies on
    for last in (None, p[8]):
        refused("loom_hip_cache_decode" + ("_f16" if f16 else ""), *p, last, ws, *dims,
                ctypes.c_float(scale))


@FUZZ
@given(st.lists(extents, min_size=6, max_size=6), st.booleans())
def test_workspace_bytes(dims, weights):
    n = loom_hip.cache_decode_workspace_bytes(*dims, weights)
    B, G, H, D, P, S = dims
    if min(B, G, H, D, S) <= 0 or P < 0:
        assert n == 0
    else:
        assert n > 0
