"""cache_decode refuses outputs and workspaces that share a byte with another
tensor, as cache_append and cache_evict do (CPU only: nothing is launched)."""
import pytest

import loom_hip as lh
from tests.test_cache_validation import P, decode

# prefix_k, prefix_v, k, v, q, lens, weights, weights_out, out, workspace of the
# default call (B2 G2 H4 D64 P64 S128): their bytes
DIMS = (2, 2, 4, 64, 64, 128)
BYTES = [2 * 64 * 64 * 2] * 2 + [2 * 2 * 128 * 64 * 2] * 2 + \
    [2 * 2 * 4 * 64 * 2, 2 * 4, 2 * 2 * 128 * 4, 2 * 2 * 128 * 4, 2 * 2 * 4 * 64 * 2,
     lh.cache_decode_workspace_bytes(*DIMS, True)]
OUT, WEIGHTS_OUT, WORKSPACE, Q, WEIGHTS = 8, 7, 9, 4, 6


def pairs():
    for o in (WEIGHTS_OUT, OUT, WORKSPACE):
        for i in range(10):
            if i != o:
                yield o, i


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("o,i", pairs())
def test_decode_overlaps(o, i, f16):
    # the output begins 16 bytes before the other's end, or ends 16 bytes past its start
    for at in (P(i, max(0, BYTES[i] // 16 * 16 - 16)), P(i, 16 - BYTES[o] // 16 * 16)):
        rc, msg = decode({o: at}, f16=f16)
        assert rc == 1 and "overlap" in msg, (o, i, msg)
    # beside it is fine: what is refused then is the workspace's size, looked at before
    rc, msg = decode({o: P(i, (BYTES[i] + 15) // 16 * 16)}, ws=BYTES[WORKSPACE] - 1, f16=f16)
    assert rc == 1 and "workspace needs" in msg, (o, i, msg)


@pytest.mark.parametrize("o,i", [(WEIGHTS_OUT, WEIGHTS), (OUT, Q)])
def test_decode_in_place(o, i):
    """weights_out may be weights and out may be q, but nothing else then lies on them."""
    rc, msg = decode({o: P(i), WORKSPACE: P(i, 256)})
    assert rc == 1 and "overlap" in msg, msg
    rc, msg = decode({o: P(i, 16)})
    assert rc == 1 and "overlap" in msg, msg
