"""How calls of windowed attention are launched, by the workspace that they ask for (none:
every tile of rows is one workgroup's)."""
import pytest

import loom_hip as lh


@pytest.mark.parametrize("D,H,T,B", [(128, 4, 2048, 1), (128, 4, 512, 4), (128, 4, 1024, 1),
                                     (128, 4, 512, 1), (96, 4, 2048, 1), (96, 4, 1024, 1),
                                     (64, 4, 2048, 1), (256, 2, 2048, 1)])
@pytest.mark.parametrize("window", [128, 1024, 8192])
def test_a_full_round_of_large_tiles_is_not_split(D, H, T, B, window):
    """256 tiles of 64, 128 or 256 rows, one to a CU: two halves of each would take two
    rounds and a join."""
    rows = T * H * B * 8
    assert rows in (256 * 64, 256 * 128, 256 * 256)
    assert lh.window_attention_workspace_bytes(B, 8, H, D, T, max(T, window), window, 4) == 0


def test_few_rows_and_small_tiles_are_split():
    """Fewer workgroups than fit, or tiles of which two fit a CU under a long window."""
    for D in (64, 96, 128, 256):
        assert lh.window_attention_workspace_bytes(1, 1, 32, D, 1, 4096, 512, 4)
    assert lh.window_attention_workspace_bytes(1, 8, 4, 64, 1024, 8192, 8192, 4)
    assert lh.window_attention_workspace_bytes(1, 8, 4, 96, 512, 8192, 8192, 4)
    assert not lh.window_attention_workspace_bytes(1, 8, 4, 64, 1024, 2048, 1024, 4)
    assert not lh.window_attention_workspace_bytes(1, 8, 4, 96, 512, 2048, 1024, 4)


@pytest.mark.parametrize("G,T,segments", [(1, 8192, 64), (2, 2048, 16), (16, 512, 4), (4, 4096, 32),
                                          (32, 32768, 8), (256, 4096, 0)])
def test_a_prompt_s_segments_leave_one_state_each(G, T, segments):
    """The workspace holds a state to each segment: none is cut any further for the first
    launch, whose states every segment's start adds up."""
    assert lh.linear_attention_workspace_bytes(1, G, 1, 128, 128, T) == G * segments * 128 * 128 * 4
