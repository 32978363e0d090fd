"""Sizes of the scoring operators' plans (CPU)."""
import pytest

from mica_amd import _lib


@pytest.mark.parametrize("B,N", [(32769, 512), (87382, 512), (52429, 289), (104858, 129), (1864134, 65)])
def test_no_grid_of_two_to_the_32_work_items(B, N):
    """A long cache's tiles would be divided for so many blocks of queries, too: the join's grid (64 x 32 x 4 work-items a
    block) or the attention's own would wrap round.  Undivided there, as the missing workspace shows."""
    blocks = B * -(-N // 32)
    assert blocks * 8192 >= 2 ** 32 or 2 * blocks * 256 * 64 >= 2 ** 32
    assert _lib.load().mica_attention_tree_workspace_bytes(B, N, 1, 2 ** 31 - 1) == 0
    assert _lib.load().mica_attention_window_workspace_bytes(B, N, 2 ** 31 - 1, 1, 2 ** 31 - 1, 0) == 0


def test_division_below_that():
    """The bound takes no ordinary division away: partial rows of 1032 bytes, 128 a workgroup."""
    size = _lib.load().mica_attention_tree_workspace_bytes
    assert size(2, 255, 4, 3000) == 256 * 128 * 1032
    assert size(1, 65, 4, 1000) > 0 and size(16383, 512, 1, 2 ** 31 - 1) >= 0
