"""Which packed calls divide a block's keys (they then ask for a workspace): those that were measured faster so (CPU)."""
import pytest

from mica_amd import _lib


def divided(counts, HK):
    return _lib.load().mica_attention_packed_workspace_bytes(len(counts), sum(counts), HK, max(counts)) > 0


@pytest.mark.parametrize("counts,HK", [
    ([768], 4), ([1000], 4), ([2017], 4), ([2018], 4), ([2048], 4), ([2300], 4), ([2400], 4), ([1000, 250], 4), ([1000, 500], 4),
    ([1500] + [50] * 10, 4), ([1000] * 4, 1), ([2000] * 4, 1), ([5000], 2), ([10000], 1), ([1500] + [50] * 50, 1), ([1000], 6)])
def test_divided(counts, HK):
    assert divided(counts, HK)


@pytest.mark.parametrize("counts,HK", [
    ([300], 4), ([2600], 4), ([3000], 4), ([768, 768], 4), ([900, 900], 4), ([950, 950], 4), ([1000, 1000], 4), ([1500, 1500], 4),
    ([768] * 4, 4), ([1000] * 8, 1), ([1000], 8), ([1500, 1125], 4), ([2000] + [100] * 20, 4), ([1000] + [30] * 60, 4)])
def test_not_divided(counts, HK):
    assert not divided(counts, HK)


@pytest.mark.parametrize("T", [2000, 2400, 9600])
def test_states_of_many_sequences_stay_small(T):
    """The most blocks that the call could have bound the states, not its rows: 320 blocks and heads x 3 chunks x 128 rows."""
    for B in (1, 10, 100, 1000):
        for HK in (1, 2, 4):
            n = _lib.load().mica_attention_packed_workspace_bytes(B, T, HK, min(1500, T))
            assert 0 <= n <= 320 * 3 * 128 * 1032


@pytest.mark.parametrize("B,T,HK,want", [(4, 1600, 4, False), (5, 1500, 4, False), (3, 1800, 4, False), (8, 1600, 4, False),
                                         (10, 4000, 1, False), (1, 1000, 4, True), (1, 2048, 4, True), (4, 4000, 1, True)])
def test_without_a_hint_as_if_all_had_as_many_rows(B, T, HK, want):
    """A batch of short prompts asks for no division that none of its blocks would take."""
    assert (_lib.load().mica_attention_packed_workspace_bytes(B, T, HK, 0) > 0) == want
