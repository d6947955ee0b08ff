"""How many tiles of 32 tokens a block of the selective scan's gradient takes, seen in the workspace that it asks for: one
while the card holds the blocks less than twice, then two.  A compute unit's 160 KB of LDS hold three blocks, of 64 states two
(64512 bytes each)."""

import pytest

from boltz_lumi_amd import _native as N


def ranges(b, t, c, n, groups):
    """Ranges of tiles of a sequence, from the parts of the workspace: per range the carried states and the steps, and the
    partial sums dA, dD and the bias's; a group's channels are one span here, so there are none for the maps."""
    floats = N.lib().bmx_selective_scan_bwd_workspace_bytes(b, t, c, n, groups) // 4
    parts, rest = divmod(floats, 2 * c * n + 3 * c)
    assert rest == 0 and parts % b == 0
    return parts // b


@pytest.mark.parametrize("n,held", [(8, 768), (16, 768), (32, 768), (64, 512)])
def test_two_tiles_where_that_is_a_round(n, held):
    groups, tiles = 32, 4
    b = 2 * held // (groups * tiles)
    assert ranges(b, 32 * tiles, 8 * groups, n, groups) == tiles // 2
    assert ranges(b - 1, 32 * tiles, 8 * groups, n, groups) == tiles
    assert ranges(b, 32 * tiles + 1, 8 * groups, n, groups) == tiles // 2 + 1
