"""How group norm cuts its work, without a GPU."""
from opendressi_amd._lib import lib


def _scratch(n, px, c, groups, backward, kind=0):
    return lib.dressi_group_norm_scratch(kind, n, px, c, px * c, c, groups, 0, backward)


def test_blocks_stay_within_a_launch():
    """A workgroup for each group, in one pass, is a launch's y dimension: where they are more than
    65535, two passes over blocks of many groups, which need scratch between them."""
    for groups, two in ((65535, False), (65536, True), (131072, True), (2 ** 20, True)):
        assert (_scratch(1, 4096, groups, groups, 0) > 0) == two, groups
        assert (_scratch(1, 2048, groups, groups, 1) > 8 * groups) == two, groups
    # few pixels: a workgroup takes several groups
    assert _scratch(1, 64, 2 ** 20, 2 ** 20, 0) == 0
