"""How the backward of a norm and a joint splits rows among blocks: groups of which several blocks have a part each, blocks
that have several groups, rows gone over in passes and rows in registers of one, four and eight waves."""
from __future__ import annotations

import pytest

from tests.test_gpu_norm import Joint

pytestmark = pytest.mark.gpu


# rows beyond 8192 values (with 9 strips of columns) and below 4: pieces of a group, no groups, more groups than blocks
@pytest.mark.parametrize("m,n,groups", [(300, 9001, 0), (300, 9001, 1), (300, 9001, 2), (400, 8200, 200), (5000, 3, 0),
                                        (5000, 3, 1), (5000, 3, 5), (5000, 3, 2500), (3000, 1, 1000), (3000, 2, 3)])
@pytest.mark.parametrize("post,next,p", [("layer", "rms", 0.1), ("none", "none", 0.0)])
def test_rows_in_passes(ctx, m, n, groups, post, next, p):
    print(f"passes {m} x {n} groups {groups} {post} {next}", flush=True)
    Joint(ctx, m + n + groups, m, n, post, next, groups, p).check()


# two rows a group and more groups than blocks: a block's second group and on
@pytest.mark.parametrize("m,n,groups", [(2200, 900, 1100), (1200, 1100, 600), (1200, 2600, 600), (700, 4100, 350),
                                        (1101, 1501, 367)])
@pytest.mark.parametrize("post,next,p,bias", [("layer", "layer", 0.1, True), ("rms", "none", 0.2, False),
                                              ("none", "rms", 0.0, True)])
def test_several_groups_a_block(ctx, m, n, groups, post, next, p, bias):
    print(f"groups {m} x {n} groups {groups} {post} {next}", flush=True)
    Joint(ctx, m + n + groups, m, n, post, next, groups, p, bias=bias).check()


# a few groups of many rows: pieces of a group in registers
@pytest.mark.parametrize("m,n,groups", [(900, 700, 3), (600, 1501, 2), (600, 3001, 4), (400, 8000, 2)])
def test_pieces_of_a_group(ctx, m, n, groups):
    print(f"pieces {m} x {n} groups {groups}", flush=True)
    Joint(ctx, m + n + groups, m, n, "layer", "rms", groups, 0.1).check()
