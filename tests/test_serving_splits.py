"""The split counts that the serving calls choose (CPU only)."""

from __future__ import annotations

import pytest

from tqb.serving import _splits


@pytest.mark.parametrize("group,groups", [(1, 296), (4, 296), (5, 148), (8, 148)])
@pytest.mark.parametrize("items,tokens", [(296, 777), (512, 1024), (64, 2048), (128, 3000), (8, 4096), (1184, 512), (5000, 300)])
def test_splits_fill_the_rounds_of_their_kernel(group, groups, items, tokens):
    """Two groups of warps to an SM up to 4 query heads a KV head, one above; 8 (sequence, head, split) items a group.  One
    more split than chosen takes another round, unless splits would fall below 32 tokens or hold fewer pages."""
    s = _splits(items, tokens, group)
    rounds = lambda n: -(-items * n // (8 * groups))  # noqa: E731
    pages = -(-tokens // 16)
    more = s + 1
    while -(-pages // more) == -(-pages // s):  # the next count with fewer pages to a split
        more += 1
    assert rounds(more) > rounds(s) or tokens < 32 * more


def test_splits_of_known_shapes():
    assert [_splits(296, 777, g) for g in (4, 8)] == [7, 4]
    assert [_splits(512, 1024, g) for g in (4, 8)] == [4, 2]
    assert _splits(1, 1, 8) == _splits(10 ** 6, 4096, 1) == 1
