"""A step over trees of drafted tokens without a GPU: descriptors at an edge of what their description allows."""
from __future__ import annotations

import pytest

from aether_nexus_amd import ops as O
from test_step import A, tree


@pytest.mark.parametrize("kw", [dict(v_stride=257), dict(v_stride=8), dict(v_stride=1 << 40), dict(k_stride=1536, k=A["q"] + 2 * 1024, q_stride=1536)])
def test_v_stride_is_not_read_without_v(kw):
    assert O.tree_plan(tree(v=0, hot_v=0, **kw)).work_groups
