"""Attention of trees where its descriptor, offsets or plan are at an edge, against the float64 oracle with the tolerance
of test_gpu_tree.py, whose inputs it takes."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import WAYS, Case, dev, error_of, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(engine):
    from aether_nexus_amd.ops import OpsEngine
    return OpsEngine(engine)


def plan_of(d):
    import torch
    from aether_nexus_amd import ops as O
    plan = O.tree_plan(d, torch.cuda.get_device_properties(0).multi_processor_count)
    return plan.row_tile if plan.workspace_bytes else 0


# One launch, then units of 16, 32 and 128 rows, 64 and 128 dims each.
SPLITS = [WAYS[i] for i in (0, 1, 4, 5, 6, 7, 8, 9)]
IDS = [f"{w[2]}-{w[6]}" for w in SPLITS]


@pytest.mark.parametrize("way", SPLITS, ids=IDS)
def test_k_of_a_fused_product_as_values(ops, engine, way):
    """Without v the values are the K rows, wherever those lie: a part of a fused product, further apart than their width."""
    hq, hk, hd, nodes, held, spare, tile = way
    c = Case(41, hq, hk, hd, nodes, held, pad=2, spare=spare, qscale=1.0)
    d = c.desc(v=None, hot_v=None)
    assert d.k_stride == (hq + 2 * hk) * hd and plan_of(d) == tile
    ops.tree_attention(d)
    assert error_of(engine) == ""
    c.check("K rows are the values", v=c.k, hot_v=c.hot_k)
    d.v_stride = 0  # as a C caller leaves it
    c.out.fill_(7.0)
    ops.tree_attention(d)
    c.check("and no stride of v", v=c.k, hot_v=c.hot_k)


def test_many_sequences_that_share_rows_equally(ops, engine):
    """2^18 sequences of one row: each sees itself alone, its values come back as they are."""
    import torch
    from aether_nexus_amd import ops as O
    n, heads, hd = 1 << 18, 8, 64
    q, k, v = torch.randn((n, 3 * heads, hd), dtype=torch.float16, device="cuda:0").split(heads, 1)
    out = torch.full((n, heads, hd), 7.0, dtype=torch.float16, device="cuda:0")
    ops.tree_attention(O.make_tree_desc(batch=n, num_tokens=n, q_heads=heads, kv_heads=heads, head_dim=hd, q=q, k=k, v=v, out=out))
    assert error_of(engine) == ""
    assert torch.equal(out, v)
