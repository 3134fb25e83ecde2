"""Attention of trees where its descriptor, offsets or plan are at an edge, against the float64 oracle with the tolerance
of test_gpu_tree.py, whose inputs it takes."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import prefix_errors
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


# Offsets as a caller should not give them; the sequences among them that lie within the rows and ascend.
BAD_OFFSETS = [[0, 9, 3], [0, 3, 40], [5, 2, 23], [9, 4, 7, 23], [0, 100, 7, 23], [0, 2, 1 << 31, 2, 23], [3, 3, 23, 0], [0, 0xFFFFFFFF, 0, 23, 22]]


@pytest.mark.parametrize("spare", [0, 9000], ids=["one", "shared"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("offsets", BAD_OFFSETS, ids=lambda o: "-".join(map(str, o)))
def test_sequences_beside_bad_offsets(ops, engine, offsets, hd, spare):
    """Reported; each sequence whose own offsets are good is computed, and nothing is written beside those rows."""
    import torch
    n = len(offsets) - 1
    good = [b for b in range(n) if offsets[b] <= offsets[b + 1] <= 23]
    c = Case(11, 8, 2, hd, [3, 20] + [0] * (n - 2), [48, 17] + [33] * (n - 2), spare=spare)
    around = torch.full((c.rows + 40, 8, hd), 7.0, dtype=torch.float16, device="cuda:0")
    d = c.desc(token_offsets=dev(np.array(offsets)), out=around[20:20 + c.rows])
    assert (plan_of(d) == 0) == (spare == 0)
    ops.tree_attention(d)
    assert "sequence length" in error_of(engine)
    got = host(around).astype(np.float64)
    left = np.ones(len(got), dtype=bool)
    for b in good:
        first, end = offsets[b], offsets[b + 1]
        if first == end:
            continue
        left[20 + first:20 + end] = False
        want, absolute, total = c.want(offsets=[first, end], refs=c.refs[b:b + 1], held=c.held[b:b + 1])
        worst, _ = prefix_errors(got[20 + first:20 + end], want[first:end], absolute[first:end], total[first:end], 48 + 23, 6.0)
        assert worst <= 1.0, (b, worst)
    assert (got[left] == 7.0).all()


def test_steps_just_past_32_bits_by_bad_offsets(ops, engine):
    """Sequences of all rows each, whose steps together are a little more than 2^32: reported, and nothing is computed.  The sum
    has to be exact: in fp32, one after another, the short sequences at its end do not count, and the rest is below 2^32."""
    import torch
    from aether_nexus_amd import ops as O
    n, hd = 1 << 17, 64
    steps = lambda nodes: -(-nodes // 16) * -(-nodes // 64)  # of a sequence without pages in units of 16 rows
    sizes = [n] * 255
    sizes += [max(m for m in range(n) if steps(m) + 255 * steps(n) < 4294950000)] + [320] * 600
    total, fp32 = sum(map(steps, sizes)), np.float32(0)
    for m in sizes:
        fp32 += np.float32(steps(m))
    assert 2 ** 32 < total < 2 ** 32 + 2 ** 16 and fp32 < 4294960000
    offsets = np.zeros(256 * len(sizes) + 1, dtype=np.int64)  # every 256th sequence, which one thread counts, has rows
    offsets[1::256] = sizes
    q = torch.zeros((n, 1, hd), dtype=torch.float16, device="cuda:0")
    out = torch.full_like(q, 7.0)
    d = O.make_tree_desc(batch=len(offsets) - 1, num_tokens=n, q_heads=1, kv_heads=1, head_dim=hd, q=q, k=q, v=q, out=out,
                         token_offsets=dev(offsets))
    assert plan_of(d) == 16
    ops.tree_attention(d)
    assert "sequence length" in error_of(engine)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("way", SPLITS, ids=IDS)
def test_bad_refs_and_unseen_infinities_in_each_split(ops, engine, way):
    """Bad refs hide their pages, whatever lies in the page that is read in their place; NaN and infinities of nodes reach the rows that
    see them alone."""
    hq, hk, hd, nodes, held, spare, tile = way
    c = Case(42, hq, hk, hd, nodes, held, pad=1, spare=spare, qscale=1.0)
    # Page 0, which is read for a bad ref, holds no token and NaN and inf alone.
    free = [p for p in range(c.blocks) if p not in set((c.refs & 0x7FFFFFFF).ravel().tolist())][0]
    moved = (c.refs & 0x7FFFFFFF) == 0
    c.refs[moved] = c.refs[moved] & (1 << 31) | free
    for p in (c.hot_k, c.hot_v):
        p[free] = p[0]
        p[0] = np.inf
        p[0, ::2] = np.nan
    longest = int(np.argmax(held))
    pages = -(-held[longest] // 16)
    c.refs[longest, [0, pages // 2, pages - 1]] = c.blocks, 0x7FFFFFFF, c.blocks + 7
    # A node of the widest tree that only the last row sees, and one that none sees.
    wide = int(np.argmax(nodes))
    first, last = c.offsets[wide], c.offsets[wide + 1] - 1
    c.mask[first:last, 0] &= ~np.uint32(1 << 1)
    c.mask[last, 0] |= 1 << 1
    c.v[first + 1, 0, 5] = np.inf
    d = c.desc()
    assert plan_of(d) == tile
    ops.tree_attention(d)
    assert "hot block ref" in error_of(engine)
    got = host(c.out)[:c.offsets[-1]].astype(np.float64)
    heads = range(hq // hk)
    bad = sorted(map(tuple, np.argwhere(~np.isfinite(got))))
    assert bad == [(last, h, 5) for h in heads] and all(got[i] == np.inf for i in bad)
    c.v[first + 1, 0, 5] = 0.0  # its weight counts in every dim; with 0 in this one the oracle is finite
    want, absolute, total = c.want()
    n = int(c.offsets[-1])
    for i in bad:
        got[i] = want[i]
    worst, _ = prefix_errors(got, want[:n], absolute[:n], total[:n], max(held) + max(nodes), 6.0)
    assert worst <= 1.0
