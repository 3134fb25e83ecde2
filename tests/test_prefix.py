"""Shared-prefix attention without a GPU: the descriptor's layout, what the host refuses, and how requests are split."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from aether_nexus_amd import _lib
from aether_nexus_amd import ops as O
from aether_nexus_amd.types import (AW_E_ALIGN, AW_E_INVALID_ARG, AW_E_UNSUPPORTED, AW_F_CAUSAL, PrefixDesc,
                                    PrefixPlanInfo)
from aether_nexus_amd.weaver import WeaverError

A = {n: (i + 1) << 36 for i, n in enumerate(("q", "out", "hot_k", "hot_v", "prefix_refs", "refs", "seq_own"))}


def desc(**kw):
    d = PrefixDesc(batch=4, queries=2, q_heads=8, kv_heads=2, head_dim=128, prefix_tokens=100, own_count=3, refs_stride=3,
                   flags=AW_F_CAUSAL, scale=0.1, hot_blocks=50, **A)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def test_struct_sizes_match():
    sizes = (ctypes.c_size_t * 2)()
    _lib.load().aw_abi_prefix_sizes(sizes)
    assert tuple(sizes) == (ctypes.sizeof(PrefixDesc), ctypes.sizeof(PrefixPlanInfo))


@pytest.mark.parametrize("kw", [dict(), dict(hot_v=0), dict(seq_own=0), dict(prefix_tokens=0, prefix_refs=0),
                                dict(own_count=0, refs=0, refs_stride=0), dict(flags=0), dict(head_dim=64), dict(queries=500),
                                dict(prefix_tokens=0, own_count=0, hot_k=0, hot_v=0, hot_blocks=0), dict(q_heads=2 * 70),
                                dict(prefix_tokens=1 << 26, own_count=1 << 18, refs_stride=1 << 18), dict(hot_blocks=1 << 31),
                                dict(out=A["q"]), dict(scale=2e38)])
def test_accepted_requests_are_covered_by_their_parts(kw):
    d = desc(**kw)
    for cus in (0, 1, 64, 304):
        p = O.prefix_plan(d, cus)
        assert p.prefix_splits + p.own_splits <= 64
        if p.prefix_splits + p.own_splits == 0:  # in one part, without a workspace
            assert d.prefix_tokens + 16 * d.own_count <= 512 and p.workspace_bytes == 0
            continue
        for tokens, parts, span in ((d.prefix_tokens, p.prefix_splits, p.prefix_tokens_per_split),
                                    (16 * d.own_count, p.own_splits, p.own_tokens_per_split)):
            assert (parts == 0) == (tokens == 0) and parts * span >= tokens and span % 32 == 0
            assert parts == 0 or (parts - 1) * span < tokens  # no empty part
        # bytes of the parts' maxima, sums and rows
        floats = d.kv_heads * (p.prefix_splits + p.own_splits) * d.batch * d.queries * (d.q_heads // d.kv_heads)
        assert floats * (d.head_dim + 2) * 4 <= p.workspace_bytes + 1024


@pytest.mark.parametrize("batch,queries,own_count", [
    (64, 512, 160), (1, 4096, 512), (16, 2048, 2048), (8, 2048, 256), (32, 2048, 512), (1, 8192, 2048), (64, 1, 2048),
    (256, 1, 2048), (1, 64, 2048), (4, 16, 1 << 18), (1, 1 << 20, 1 << 10)])
@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64)], ids=str)
def test_workspace_of_many_queries_and_wide_tables(batch, queries, own_count, heads):
    """Parts are for filling the GPU: their sums stay within 128 MiB (and two numbers a row: 1 / 32 of 64 dims), or,
    where the queries are many, one part of the prefix and one of the own tokens, 4 bytes for each 2 of q."""
    hq, hk, hd = heads
    for prefix in (0, 2048, 32768):
        for cus in (256, 304):
            d = desc(batch=batch, queries=queries, q_heads=hq, kv_heads=hk, head_dim=hd, prefix_tokens=prefix,
                     own_count=own_count, refs_stride=own_count, q=1 << 50, out=2 << 50)
            p = O.prefix_plan(d, cus)
            q_bytes = 2 * batch * queries * hq * hd
            assert p.workspace_bytes <= max(133 << 20, 4.2 * q_bytes)
            if 4 * q_bytes > 128 << 20:
                assert p.own_splits == 1 and p.prefix_splits == (prefix > 0)


@pytest.mark.parametrize("batch,own_count,splits", [(64, 17, 1), (64, 256, 8), (64, 1024, 32), (96, 94, 3)])
def test_parts_of_few_queries(batch, own_count, splits):
    """A step of few queries is cut as its own tokens ask for: at most 512 a part."""
    d = desc(batch=batch, queries=1, q_heads=32, kv_heads=8, prefix_tokens=8192, own_count=own_count, refs_stride=own_count)
    assert O.prefix_plan(d, 256).own_splits == splits


@pytest.mark.parametrize("kw", [dict(batch=0), dict(queries=0), dict(kv_heads=0), dict(q_heads=7), dict(q_heads=0), dict(flags=2),
                                dict(flags=AW_F_CAUSAL | 8), dict(scale=math.inf), dict(scale=math.nan), dict(refs_stride=2),
                                dict(q=0), dict(out=0), dict(prefix_refs=0), dict(refs=0), dict(hot_k=0), dict(hot_blocks=0),
                                dict(hot_blocks=(1 << 31) + 1), dict(scale=3e38), dict(out=A["q"] + 16), dict(q=A["out"] + 16)])
def test_invalid(kw):
    with pytest.raises(WeaverError) as e:
        O.prefix_plan(desc(**kw))
    assert e.value.status == AW_E_INVALID_ARG and "shared_prefix_attention" in str(e.value)


@pytest.mark.parametrize("pool", ["hot_k", "hot_v"])
def test_out_over_a_pool(pool):
    """Rows written into pages that other work-groups still read."""
    size = 50 * 16 * 2 * 128 * 2
    for at in (0, 16, size - 8, -16, 8 - 4 * 2 * 8 * 128 * 2):
        with pytest.raises(WeaverError) as e:
            O.prefix_plan(desc(out=A[pool] + at))
        assert e.value.status == AW_E_INVALID_ARG and "pool" in str(e.value)
    for at in (size, -4 * 2 * 8 * 128 * 2):  # right behind it, right before it
        O.prefix_plan(desc(out=A[pool] + at))
    O.prefix_plan(desc(out=A["hot_k"], prefix_tokens=0, own_count=0))  # no token: the pool is not read


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(head_dim=256), dict(prefix_tokens=(1 << 26) + 1),
                                dict(own_count=(1 << 18) + 1, refs_stride=1 << 19), dict(kv_heads=1024, q_heads=1024),
                                dict(batch=1 << 20, queries=1 << 10), dict(batch=1 << 26, queries=1 << 26),
                                dict(batch=1 << 23, queries=1)])
def test_unsupported(kw):
    with pytest.raises(WeaverError) as e:
        O.prefix_plan(desc(**kw))
    assert e.value.status == AW_E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(q=A["q"] + 8), dict(hot_k=A["hot_k"] + 2), dict(hot_v=A["hot_v"] + 8), dict(out=A["out"] + 4)])
def test_misaligned(kw):
    with pytest.raises(WeaverError) as e:
        O.prefix_plan(desc(**kw))
    assert e.value.status == AW_E_ALIGN


def test_null_descriptor():
    assert _lib.load().aw_shared_prefix_plan(None, 0, None, None, 0) == AW_E_INVALID_ARG


def test_descriptors_take_gpu_tensors_only():
    q = torch.zeros(4, 2, 8, 128, dtype=torch.float16)
    with pytest.raises(WeaverError) as e:
        O.make_prefix_desc(batch=4, queries=2, q_heads=8, kv_heads=2, head_dim=128, prefix_tokens=0, q=q, out=q, hot_k=A["hot_k"],
                           hot_blocks=1)
    assert "GPU" in str(e.value)
    with pytest.raises(WeaverError) as e:  # a raw pool's pages are not known
        O.make_prefix_desc(batch=4, queries=2, q_heads=8, kv_heads=2, head_dim=128, prefix_tokens=0, q=A["q"], out=A["out"],
                           hot_k=A["hot_k"])
    assert "hot_blocks" in str(e.value)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(queries=-1), dict(prefix_tokens=-1), dict(own_count=1 << 32), dict(hot_blocks=-1)])
def test_numbers_that_do_not_fit_are_refused(kw):
    base = dict(batch=1, queries=1, q_heads=8, kv_heads=2, head_dim=128, prefix_tokens=16, q=A["q"], out=A["out"],
                hot_k=A["hot_k"], hot_blocks=4, prefix_refs=A["hot_v"])
    with pytest.raises(WeaverError) as e:
        O.make_prefix_desc(**{**base, **kw})
    assert e.value.status == AW_E_INVALID_ARG and "within" in str(e.value)
