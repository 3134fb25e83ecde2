"""Page tables, adjusted logits and accepted trees where tensors, lists or tables are at an edge, against oracle/step_oracle.py as
test_gpu_step.py compares them, whose inputs it takes."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import step_oracle as S
from test_gpu_step import Accept, Logits, Tables, dev, empty, error_of, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(engine):
    from aether_nexus_amd.ops import OpsEngine
    return OpsEngine(engine)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_logits_of_a_padded_vocabulary(ops, engine, half):
    """Contiguous rows longer than the vocabulary, of logits, outputs and grammar words: what lies past it stays."""
    import torch
    c = Logits(21, 9001, [3, 0, 5], half=half, history=50, bias=5, allowed=0.5, pad=2)
    d = c.desc()
    rows, vocab = c.x.shape
    src = torch.full((rows, 9216), 3.0, dtype=c.src.dtype, device="cuda:0")
    src[:, :vocab] = c.src
    out = torch.full_like(src, 7.0)
    words = torch.full((c.kw["allowed"].shape[0], 288), -1, dtype=torch.int32, device="cuda:0")
    words[:, :c.kw["allowed"].shape[1]] = dev(c.kw["allowed"])
    ops.adjust_logits(c.desc(logits=src, out=out, allowed=words))
    assert error_of(engine) == ""
    c.out = out[:, :vocab]
    c.check()
    assert (host(out)[:, vocab:] == 7.0).all()
    c.best.fill_(-77)
    d = c.desc(logits=src, out=src, allowed=words)
    ops.adjust_logits(d)
    c.check(out=src[:, :vocab])
    assert (host(src)[:, vocab:] == 3.0).all() and np.array_equal(host(src)[8:, :vocab], c.x[8:])


def test_accept_rows_of_a_larger_buffer(ops, engine):
    """K and V rows of a step in buffers of more tokens: each layer's own, not those behind the first one's."""
    import torch
    c = Accept(22, [7, 12, 1], layers=3, agree=1.0)
    k, v = (torch.full((3, c.rows + 13, 2, 64), float("nan"), dtype=torch.float16, device="cuda:0") for _ in range(2))
    k[:, :c.rows], v[:, :c.rows] = dev(c.k), dev(c.v)
    ops.accept_tree(c.desc(k=k, v=v))
    assert error_of(engine) == ""
    c.check()


def test_accept_into_pools_of_more_layers_and_blocks(ops, engine):
    """The first layers and blocks of a larger pool: the rest stays."""
    import torch
    c = Accept(23, [7, 12, 1], layers=2, agree=1.0)
    pools = [torch.full((4, c.blocks + 3, 16, 2, 64), 5.0, dtype=torch.float16, device="cuda:0") for _ in range(2)]
    for p, x in zip(pools, (c.pool, -c.pool)):
        p[:2, :c.blocks] = dev(x)
    ops.accept_tree(c.desc(hot_k=pools[0], hot_v=pools[1], hot_blocks=c.blocks))
    assert error_of(engine) == ""
    c.hot_k, c.hot_v = (p[:2, :c.blocks].contiguous() for p in pools)
    c.check()
    for p in pools:
        assert (host(p)[2:] == 5.0).all() and (host(p)[:, c.blocks:] == 5.0).all()
    for p, x in zip(pools, (c.pool, -c.pool)):
        p[:2, :c.blocks] = dev(x)
    ops.accept_tree(c.desc(hot_k=pools[0], hot_v=pools[1]))
    c.hot_k, c.hot_v = (p[:2, :c.blocks].contiguous() for p in pools)
    c.check()


# ---------------------------------------------------------------- a list of free pages that ends

@pytest.mark.parametrize("tree", [None, "random"], ids=["plain", "tree"])
@pytest.mark.parametrize("short", [1, 3, 5])
def test_tables_after_a_list_that_ended(ops, engine, tree, short):
    """Only pages that a step took are counted: when the list is full again, the next step of the same lengths takes the rest."""
    c = Tables(24, [3, 16, 0, 31, 48, 10], [14, 40, 2, 9, 33, 5], extra=[0, 0, 1, 0, 0, 0], tree=tree, free_short=short)
    full = Tables(24, c.held, c.new, extra=[0, 0, 1, 0, 0, 0], tree=tree)
    d = c.desc()
    ops.page_tables(d)
    want = c.want()
    assert want["errors"] == {"free pages"} and "free pages" in error_of(engine)
    c.check(want)
    assert int((want["pages_out"] - c.pages).sum()) == len(c.free) - c.first
    # The same lengths again, the pages that were taken, the rest of the list.
    c.refs, c.pages, c.first = want["refs"], want["pages_out"], int(want["free_next"])
    c.free = full.free
    ops.page_tables(c.desc())
    assert error_of(engine) == ""
    want = c.want()
    assert not want["errors"] and (want["slots"] >= 0).all()
    c.check(want)


def test_tables_of_held_tokens_without_pages(ops, engine):
    """A sequence that holds more than its pages takes none: its new tokens have no slot, and their entries name no page."""
    c = Tables(25, [20, 33, 16, 40], [14, 1, 0, 30], first=0)
    c.pages = np.array([1, 3, 0, 2])
    ops.page_tables(c.desc())
    want = c.want()
    assert want["errors"] == {"sequence length"} and "sequence length" in error_of(engine)
    assert want["pages_out"].tolist() == [1, 3, 0, 2] and (want["slots"][:14] < 0).all() and (want["slots"][15:] < 0).all() and want["slots"][14] >= 0
    c.check(want)
    # An entry that is counted but names no page is reported whenever a new token falls into it.
    c = Tables(26, [20, 33], [14, 1], first=0)
    c.refs[0, 1] = 0xFFFFFFFF  # bit 31 masked: 0x7FFFFFFF
    ops.page_tables(c.desc())
    want = c.want()
    assert want["errors"] == {"free pages"} and "free pages" in error_of(engine) and (want["slots"][:12] < 0).all()
    c.check(want)
