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


@pytest.mark.parametrize("layers", [0, 2])
def test_accept_before_a_row_without_a_slot(ops, engine, layers):
    """A path ends where its sequence has no page: nothing is kept, counted or written from there on."""
    import torch
    c = Accept(27, [5, 9, 2, 0, 130, 3], agree=1.0, shape="chain", history=400)
    none = {1: 0, 2: 0, 4: 77}  # sequence: its first row without a slot
    slots = c.slots.copy()
    for b, j in none.items():
        slots[c.offsets[b] + j:c.offsets[b + 1]] = S.NO_SLOT
    slots[c.offsets[4] + 100:c.offsets[5]] = 7  # behind the first
    rows = {} if layers else dict(layers=0, kv_heads=0, head_dim=0, k=None, v=None, hot_k=None, hot_v=None)
    ops.accept_tree(c.desc(slots=torch.from_numpy(slots).cuda(), **rows))
    assert error_of(engine) == ""
    paths = S.accept_tree(c.parents, c.tokens, c.targets, c.offsets, slots)
    assert [len(p) for p in paths] == [5, 0, 0, 0, 77, 3]
    kept = np.array([len(p) for p in paths])
    assert host(c.got["accepted"]).tolist() == kept.tolist()
    assert host(c.got["seq_hot"]).tolist() == (c.held + kept).tolist()
    assert host(c.got["history_count_out"]).tolist() == (c.count + kept).tolist()
    k, history = c.pool.copy(), c.history.copy()
    for b, p in enumerate(paths):
        first, end = c.offsets[b], c.offsets[b + 1]
        following = c.targets[first + p[-1]] if p else c.tokens[first] if end > first else -1
        assert int(host(c.got["next_token"])[b]) & 0xFFFFFFFF == int(following) & 0xFFFFFFFF
        assert host(c.got["path"])[first:end].tolist() == p + [-1] * (end - first - len(p))
        for j, node in enumerate(p):
            k[:, slots[first + j] // 16, slots[first + j] % 16] = c.k[:, first + node]
            history[b, c.count[b] + j] = c.tokens[first + node]
    assert np.array_equal(host(c.got["history"]).astype(np.int64) & 0xFFFFFFFF, history & 0xFFFFFFFF)
    assert np.array_equal(host(c.hot_k).view(np.int16), (k if layers else c.pool).view(np.int16))


def test_generation_over_a_list_that_ends_and_is_filled_again(ops, engine):
    """While there is no page a sequence keeps nothing and takes its token again; what it keeps is in its pages."""
    import torch
    from test_gpu_step_run import HK, HQ, Run
    run = Run(64)
    whole = run.d_tables.free_count
    run.d_tables.free_count = 3
    held, errors = [], []
    for i in range(14):
        if i == 7:
            run.d_tables.free_count = whole
        run.step(ops)
        errors.append(error_of(engine))
        held.append(run.held.cpu().numpy().copy())
    print(np.array(held), errors, flush=True)
    assert all("free pages" in e for e in errors[4:7]) and not any(errors[7:])
    assert (held[6] == held[5]).any() and (held[13] > held[6]).all()
    pages, refs, history, count = (x.cpu().numpy() for x in (run.pages, run.refs, run.history, run.count))
    assert np.array_equal(count, held[13])
    for b in range(len(count)):
        n = int(count[b])
        assert n <= 16 * pages[b]
        rows = (run.embed[:, torch.from_numpy(history[b, :n]).cuda().long()] * run.turn[:n]).half()
        at = torch.from_numpy(refs[b, np.arange(n) // 16].astype(np.int64)).cuda(), torch.arange(n, device="cuda:0") % 16
        assert torch.equal(run.hot_k[:, at[0], at[1]], rows[:, :, HQ:HQ + HK]) and torch.equal(run.hot_v[:, at[0], at[1]], rows[:, :, HQ + HK:])


def test_logits_report_offsets_wherever_they_descend(ops, engine):
    """Also where no row's search meets them: here rows 2 to 9 of the second of 128 sequences."""
    c = Logits(28, 300, [10], history=9)
    kw = {k: np.repeat(v, 128, axis=0) for k, v in c.kw.items() if k in ("history", "history_count", "prompt_count", "repetition", "frequency", "presence")}
    offsets = np.array([0, 0, 10] + [2] * 126)
    c.kw.update(kw, offsets=offsets)
    c.batch = 128
    ops.adjust_logits(c.desc())
    assert "sequence length" in error_of(engine)
    offsets[3:] = 10  # all of them empty
    ops.adjust_logits(c.desc())
    assert error_of(engine) == ""
    c.check()


@pytest.mark.parametrize("vocab,half", [(257, False), (1025 + 256, False), (4096 + 769, False), (513, True), (2048 + 1537, True), (1, False), (7, True)])
def test_masks_in_place_where_pieces_of_two_waves_overlap(ops, engine, vocab, half):
    """Without counts a value may be made again from the output: masked twice it is what it is masked once."""
    c = Logits(29, vocab, [40], half=half, nodes=False, allowed=0.5, extreme=True)
    d = c.desc(token_offsets=None, batch=0)
    d.out, d.out_stride = d.logits, d.logits_stride
    ops.adjust_logits(d)
    assert error_of(engine) == ""
    c.check(out=c.src)


@pytest.mark.parametrize("tree", ["random", "chain", None])
@pytest.mark.parametrize("what", ["full", "past", "nodes", "many_nodes", "held", "wrap"])
def test_tables_of_a_sequence_past_its_table_leave_the_others(ops, engine, what, tree):
    """What is wrong with one sequence moves no row of another: their offsets, slots, positions and masks are those beside a sequence
    that fits."""
    held, new = [3, 20, 0, 31, 7], [14, 40, 2, 9, 30]
    words = 2
    if what == "nodes":
        words = 1
    elif what == "many_nodes":
        new[1] = 1400
    c = Tables(30, held, new, tree=tree, pad=3, words=words)
    good = c.want(held=np.array(held), words=words)
    if what == "full":
        held[1] = 16 * c.count - 7
    elif what == "past":
        held[1] = 16 * c.count
    elif what == "held":
        held[1] = 16 * c.count + 500
    elif what == "wrap":
        held[1] = 0xFFFFFFFF - 20
    c.held = np.array(held)
    c.pages = None
    ops.page_tables(c.desc())
    want, text = c.want(), error_of(engine)
    fits = tree is None and what in ("nodes", "many_nodes") and new[1] + 20 <= 16 * c.count
    assert want["errors"] == (set() if fits else {"sequence length"})
    assert ("sequence length" in text) == (not fits) and "free pages" not in text
    c.check(want, skip=("seq_hot", "pages_out", "positions") if what == "wrap" else ())
    a, e = good["token_offsets"][1:3]
    for name in ("positions", "tree_mask"):
        if name in c.got:
            got = host(c.got[name]).astype(np.int64) & 0xFFFFFFFF
            assert np.array_equal(got[:a], good[name][:a]) and np.array_equal(got[e:], good[name][e:])
    assert np.array_equal(host(c.got["token_offsets"]), good["token_offsets"])


def test_generation_past_the_end_of_a_table(ops, engine):
    """A sequence whose table is full keeps what fits and then nothing; the others go on as they do beside it."""
    import torch
    from test_gpu_step_run import HK, HQ, PAGES, Run
    run = Run(64)
    run.turn = torch.cat([run.turn, torch.ones((64, 1, 1), device="cuda:0")])  # positions behind the table's end
    run.held[0] = 16 * PAGES - 5  # of pages that hold something: the whole table is its own
    run.pages[0] = PAGES
    run.refs[0] = torch.arange(PAGES, device="cuda:0", dtype=torch.int32) % 3 + run.blocks
    for p in ("hot_k", "hot_v"):
        pool = getattr(run, p)
        setattr(run, p, torch.cat([pool, torch.zeros((2, 3) + tuple(pool.shape[2:]), dtype=pool.dtype, device="cuda:0")], 1).contiguous())
    from aether_nexus_amd import ops as O
    k, v = run.rows[:, :, HQ:HQ + HK], run.rows[:, :, HQ + HK:]
    run.d_tree = [O.make_tree_desc(batch=4, num_tokens=run.rows.shape[1], q_heads=HQ, kv_heads=HK, head_dim=64, q=run.rows[l, :, :HQ], k=k[l], v=v[l],
                                   out=run.out[l], hot_k=run.hot_k[l], hot_v=run.hot_v[l], refs=run.refs, hot_count=PAGES, seq_held=run.held,
                                   token_offsets=run.offsets, tree_mask=run.mask) for l in range(2)]
    run.d_accept = O.make_accept_desc(batch=4, num_tokens=run.rows.shape[1], layers=2, kv_heads=HK, head_dim=64, parents=run.parents,
                                      node_tokens=run.nodes, targets=run.best, token_offsets=run.offsets, seq_held=run.held, slots=run.slots, k=k, v=v,
                                      hot_k=run.hot_k, hot_v=run.hot_v, accepted=run.accepted, next_token=run.following, seq_hot=run.after,
                                      path=run.path, history=run.history, history_count=run.count, history_count_out=run.count)
    before = run.held.cpu().numpy().copy()
    starts = [len(p) for p in run.prompts]
    for i in range(10):
        run.step(ops)
        assert "sequence length" in error_of(engine)
    held = run.held.cpu().numpy()
    assert held[0] <= 16 * PAGES and (held[1:] > before[1:]).all()
    count, history, refs = (x.cpu().numpy() for x in (run.count, run.history, run.refs))
    for b in range(1, 4):
        n = int(count[b])
        assert n == held[b] and n > starts[b]
        rows = (run.embed[:, torch.from_numpy(history[b, :n]).cuda().long()] * run.turn[:n]).half()
        at = torch.from_numpy(refs[b, np.arange(n) // 16].astype(np.int64)).cuda(), torch.arange(n, device="cuda:0") % 16
        assert torch.equal(run.hot_k[:, at[0], at[1]], rows[:, :, HQ:HQ + HK])


def test_accept_into_pools_of_one_buffer(ops, engine):
    """K and V pages of a layer side by side."""
    import torch
    c = Accept(31, [7, 12, 1], layers=3, agree=1.0)
    both = torch.stack([dev(c.pool), dev(-c.pool)], 1).contiguous()
    ops.accept_tree(c.desc(hot_k=both[:, 0], hot_v=both[:, 1]))
    assert error_of(engine) == ""
    c.hot_k, c.hot_v = both[:, 0].contiguous(), both[:, 1].contiguous()
    c.check()


def test_capture_refuses_workspace_growth():
    """A captured call whose scratch does not fit yet is refused before anything is enqueued; after an eager one it is captured."""
    import torch
    from aether_nexus_amd.ops import OpsEngine
    from aether_nexus_amd.types import AW_E_UNSUPPORTED
    from aether_nexus_amd.weaver import WeaverError
    from test_gpu_tree import Case
    logits, tree = Logits(32, 40001, [3, 5], history=50, bias=5, allowed=0.5), Case(33, 8, 2, 64, [5, 80], [3000, 30])  # in several parts
    for call, c, d in (("adjust_logits", logits, logits.desc()), ("tree_attention", tree, tree.desc())):
        fresh = OpsEngine()
        try:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g = torch.cuda.CUDAGraph()
                with pytest.raises(WeaverError) as e:
                    with torch.cuda.graph(g, stream=s):
                        getattr(fresh, call)(d)
                assert e.value.status == AW_E_UNSUPPORTED and "eager" in str(e.value)
                del g
                torch.cuda.synchronize()
                assert bool((c.out == 7.0).all())
                getattr(fresh, call)(d)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    getattr(fresh, call)(d)
                for _ in range(3):
                    c.out.fill_(7.0)
                    g.replay()
                    s.synchronize()
                    c.check(*(["captured"] if call == "tree_attention" else []))
                del g
            torch.cuda.synchronize()
        finally:
            fresh.close()


def test_logits_past_32_bits(ops, engine):
    """Rows whose elements lie past 2^32 of the tensor, in place, with masks by a row of their own and tokens of their sequences."""
    import torch
    from aether_nexus_amd import ops as O
    vocab, rows = 128256, (1 << 32) // 128256 + 40
    x = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda:0")
    c = Logits(33, vocab, [1, 8], half=True, history=40, bias=6, nodes=False)
    c.kw["offsets"] = [0, rows - 8, rows]
    x[-8:] = torch.from_numpy(c.x[-8:]).cuda()
    best = empty(rows)
    names = {"offsets": "token_offsets"}
    d = O.make_logits_desc(num_tokens=rows, vocab_size=vocab, batch=2, logits=x, out=x, best=best,
                           **{names.get(k, k): dev(np.asarray(v)) for k, v in c.kw.items()})
    ops.adjust_logits(d)
    assert error_of(engine) == ""
    second = {k: np.asarray(v)[1:2] for k, v in c.kw.items() if k != "offsets"}
    want, top = S.adjust_logits(c.x[-8:], offsets=[0, 8], **second)
    assert np.array_equal(host(x[-8:]), want.astype(np.float16)) and host(best)[-8:].tolist() == top.tolist()
    assert bool((best[:-8] == best[0]).all()) and bool((x[0] == x[rows - 9]).all())


def test_a_step_of_no_rows(ops, engine):
    """A batch without a new token: what belongs to sequences is written, nothing else is touched."""
    import torch
    from aether_nexus_amd import ops as O
    c = Tables(34, [5, 16], [0, 0], tree="chain")
    ops.page_tables(c.desc())
    assert error_of(engine) == ""
    c.check(c.want())
    f16 = lambda *shape: torch.empty(shape, dtype=torch.float16, device="cuda:0")
    offsets = dev(np.array([0, 0, 0]))
    ops.tree_attention(O.make_tree_desc(batch=2, num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, q=f16(0, 4, 64), k=f16(0, 2, 64), v=f16(0, 2, 64),
                                        out=f16(0, 4, 64), token_offsets=offsets, tree_mask=empty(0, 2)))
    ops.adjust_logits(O.make_logits_desc(num_tokens=0, vocab_size=50, logits=f16(0, 50), out=f16(0, 50), best=empty(0), batch=2, token_offsets=offsets,
                                         node_tokens=empty(0), tree_mask=empty(0, 2)))
    a = Accept(35, [0, 0])
    ops.accept_tree(a.desc())
    assert error_of(engine) == ""
    a.check()


def test_logits_of_an_empty_grammar(ops, engine):
    """A table of no states with an index: none for -1, and a state that is not there allows nothing."""
    import torch
    c = Logits(36, 300, [3, 2], history=9)
    c.kw.update(allowed=np.zeros((0, 10), dtype=np.uint32), allowed_index=np.full(5, -1))
    ops.adjust_logits(c.desc())
    assert error_of(engine) == ""
    c.check()
    c.kw["allowed_index"][2] = 0
    ops.adjust_logits(c.desc())
    assert "token id" in error_of(engine)
    c.check()
