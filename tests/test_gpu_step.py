"""Page tables, adjusted logits and accepted trees on cuda:0 through the C ABI against
oracle/step_oracle.py: whole numbers equal; logits bit for bit, each step of their description one fp32
rounding (and one to f16 at the store)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import step_oracle as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(engine):
    from aether_nexus_amd.ops import OpsEngine
    return OpsEngine(engine)


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype in (np.float16, np.float32):
        return torch.from_numpy(a.copy()).cuda()
    return torch.from_numpy(a.astype(np.int64) & 0xFFFFFFFF).to(torch.int32).cuda()  # 32-bit words


def host(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


def empty(*shape, dtype="int32", value=-77):
    import torch
    return torch.full(shape, value, dtype=getattr(torch, dtype), device="cuda:0")


def trees(rng, counts, depth=None):
    """Parents of each tree; depth 1: stars, None: random."""
    out = []
    for n in counts:
        out.append([-1 if i == 0 else (0 if depth == 1 else i - 1 if depth == "chain" else int(rng.integers(0, i))) for i in range(n)])
    return out


def error_of(engine):
    from aether_nexus_amd.weaver import WeaverError
    try:
        engine.check_device_errors()
    except WeaverError as e:
        return str(e)
    return ""


# ---------------------------------------------------------------- page tables

class Tables:
    def __init__(self, seed, held, new, *, extra=None, first=3, pad=0, tree=None, spare=1, free_short=0, words=None):
        rng = np.random.default_rng(seed)
        self.held, self.new = np.asarray(held), np.asarray(new)
        extra = np.zeros(len(held), dtype=int) if extra is None else np.asarray(extra)
        self.pages = -(-self.held // 16) + extra
        last = np.maximum(self.pages, -(-(self.held + self.new) // 16))
        self.count = int(max(last.max(initial=0), 1)) + spare
        order = rng.permutation(int(last.sum()) + first + 4)
        self.refs = rng.integers(0, 1 << 31, (len(held), self.count))
        at = 0
        for b, p in enumerate(self.pages):
            self.refs[b, :p] = order[at:at + p]
            at += int(p)
        need = int((last - self.pages).sum())
        self.free = order[at:][:first + need - free_short] if free_short else order[at:]
        self.first, self.rows = first, int(self.new.sum()) + pad
        self.parents = None
        self.words = 0
        if tree is not None:
            self.parents = np.array([p for t in trees(rng, self.new, tree if tree != "random" else None) for p in t] + [5] * pad, dtype=np.int64)
            self.words = -(-int(max(self.new.max(initial=0), 1)) // 32) if words is None else words
        self.got = dict(seq_hot=empty(len(held)), pages_out=empty(len(held)), token_offsets=empty(len(held) + 1), free_next=empty(1),
                        slots=empty(self.rows, dtype="int64"), positions=empty(self.rows))
        if tree is not None:
            self.got["tree_mask"] = empty(self.rows, self.words)

    def desc(self, **kw):
        from aether_nexus_amd import ops as O
        self.got["refs"] = dev(self.refs)
        base = dict(batch=len(self.held), num_tokens=self.rows, seq_held=dev(self.held), seq_new=dev(self.new), seq_pages=None if self.pages is None else dev(self.pages),
                    free_pages=dev(self.free), free_first=dev(np.array([self.first])), parents=None if self.parents is None else dev(self.parents),
                    **self.got)
        return O.make_tables_desc(**{**base, **kw})

    def want(self, **kw):
        base = dict(held=self.held, new=self.new, pages=self.pages, free=self.free, first=self.first, rows=self.rows, hot_count=self.count,
                    parents=self.parents, words=self.words)
        return S.page_tables(self.refs, **{**base, **kw})

    def check(self, want, skip=()):
        for name, t in self.got.items():
            if name not in skip:
                w = np.asarray(want[name])
                g = host(t).astype(np.int64).reshape(w.shape)
                if name != "slots":
                    g &= 0xFFFFFFFF
                assert np.array_equal(g, w), (name, np.argwhere(g != w)[:3])


TABLES = {
    "one": dict(held=[0], new=[1]), "decode": dict(held=list(range(64)), new=[1] * 64), "none_new": dict(held=[5, 16], new=[0, 0], pad=3),
    "ragged": dict(held=[0, 1, 15, 16, 17, 100, 0, 33], new=[3, 15, 1, 1, 0, 30, 0, 47], extra=[0, 1, 0, 0, 0, 2, 3, 0], pad=5),
    "prompts": dict(held=[0, 7, 300], new=[3001, 16, 777]), "many": dict(held=[i % 37 for i in range(3000)], new=[i % 5 for i in range(3000)], pad=9),
    "edge": dict(held=[16] * 1024, new=[1] * 1024), "edge+1": dict(held=[15] * 1025, new=[1] * 1025, spare=0),
    "one_long": dict(held=[0] * 2047 + [12345], new=[0] * 2047 + [1000]), "empty": dict(held=[], new=[], pad=4),
}


@pytest.mark.parametrize("name", sorted(TABLES))
@pytest.mark.parametrize("tree", [None, "random", 1, "chain"], ids=["plain", "random", "star", "chain"])
def test_tables(ops, engine, name, tree):
    if tree is not None and max(TABLES[name]["new"] + [0]) > 1024:
        pytest.skip("a tree has at most 1024 nodes")
    c = Tables(1, tree=tree, **TABLES[name])
    ops.page_tables(c.desc())
    assert error_of(engine) == ""
    want = c.want()
    assert not want["errors"]
    c.check(want)


def test_tables_of_wide_trees(ops, engine):
    for tree in ("random", "chain", 1):
        c = Tables(2, [30, 0, 5], [1024, 1, 300], tree=tree, pad=2)
        ops.page_tables(c.desc())
        assert error_of(engine) == ""
        c.check(c.want())
    c = Tables(3, [30, 0], [7, 33], tree="random", words=32)  # more words than nodes
    ops.page_tables(c.desc())
    c.check(c.want())


def test_tables_without_the_optional_parts(ops, engine):
    c = Tables(4, [3, 20, 0], [14, 1, 2])
    ops.page_tables(c.desc(seq_pages=None, free_first=None, pages_out=None, free_next=None, slots=None, positions=None))
    assert error_of(engine) == ""
    c.check(c.want(pages=None, first=0), skip=("pages_out", "free_next", "slots", "positions"))
    for name in ("pages_out", "free_next", "slots", "positions"):
        assert (host(c.got[name]) == -77).all()


def test_tables_refs_of_a_wider_table(ops):
    import torch
    c = Tables(5, [3, 20, 0], [14, 40, 2])
    wide = torch.full((3, c.count + 5), -9, dtype=torch.int32, device="cuda:0")
    wide[:, :c.count] = dev(c.refs)
    ops.page_tables(c.desc(refs=wide, hot_count=c.count))
    assert (host(wide)[:, c.count:] == -9).all()
    assert np.array_equal(host(wide)[:, :c.count].astype(np.int64) & 0xFFFFFFFF, c.want()["refs"])


@pytest.mark.parametrize("what", ["free", "rows", "capacity", "pages", "nodes", "held", "parents", "huge"])
def test_tables_report(ops, engine, what):
    errors = {"sequence length"}
    c = Tables(6, [3, 20, 0, 31], [14, 40, 2, 9], tree="random" if what in ("nodes", "parents") else None, free_short=2 if what == "free" else 0,
               words=1 if what == "nodes" else None)
    if what == "free":
        errors = {"free pages"}
    elif what == "rows":
        c.rows -= 11
        c.got.update(slots=empty(c.rows, dtype="int64"), positions=empty(c.rows))
    elif what == "capacity":
        c.count = 3
        c.refs = c.refs[:, :3]
    elif what == "pages":
        c.pages = c.pages - np.array([0, 1, 0, 0])
    elif what == "held":
        c.held = c.held.copy()
        c.held[1] = 3000
    elif what == "parents":
        c.parents[14 + 5], c.parents[14 + 9] = 5, 1000
    elif what == "huge":
        c.new = np.array([14, 0xFFFFFFFF, 0xFFFFFFF0, 9])
        c.held = np.array([3, 20, 0xFFFFFFFF, 31])
        c.pages = None
    ops.page_tables(c.desc())
    want = c.want()
    assert want["errors"] == errors
    text = error_of(engine)
    assert all(e in text for e in errors) and ("free pages" in text) == ("free pages" in errors)
    if what == "huge":  # lengths past the table are as they are; their place in 32 bits is not defined
        c.check(want, skip=("seq_hot", "pages_out"))
    else:
        c.check(want)
    assert error_of(engine) == ""


# ---------------------------------------------------------------- logits

class Logits:
    def __init__(self, seed, vocab, counts, *, half=False, history=0, bias=0, allowed=0.0, nodes=True, index=True, pad=0, odd=0, extreme=False):
        rng = self.rng = np.random.default_rng(seed)
        b, rows = len(counts), int(sum(counts)) + pad
        x = rng.standard_normal((rows, vocab)) * 3
        self.x = x.astype(np.float16 if half else np.float32)
        if extreme:
            bad = np.array([np.nan, np.inf, -np.inf, np.finfo(self.x.dtype).min, np.finfo(self.x.dtype).max, 0.0, -0.0], dtype=self.x.dtype)
            at = rng.random((rows, vocab)) < 0.3
            self.x[at] = bad[rng.integers(0, len(bad), int(at.sum()))]
        self.offsets = S.offsets_of(counts)
        self.kw = dict(offsets=self.offsets)
        if history:
            self.kw.update(history=rng.integers(0, max(2, vocab // 3), (b, history)), history_count=rng.integers(0, history + 1, b),
                           prompt_count=rng.integers(0, history + 1, b))
            self.kw["history_count"][0] = history
        if nodes:
            words = -(-max(max(counts), 1) // 32)
            self.kw.update(node_tokens=rng.integers(0, max(2, vocab // 5), rows), mask=S.mask_of(trees(rng, counts), rows, words))
        if history or nodes:
            self.kw.update(repetition=(1 + rng.random(b)).astype(np.float32), frequency=rng.random(b).astype(np.float32),
                           presence=rng.random(b).astype(np.float32))
        if bias:
            self.kw.update(bias_ids=rng.integers(0, vocab, (b, bias)), bias_values=rng.standard_normal((b, bias)).astype(np.float32),
                           bias_count=rng.integers(0, bias + 1, b))
            self.kw["bias_count"][-1] = bias
            self.kw["bias_ids"][:, bias // 2:] = self.kw["bias_ids"][:, :bias - bias // 2]  # ids twice
        if allowed:
            n = max(2, rows // 2) if index else rows
            bits = rng.random((n, -(-vocab // 32) * 32)) < allowed
            self.kw["allowed"] = np.packbits(bits, axis=1, bitorder="little").view("<u4")
            if index:
                self.kw["allowed_index"] = rng.integers(-1, n, rows)
        self.batch, self.odd = b, odd

    def desc(self, **kw):
        import torch
        from aether_nexus_amd import ops as O
        rows, vocab = self.x.shape
        stride = vocab + self.odd
        src = torch.zeros(rows * stride + 1, dtype=torch.float16 if self.x.dtype == np.float16 else torch.float32, device="cuda:0")
        src = src[1:].view(rows, stride)[:, :vocab] if self.odd else src[:rows * stride].view(rows, stride)
        src.copy_(dev(self.x))
        self.src, self.out, self.best = src, torch.full((rows, stride), 7.0, dtype=src.dtype, device="cuda:0")[:, :vocab], empty(rows)
        names = {"offsets": "token_offsets", "mask": "tree_mask"}
        base = dict(num_tokens=rows, vocab_size=vocab, batch=self.batch, logits=src, out=self.out, best=self.best,
                    **{names.get(k, k): dev(np.asarray(v)) for k, v in self.kw.items()})
        if not self.x.size:
            base["logits"] = base["out"] = None
        return O.make_logits_desc(**{**base, **kw})

    def check(self, out=None, best=True, **kw):
        x, top = S.adjust_logits(self.x, **{**self.kw, **kw})
        rows = int(self.offsets[-1])
        with np.errstate(over="ignore"):
            want = x.astype(self.x.dtype)
        got = host(self.out if out is None else out)
        same = (got[:rows] == want[:rows]) | (np.isnan(got[:rows]) & np.isnan(want[:rows]))
        assert same.all(), (np.argwhere(~same)[:4], got[:rows][~same][:4], want[:rows][~same][:4])
        if out is None:
            assert (got[rows:] == 7.0).all()  # behind the last sequence: as they were
        if best:
            assert host(self.best)[:rows].tolist() == top[:rows].tolist() and (host(self.best)[rows:] == -77).all()


LOGITS = {
    "one": (40, [1], dict(history=3)), "tiny": (1, [1, 2], dict(history=2, bias=1, allowed=0.5)), "step": (151936, [1], dict(history=700, bias=9)),
    "batch": (49155, [1] * 9, dict(history=200, bias=40, allowed=0.01)), "tree": (4099, [17, 1, 0, 33, 2], dict(history=64, allowed=0.9, pad=3)),
    "wide_tree": (1000, [300, 70], dict(history=10)), "nodes_alone": (2049, [5, 9], {}), "bias_alone": (8193, [1, 1, 1], dict(nodes=False, bias=1023)),
    "history_alone": (4096, [2, 1], dict(nodes=False, history=5000)), "masks_alone": (100003, [3, 0, 4], dict(nodes=False, allowed=0.001, index=False, pad=2)),
    "nothing": (8192, [2, 3], dict(nodes=False)), "all_masked": (333, [4, 4], dict(allowed=1e-9)), "many": (515, [i % 4 for i in range(150)], dict(history=7)),
    "extreme": (777, [6, 7], dict(history=500, bias=30, allowed=0.7, extreme=True)), "extreme_alone": (9001, [3], dict(nodes=False, extreme=True)),
}


@pytest.mark.parametrize("odd", [0, 3], ids=["rows", "odd"])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("name", sorted(LOGITS))
def test_logits(ops, engine, name, half, odd):
    vocab, counts, kw = LOGITS[name]
    c = Logits(len(name), vocab, counts, half=half, odd=odd, **kw)
    ops.adjust_logits(c.desc())
    assert error_of(engine) == ""
    c.check()


def test_logits_in_place_and_each_output_alone(ops, engine):
    c = Logits(1, 9001, [3, 5], history=50, bias=5, allowed=0.5)
    ops.adjust_logits(c.desc(out=None))
    assert host(c.best).tolist() == S.adjust_logits(c.x, **c.kw)[1].tolist()
    d = c.desc(best=None)
    ops.adjust_logits(d)
    c.check(best=False)
    assert (host(c.best) == -77).all()
    d = c.desc()
    d.out, d.out_stride = d.logits, d.logits_stride
    ops.adjust_logits(d)
    c.check(out=c.src)


# Rows of which a work-group takes 2, 4 or 16 of a sequence, or of two; a last slice of one token and of a piece less one.
GROUPS = {"2": (40001, [7] * 60 + [0, 1, 90], False), "2_f16": (20481, [7] * 60 + [0, 1, 400], True), "4": (4099, [1] * 900 + [64] * 40, False),
          "16": (1031, [33] * 990 + [1, 0, 2], False), "16_f16": (4101, [40] * 450 + [300, 2], True)}


@pytest.mark.parametrize("name", sorted(GROUPS))
def test_logits_of_many_rows(ops, engine, name):
    vocab, counts, half = GROUPS[name]
    c = Logits(11, vocab, counts, half=half, history=70, bias=9, allowed=0.8, pad=3)
    d = c.desc()
    ops.adjust_logits(d)
    c.check()
    d.out, d.out_stride = d.logits, d.logits_stride  # in place
    c.best.fill_(-77)
    ops.adjust_logits(d)
    rows = int(c.offsets[-1])
    assert np.array_equal(host(c.src)[:rows], host(c.out)[:rows]) and np.array_equal(host(c.src)[rows:], c.x[rows:])
    assert error_of(engine) == ""


def test_logits_penalties_left_out(ops):
    for name in ("repetition", "frequency", "presence", "prompt_count", "bias_count"):
        c = Logits(2, 2000, [3, 2], history=90, bias=12)
        ops.adjust_logits(c.desc(**{name: None}))
        c.check(**{name: None})


def test_logits_rows_that_share_equally(ops):
    c = Logits(3, 700, [3, 3, 3], history=30)
    ops.adjust_logits(c.desc(token_offsets=None))
    c.check()


def test_logits_ties_and_zeros(ops):
    """The lowest of equal tokens, -0 equal to 0, over slices and lanes."""
    c = Logits(4, 70000, [1] * 6, nodes=False)
    c.x[:] = -1.0
    c.x[0, [69999, 40000, 123]] = 2.0
    c.x[1, [5, 6]] = -0.0, 0.0
    c.x[2, [60001, 9000]] = 0.0, -0.0
    c.x[3] = -np.inf
    c.x[4] = np.nan
    c.x[4, 65000] = -5.0
    c.x[5, 17] = np.inf
    ops.adjust_logits(c.desc())
    c.check()
    assert host(c.best).tolist() == [123, 5, 9000, -1, 65000, 17]


def test_logits_tokens_past_the_vocabulary_are_passed_over(ops, engine):
    c = Logits(5, 300, [2, 2], history=40, bias=8)
    c.kw["history"][:, ::3] = 300
    c.kw["history"][:, 1::5] = 0xFFFFFFFF
    c.kw["bias_ids"][:, ::2] = 1 << 20
    c.kw["node_tokens"][1] = 299 + (1 << 24)
    ops.adjust_logits(c.desc())
    assert error_of(engine) == ""
    c.check()


def test_logits_report(ops, engine):
    c = Logits(6, 300, [2, 2], history=40, bias=8, allowed=0.5)
    c.kw["history_count"][:] = 41, 40
    ops.adjust_logits(c.desc())
    assert "sequence length" in error_of(engine)
    c.check()
    c.kw["history_count"][:] = 40
    c.kw["bias_count"][:] = 9, 8
    ops.adjust_logits(c.desc())
    assert "sequence length" in error_of(engine)
    c.check()
    c.kw["bias_count"][:] = 8
    c.kw["allowed_index"][2] = c.kw["allowed"].shape[0]
    ops.adjust_logits(c.desc())
    assert "token id" in error_of(engine)
    c.check()
    d = c.desc(token_offsets=dev(np.array([0, 3, 2])))  # offsets that descend end in an error, no rows of others
    ops.adjust_logits(d)
    assert "sequence length" in error_of(engine)


# ---------------------------------------------------------------- accepted trees

class Accept:
    def __init__(self, seed, counts, *, layers=2, hk=2, hd=64, pad=0, agree=0.8, history=40, shape=None):
        rng = np.random.default_rng(seed)
        self.layers, self.hk, self.hd = layers, hk, hd
        grown = trees(rng, counts, shape)
        self.offsets = S.offsets_of(counts)
        rows = self.rows = int(sum(counts)) + pad
        self.parents = np.array([p for t in grown for p in t] + [3] * pad, dtype=np.int64)
        self.tokens = rng.integers(0, 1 << 32, rows)
        self.targets = rng.integers(0, 1 << 32, rows)
        for b, t in enumerate(grown):
            first = self.offsets[b]
            for i in range(len(t)):
                children = [j for j, p in enumerate(t) if p == i]
                if children and rng.random() < agree:
                    self.targets[first + i] = self.tokens[first + int(rng.choice(children))]
                    if rng.random() < 0.3:  # two children with the same token: the lower is kept
                        self.tokens[first + int(rng.choice(children))] = self.targets[first + i]
        self.held = rng.integers(0, 100, len(counts))
        self.blocks = rows // 16 + 3
        self.slots = rng.permutation(self.blocks * 16)[:rows].astype(np.int64)
        self.k, self.v = (rng.standard_normal((layers, rows, hk, hd)).astype(np.float16) for _ in range(2))
        self.pool = rng.standard_normal((layers, self.blocks, 16, hk, hd)).astype(np.float16)
        self.history = rng.integers(0, 1000, (len(counts), max(history, 1)))
        self.count = rng.integers(0, max(history // 2, 1), len(counts))

    def desc(self, **kw):
        import torch
        from aether_nexus_amd import ops as O
        n = len(self.held)
        self.got = dict(accepted=empty(n), next_token=empty(n), seq_hot=empty(n), path=empty(self.rows), history=dev(self.history),
                        history_count_out=empty(n))
        self.hot_k, self.hot_v = dev(self.pool), dev(-self.pool)
        base = dict(batch=n, num_tokens=self.rows, layers=self.layers, kv_heads=self.hk, head_dim=self.hd, parents=dev(self.parents),
                    node_tokens=dev(self.tokens), targets=dev(self.targets), token_offsets=dev(np.array(self.offsets)), seq_held=dev(self.held),
                    k=dev(self.k), v=dev(self.v), hot_k=self.hot_k, hot_v=self.hot_v, slots=torch.from_numpy(self.slots).cuda(),
                    history_count=dev(self.count), **self.got)
        return O.make_accept_desc(**{**base, **kw})

    def check(self, pools=True, skip=(), slots=None):
        paths = S.accept_tree(self.parents, self.tokens, self.targets, self.offsets)
        slots = self.slots if slots is None else slots
        n = len(self.held)
        path, k, v, history = np.full(self.rows, -77, dtype=np.int64), self.pool.copy(), (-self.pool).copy(), self.history.copy()
        following = np.full(n, -1, dtype=np.int64)
        for b, p in enumerate(paths):
            first = self.offsets[b]
            path[first:self.offsets[b + 1]] = -1
            path[first:first + len(p)] = p
            if p:
                following[b] = self.targets[first + p[-1]]
            for j, node in enumerate(p):
                history[b, self.count[b] + j] = self.tokens[first + node]
                s = slots[first + j]
                if 0 <= s < self.blocks * 16:
                    k[:, s // 16, s % 16], v[:, s // 16, s % 16] = self.k[:, first + node], self.v[:, first + node]
        kept = np.array([len(p) for p in paths], dtype=np.int64)
        want = dict(accepted=kept, next_token=following, seq_hot=self.held + kept, path=path, history=history, history_count_out=self.count + kept)
        for name, t in self.got.items():
            if name not in skip:
                w = np.asarray(want[name], dtype=np.int64)
                assert np.array_equal(host(t).astype(np.int64).reshape(w.shape) & 0xFFFFFFFF, w & 0xFFFFFFFF), name
        if pools:
            assert np.array_equal(host(self.hot_k).view(np.int16), k.view(np.int16))
            assert np.array_equal(host(self.hot_v).view(np.int16), v.view(np.int16))


ACCEPT = {"one": dict(counts=[1]), "ragged": dict(counts=[5, 1, 0, 17, 40], pad=3), "deep": dict(counts=[64, 65, 3], agree=1.0, shape="chain", history=200),
          "wide": dict(counts=[300, 64], agree=1.0), "longest": dict(counts=[1024, 2], agree=1.0, shape="chain", layers=1, history=2100),
          "longest_random": dict(counts=[1024], agree=1.0, layers=1), "star": dict(counts=[200, 9], shape=1, agree=1.0), "none": dict(counts=[0, 0], pad=2),
          "odd_rows": dict(counts=[6, 9], hk=3, hd=7), "layers": dict(counts=[4, 4, 4], layers=33), "many": dict(counts=[i % 3 for i in range(500)], layers=1)}


@pytest.mark.parametrize("name", sorted(ACCEPT))
def test_accept(ops, engine, name):
    c = Accept(len(name), **ACCEPT[name])
    ops.accept_tree(c.desc())
    assert error_of(engine) == ""
    c.check()


def test_accept_without_rows_without_history_in_place(ops, engine):
    c = Accept(1, [5, 9, 2], agree=1.0)
    ops.accept_tree(c.desc(layers=0, kv_heads=0, head_dim=0, k=None, v=None, hot_k=None, hot_v=None, slots=None))
    c.check(pools=False)
    ops.accept_tree(c.desc(history=None, history_count=None, history_count_out=None))
    c.check(skip=("history", "history_count_out"))
    held, count = dev(c.held), dev(c.count)
    d = c.desc(seq_held=held, seq_hot=held, history_count=count, history_count_out=count)
    c.got.update(seq_hot=held, history_count_out=count)
    ops.accept_tree(d)
    c.check()
    d = c.desc(v=None, hot_v=None)  # K rows are the values
    ops.accept_tree(d)
    before = c.hot_v
    c.hot_v = dev(-c.pool)
    assert np.array_equal(host(before), host(c.hot_v))
    assert error_of(engine) == ""


def test_accept_rows_of_fused_products(ops):
    import torch
    c = Accept(2, [7, 12], layers=3)
    rows = torch.zeros((3, c.rows, 9, 64), dtype=torch.float16, device="cuda:0")
    k, v = rows[:, :, 5:7], rows[:, :, 7:9]
    k.copy_(dev(c.k))
    v.copy_(dev(c.v))
    ops.accept_tree(c.desc(k=k, v=v))
    c.check()
    flat = torch.zeros(3 * c.rows * 128 + 1, dtype=torch.float16, device="cuda:0")[1:].view(3, c.rows, 2, 64)  # not 16-byte aligned
    flat.copy_(dev(c.k))
    ops.accept_tree(c.desc(k=flat))
    c.check()


def test_accept_reports(ops, engine):
    import torch
    c = Accept(3, [5, 9, 2], agree=1.0, history=60)
    bad = c.slots.copy()
    bad[0], bad[6], bad[14] = c.blocks * 16, -1, 1 << 40
    ops.accept_tree(c.desc(slots=torch.from_numpy(bad).cuda()))
    assert "hot block ref" in error_of(engine)
    c.check(slots=bad)
    bad[0], bad[14] = -1, -5  # tokens without a page are no error here
    ops.accept_tree(c.desc(slots=torch.from_numpy(bad).cuda()))
    assert error_of(engine) == ""
    c.check(slots=bad)
    d = c.desc(history_count=dev(np.array([60, 59, 70])))
    ops.accept_tree(d)
    assert "sequence length" in error_of(engine)
    assert host(c.got["history_count_out"]).tolist() == [60, 60, 60]
    c = Accept(4, [1500, 3], agree=1.0, shape="chain", layers=1, history=3000)
    ops.accept_tree(c.desc())
    assert "sequence length" in error_of(engine)
    c.check()


def test_accept_a_target_that_is_no_token(ops, engine):
    c = Accept(5, [5, 9, 2, 33], agree=1.0)
    c.tokens[[1, 2, 3, 6, 7, 17, 18]] = 0xFFFFFFFF
    c.targets[[0, 5, 16]] = 0xFFFFFFFF  # a best of -1: nothing continues it, also not a token of the same bits
    ops.accept_tree(c.desc())
    assert error_of(engine) == ""
    c.check()


# ---------------------------------------------------------------- streams and graphs

def test_each_call_in_a_graph(ops, engine):
    """Captured and replayed with other inputs and eager work in between."""
    import torch
    t, l, a = Tables(7, [3, 20, 0, 31], [14, 40, 2, 9], tree="random"), Logits(7, 40001, [3, 5], history=50, bias=5, allowed=0.5), \
        Accept(7, [5, 9, 2], agree=1.0)
    calls = [(ops.page_tables, t.desc()), (ops.adjust_logits, l.desc()), (ops.accept_tree, a.desc())]
    for f, d in calls:
        f(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f, d in calls:
            f(d)
    for i in range(3):
        l.x = np.roll(l.x, 1, axis=1)
        l.src.copy_(dev(l.x))
        for x in (t.got["slots"], t.got["positions"], l.out, l.best, a.got["path"]):
            x.fill_(-77)
        other = Logits(8 + i, 30011, [2], history=9)
        ops.adjust_logits(other.desc())  # the same workspace, eagerly
        other.check()
        graph.replay()
        torch.cuda.synchronize()
        t.check(t.want())
        l.check()
        a.check()
    assert error_of(engine) == ""


def test_on_another_stream(ops, engine):
    import torch
    s = torch.cuda.Stream()
    c = Logits(9, 50000, [4, 4], history=100)
    d = c.desc()
    t = Tables(9, [3, 20], [14, 40])
    td = t.desc()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adjust_logits(d)
        ops.page_tables(td)
    s.synchronize()
    c.check()
    t.check(t.want())


def test_calls_of_no_rows(ops, engine):
    from aether_nexus_amd import ops as O
    ops.adjust_logits(O.make_logits_desc(num_tokens=0, vocab_size=9, logits=None, out=None, best=empty(1)))
    ops.accept_tree(O.make_accept_desc(batch=0, num_tokens=0, parents=None, node_tokens=None, targets=None, seq_held=None, accepted=None,
                                       next_token=None, seq_hot=None, path=None))
    assert error_of(engine) == ""
