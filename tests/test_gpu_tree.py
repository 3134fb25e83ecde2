"""Attention of trees over pages on cuda:0 through the C ABI against the float64 oracle
(oracle/step_oracle.py).  The tolerance is that of helpers.prefix_errors: the f16 store, weights as
f16 operands, fp32 scores and sums."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import prefix_errors
from oracle import step_oracle as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(engine):
    from aether_nexus_amd.ops import OpsEngine
    return OpsEngine(engine)


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype == np.float16:
        return torch.from_numpy(a.view(np.int16).copy()).cuda().view(torch.float16)
    return torch.from_numpy(a.astype(np.int64) & 0xFFFFFFFF).to(torch.int32).cuda()


def host(t):
    import torch
    torch.cuda.synchronize()
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.float16)


def error_of(engine):
    from aether_nexus_amd.weaver import WeaverError
    try:
        engine.check_device_errors()
    except WeaverError as e:
        return str(e)
    return ""


STALE = np.array([np.nan, np.inf, -np.inf, 65504.0], dtype=np.float16)


class Case:
    """Inputs of one request: pages in a mixed order, stale rows (NaN, inf) wherever no token is, rows of one fused
    product (q, k, v side by side), nodes behind the last sequence stale too."""

    def __init__(self, seed, hq, hk, hd, nodes, held, *, chain=False, pad=0, fused=True, qscale=1.5, spare=0, words=None):
        rng = self.rng = np.random.default_rng(seed)
        self.heads = (hq, hk, hd)
        self.nodes, self.held = list(nodes), np.asarray(held)
        self.offsets = S.offsets_of(nodes)
        total, self.rows = int(sum(nodes)), int(sum(nodes)) + pad
        pages = [-(-int(h) // 16) for h in held]
        self.blocks = sum(pages) + 2
        order = rng.permutation(self.blocks).astype(np.int64)
        self.count = max(pages + [0]) + spare
        self.refs = np.full((len(nodes), max(self.count, 1)), 0x7FFFFFFF, dtype=np.int64)
        at = 0
        for b, n in enumerate(pages):
            self.refs[b, :n] = order[at:at + n]
            at += n
        self.hot_k, self.hot_v = (rng.standard_normal((self.blocks, 16, hk, hd)).astype(np.float16) for _ in range(2))
        live = np.zeros((self.blocks, 16), dtype=bool)
        for b, h in enumerate(held):
            t = np.arange(int(h))
            live[self.refs[b][t // 16], t % 16] = True
        for p in (self.hot_k, self.hot_v):
            p[~live] = STALE[rng.integers(0, 4, p[~live].shape)]
        self.refs[:, ::2] |= 1 << 31  # masked
        self.q = (rng.standard_normal((self.rows, hq, hd)) * qscale).astype(np.float16)
        self.k, self.v = (rng.standard_normal((self.rows, hk, hd)).astype(np.float16) for _ in range(2))
        for p in (self.k, self.v):
            p[total:] = STALE[rng.integers(0, 4, p[total:].shape)]
        self.trees = [[-1 if i == 0 else int(rng.integers(0, i)) for i in range(n)] for n in nodes]
        words = -(-max(max(nodes, default=1), 1) // 32) if words is None else words
        self.mask = None if chain else S.mask_of(self.trees, self.rows, words)
        self.fused = fused

    def desc(self, **kw):
        import torch
        from aether_nexus_amd import ops as O
        hq, hk, hd = self.heads
        if self.fused:
            rows = dev(np.concatenate([self.q, self.k, self.v], 1))
            q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        else:
            q, k, v = dev(self.q), dev(self.k), dev(self.v)
        self.out = torch.full((self.rows, hq, hd), 7.0, dtype=torch.float16, device="cuda:0")
        base = dict(batch=len(self.nodes), num_tokens=self.rows, q_heads=hq, kv_heads=hk, head_dim=hd, q=q, k=k, v=v, out=self.out,
                    hot_count=self.count, token_offsets=dev(np.array(self.offsets)), tree_mask=None if self.mask is None else dev(self.mask))
        if self.count:
            base.update(hot_k=dev(self.hot_k), hot_v=dev(self.hot_v), refs=dev(self.refs), seq_held=dev(self.held))
        return O.make_tree_desc(**{**base, **kw})

    def want(self, **kw):
        base = dict(q=self.q, k=self.k, v=self.v, hot_k=self.hot_k, hot_v=self.hot_v, refs=self.refs, held=self.held, offsets=self.offsets,
                    mask=self.mask, scale=self.heads[2] ** -0.5)
        with np.errstate(all="ignore"):
            return S.tree_attention(**{**base, **kw})

    def check(self, what, out=None, largest=6.0, **kw):
        want, absolute, total = self.want(**kw)
        n = int(self.offsets[-1])
        got = host(self.out if out is None else out)
        assert (got[n:] == (7.0 if out is None else got[n:])).all(), f"{what}: rows behind the last sequence"
        got = got[:n].astype(np.float64)
        assert np.isfinite(got).all(), what
        if n:
            worst, _ = prefix_errors(got, want[:n], absolute[:n], total[:n], int(self.held.max(initial=0)) + max(self.nodes), largest)
            print(f"{what}: worst error over tolerance {worst:.3f}", flush=True)
            assert worst <= 1.0, what


# q heads, kv heads, head_dim, nodes of each sequence, tokens of each in pages
CASES = [
    (1, 1, 64, [1], [0]), (4, 1, 128, [1], [1]), (14, 2, 64, [5, 1], [700, 3]), (32, 8, 128, [8, 1, 3], [16, 17, 15]),
    (32, 8, 128, [1, 0, 4, 8], [1000, 33, 0, 200]), (8, 2, 64, [2, 40], [33, 64]), (32, 8, 64, [60, 1, 7], [515, 100, 47]),
    (12, 2, 128, [33, 5], [300, 5]), (8, 8, 128, [0, 1, 0, 31, 32], [0, 257, 9, 0, 31]), (14, 2, 64, [64, 65], [1500, 128]),
    (4, 2, 128, [70, 150], [130, 1]), (32, 8, 128, [i % 4 for i in range(33)], [7 * i for i in range(33)]), (32, 8, 128, [1], [5000]),
    (12, 2, 128, [2] * 130, [95] * 130), (70, 1, 64, [3, 9], [31, 400]), (2, 1, 64, [0, 5, 0, 16, 3, 0, 1], [0] * 7), (6, 3, 128, [2, 0, 1], [63, 64, 65]),
    (2, 2, 64, [1, 1], [20000, 3]), (4, 1, 64, [257], [40]), (3, 1, 128, [128, 129], [100, 700]), (2, 1, 64, [1024, 3], [70, 2000]),
    (8, 4, 64, [1] * 1500, [i % 50 for i in range(1500)]), (16, 1, 128, [8, 9, 4], [63, 128, 1025]), (32, 8, 64, [16, 16], [4096, 4096]),
]


@pytest.mark.parametrize("chain", [False, True], ids=["tree", "chain"])
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c[:3])) + f"-{len(c[3])}x{max(c[3])}-{max(c[4])}" for c in CASES])
def test_against_float64(ops, engine, case, chain):
    c = Case(sum(case[:3]) + sum(case[3]), *case, chain=chain, pad=len(case[3]) % 3, fused=sum(case[3]) % 2 == 0)
    d = c.desc()
    ops.tree_attention(d)
    assert error_of(engine) == ""
    c.check(f"{case[:3]} {len(case[3])} sequences")


def test_rows_that_see_nothing(ops, engine):
    c = Case(1, 8, 2, 64, [5, 40, 3, 3], [0, 0, 17, 0])
    c.mask[2] = c.mask[7] = c.mask[45] = 0  # the third: its pages alone
    c.mask[48:] = 0
    ops.tree_attention(c.desc())
    assert error_of(engine) == ""
    c.check("empty masks")
    got = host(c.out)
    assert (got[[2, 7, 48, 49, 50]] == 0).all() and (got[45] != 0).any()


def test_masks_of_any_shape(ops):
    """Bits are taken as they are: nodes behind a row, not itself, beyond the sequence (no row of which exists)."""
    c = Case(2, 8, 2, 128, [70, 3, 64], [90, 0, 16], words=3)
    c.mask = c.rng.integers(0, 1 << 32, c.mask.shape)
    ops.tree_attention(c.desc())
    c.check("random masks")


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-30])
def test_scales(ops, scale):
    c = Case(3, 8, 2, 64, [9, 20], [100, 33], qscale=0.7)
    ops.tree_attention(c.desc(scale=scale))
    c.check(f"scale {scale}", scale=float(np.float32(scale)))


def test_values_that_are_not_seen_never_arrive(ops):
    """NaN and infinities in nodes that no row sees but themselves, and rows that see them."""
    for hd in (64, 128):
        c = Case(4, 8, 2, hd, [40, 70], [50, 1])
        for p in (c.k, c.v):
            p[5] = np.nan
            p[44, 0] = np.inf
        c.mask[:, 0] &= ~np.uint32(1 << 5)
        c.mask[40:, 0] &= ~np.uint32(1 << 4)
        want, absolute, total = c.want(k=np.nan_to_num(c.k, nan=0, posinf=0), v=np.nan_to_num(c.v, nan=0, posinf=0))
        ops.tree_attention(c.desc())
        got = host(c.out).astype(np.float64)
        worst, _ = prefix_errors(got, want, absolute, total, 120, 6.0)
        assert np.isfinite(got).all() and worst <= 1.0
        # Seen by one row each: that row alone is not finite, in the dims that are not.
        c = Case(5, 8, 2, hd, [40, 70], [50, 1])
        c.v[3, 1, 7] = np.inf
        c.v[60, 0, 9] = np.nan
        for r in range(110):
            c.mask[r, 0] &= ~np.uint32(1 << 3 if r < 40 else 1 << 20)
        c.mask[9, 0] |= 1 << 3
        c.mask[77, 0] |= 1 << 20
        ops.tree_attention(c.desc())
        got = host(c.out).astype(np.float64)
        bad = np.argwhere(~np.isfinite(got))
        assert sorted(map(tuple, bad)) == [(9, h, 7) for h in range(4, 8)] + [(77, h, 9) for h in range(4)]
        assert (got[9, 4:, 7] == np.inf).all()


def test_infinite_values_in_pages(ops):
    for hd in (64, 128):
        for n in (2, 40):
            c = Case(6, 8, 2, hd, [n, n], [200, 77])
            row = (int(c.refs[0, 5]) & 0x7FFFFFFF, 3)
            c.hot_v[row][1, 11] = -np.inf
            ops.tree_attention(c.desc())
            got = host(c.out).astype(np.float64)
            bad = np.argwhere(~np.isfinite(got))
            assert sorted(map(tuple, bad)) == [(r, h, 11) for r in range(n) for h in range(4, 8)]


def test_bad_refs_hide_their_tokens(ops, engine):
    c = Case(7, 8, 2, 64, [3, 20], [300, 40], spare=1)
    c.refs[0, 3], c.refs[0, 18], c.refs[1, 0] = c.blocks, 0x7FFFFFFF, c.blocks + 5
    ops.tree_attention(c.desc())
    assert "hot block ref" in error_of(engine)
    c.check("bad refs")
    c = Case(8, 8, 2, 128, [3], [33])
    c.refs[:] = 1 << 30
    ops.tree_attention(c.desc())
    assert "hot block ref" in error_of(engine)
    c.check("no page left")


def test_lengths_past_the_table(ops, engine):
    c = Case(9, 8, 2, 64, [3, 20], [48, 48])
    d = c.desc(seq_held=dev(np.array([49, 1 << 31])))
    ops.tree_attention(d)
    assert "sequence length" in error_of(engine)
    c.check("taken as the table's")
    c = Case(10, 8, 2, 64, [3, 40], [48, 17], words=1)  # 8 nodes past the mask: seen by none
    ops.tree_attention(c.desc())
    assert "sequence length" in error_of(engine)
    c.check("nodes past the mask")


@pytest.mark.parametrize("offsets", [[0, 9, 3], [0, 3, 40], [5, 2, 23]])
def test_offsets_that_descend_or_pass_the_rows(ops, engine, offsets):
    """Reported; rows that no sequence holds are left as they are, none but the request's rows are read or written."""
    c = Case(11, 8, 2, 64, [3, 20], [48, 17])
    ops.tree_attention(c.desc(token_offsets=dev(np.array(offsets))))
    assert "sequence length" in error_of(engine)


def test_rows_that_share_equally_and_k_as_values(ops, engine):
    c = Case(12, 12, 2, 128, [7, 7, 7], [48, 17, 0], fused=False)
    ops.tree_attention(c.desc(token_offsets=None))
    c.check("equal parts")
    ops.tree_attention(c.desc(v=None, hot_v=None))
    c.check("K rows are the values", v=c.k, hot_v=c.hot_k)
    assert error_of(engine) == ""


def test_in_place_and_strided_outputs(ops):
    import torch
    c = Case(13, 8, 2, 64, [7, 70], [48, 300])
    d = c.desc()
    d.out, d.out_stride = d.q, d.q_stride
    rows = d._keep[0]
    ops.tree_attention(d)
    c.check("in place", out=rows)
    wide = torch.full((c.rows, 8 * 64 + 12), 7.0, dtype=torch.float16, device="cuda:0")
    d = c.desc(out=wide[:, 4:4 + 8 * 64])
    ops.tree_attention(d)
    c.check("rows apart", out=wide[:, 4:516].reshape(c.rows, 8, 64))
    assert (host(wide)[:, :4] == 7).all() and (host(wide)[:, 516:] == 7).all()


def test_captured_and_on_another_stream(ops, engine):
    import torch
    c = Case(14, 32, 8, 128, [60, 9], [3000, 1000])
    d = c.desc()
    ops.tree_attention(d)
    torch.cuda.synchronize()
    eager = host(c.out).copy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(d)
    for i in range(3):
        c.out.fill_(7.0)
        other = Case(20 + i, 8, 2, 64, [5, 80], [900, 30])
        ops.tree_attention(other.desc())  # the same workspace, eagerly
        other.check("between replays")
        graph.replay()
        assert np.array_equal(host(c.out).view(np.int16), eager.view(np.int16))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.out.fill_(7.0)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.tree_attention(d)
    s.synchronize()
    assert np.array_equal(host(c.out).view(np.int16), eager.view(np.int16))
    c.check("eager")
    assert error_of(engine) == ""


def test_pages_past_32_bits(ops):
    """Pages whose rows lie past 2^32 bytes of the pool."""
    import torch
    hk, hd = 8, 128
    blocks = (1 << 32) // (16 * hk * hd * 2) + 40
    c = Case(15, 16, hk, hd, [9], [100], fused=False)
    k, v = (torch.zeros((blocks, 16, hk, hd), dtype=torch.float16, device="cuda:0") for _ in range(2))
    n = c.blocks
    k[-n:], v[-n:] = dev(c.hot_k), dev(c.hot_v)
    refs = c.refs.copy()
    refs[:, :7] = (refs[:, :7] & 0x7FFFFFFF) + blocks - n
    ops.tree_attention(c.desc(hot_k=k, hot_v=v, refs=dev(refs)))
    c.check("far pages")


@pytest.mark.parametrize("hd", [64, 128])
def test_a_lost_page_shows(ops, hd):
    """Scores of one size: every token counts equally, and a page left out or taken twice is past the tolerance."""
    c = Case(16, 8, 2, hd, [40, 3], [1500, 777])
    c.q[:] = 0
    for p in (c.hot_v, c.v):
        np.copyto(p, 1.0, where=np.isfinite(p))
    at = (int(c.refs[0, 50]) & 0x7FFFFFFF)
    c.hot_v[at] = 65.0
    ops.tree_attention(c.desc())
    c.check("equal weights", largest=65.0)
    want = (1500 - 16 + 16 * 65.0 + np.array([bin(int(c.mask[r, 0]) | int(c.mask[r, 1]) << 32).count("1") for r in range(40)])) / \
        (1500 + np.array([bin(int(c.mask[r, 0]) | int(c.mask[r, 1]) << 32).count("1") for r in range(40)]))
    assert np.abs(host(c.out)[:40].astype(np.float64) - want[:, None, None]).max() < 0.002


# A table far wider than the lengths (spare) has the steps planned for it shared out, few of which there are.
WAYS = [  # heads, nodes, held, entries of the table that no length reaches, query rows of a unit (0: one launch)
    (32, 8, 64, [4] * 40, [50 + i for i in range(40)], 0, 0), (32, 8, 128, [4, 0, 9, 5] * 8, [3 * i for i in range(32)], 0, 0),
    (32, 8, 128, [3, 5], [700, 64], 0, 0), (14, 2, 64, [30, 2], [900, 1], 0, 0),
    (8, 2, 64, [3, 4, 1, 0, 5], [300, 0, 1025, 77, 64], 3000, 16), (8, 2, 128, [3, 4, 1, 0, 5], [300, 0, 1025, 77, 64], 3000, 16),
    (8, 2, 64, [7, 8, 0, 9], [300, 0, 63, 1100], 8000, 32), (8, 2, 128, [7, 8, 1, 9], [300, 0, 63, 1100], 8000, 32),
    (8, 2, 64, [40, 33, 64, 1], [300, 0, 1025, 77], 9000, 128), (8, 2, 128, [40, 33, 64, 1], [300, 0, 1025, 77], 9000, 128),
    (6, 2, 64, [i % 3 for i in range(300)], [11 * i % 90 for i in range(300)], 500, 16),
    (6, 2, 128, [8 + i % 3 for i in range(260)], [11 * i % 90 for i in range(260)], 400, 32),
    (6, 2, 64, [16 + i % 3 for i in range(257)], [11 * i % 90 for i in range(257)], 400, 128),
    (4, 1, 128, [1], [40000], 0, 16), (20, 1, 64, [1], [33333], 16900, 32), (5, 1, 64, [130], [20000], 60000, 128), (5, 1, 128, [130], [20000], 60000, 128),
]


@pytest.mark.parametrize("way", WAYS, ids=[f"{c[0]}-{c[1]}-{c[2]}-{len(c[3])}x{max(c[3])}-{c[6]}" for c in WAYS])
def test_each_way_to_split(ops, engine, way):
    import torch
    from aether_nexus_amd import ops as O
    hq, hk, hd, nodes, held, spare, tile = way
    c = Case(31, hq, hk, hd, nodes, held, pad=3, spare=spare, qscale=1.0)
    d = c.desc()
    plan = O.tree_plan(d, torch.cuda.get_device_properties(0).multi_processor_count)
    assert (plan.row_tile if plan.workspace_bytes else 0) == tile
    ops.tree_attention(d)
    assert error_of(engine) == ""
    c.check("split")
    first = host(c.out).copy()
    c.out.fill_(7.0)
    ops.tree_attention(d)
    assert np.array_equal(host(c.out).view(np.int16), first.view(np.int16))  # parts are joined in one order


@pytest.mark.parametrize("tile", [16, 128])
def test_offsets_that_descend_where_steps_are_shared_out(ops, engine, tile):
    from aether_nexus_amd import ops as O
    nodes = [3, 0] * 150 if tile == 16 else [40, 0] * 6
    c = Case(32, 8, 2, 64, nodes, [90] * len(nodes), spare=9000, pad=2)
    n = c.rows
    d = c.desc(token_offsets=dev(np.array([0, n] * (len(nodes) // 2) + [0])))  # every other sequence has all rows, the rest descend
    assert O.tree_plan(d).row_tile == tile
    ops.tree_attention(d)
    assert "sequence length" in error_of(engine)
    got = host(c.out)
    assert np.isfinite(got[:sum(nodes)].astype(np.float64)).all()
