"""Shared-prefix attention on cuda:0 through the C ABI against the float64 oracle
(oracle/paged_oracle.py).

Tolerance of an output o = sum p v / sum p over n tokens, with A = sum p |v| / sum p:
half a step of the f16 store, 2^-11 |o|; the weights as f16 operands, each off by half a
step, together 2^-11 A at most, or 2^-25 (of the largest weight, 1) among the subnormals,
together n 2^-25 max |v|; the scores' fp32 sums of head_dim products, off by at most
head_dim 2^-24 scale sum |q k| <= 128 2^-24 12 = 0.2 2^-11 for the values drawn here, in
the weights and in their sum: 0.4 2^-11 A; exp2, rescaling and joining a few 2^-24 A.
Together 2^-11 |o| + 1.5 2^-11 A + n 2^-25 max |v| + 2^-25."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import LONG_PREFIXES, PREFIX_REL_L2, prefix_errors
from oracle import paged_oracle as P

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
    return torch.from_numpy(a.astype(np.uint32).view(np.int32).copy()).cuda()


def host(t):
    import torch
    torch.cuda.synchronize()
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.float16)


def plan(c):
    from aether_nexus_amd import ops as O
    return O.prefix_plan(c.desc())


class Case:
    """Inputs of one request: pages in a mixed order, stale rows (NaN, inf) wherever no token is."""

    def __init__(self, seed, batch, queries, hq, hk, hd, prefix, own, *, causal=True, stale=True, qscale=1.5, spare=0):
        rng = self.rng = np.random.default_rng(seed)
        self.shape = (batch, queries, hq, hk, hd)
        self.prefix, self.own, self.causal = prefix, np.asarray(own), causal
        pages = [-(-int(n) // 16) for n in own]
        np_ = -(-prefix // 16)
        self.blocks = np_ + sum(pages) + 2
        order = rng.permutation(self.blocks).astype(np.int64)
        self.count = max(pages + [0]) + spare
        self.prefix_refs = order[:np_]
        self.refs = np.full((batch, max(self.count, 1)), 0x7FFFFFFF, dtype=np.int64)
        at = np_
        for b, n in enumerate(pages):
            self.refs[b, :n] = order[at:at + n]
            at += n
        self.q = (rng.standard_normal((batch, queries, hq, hd)) * qscale).astype(np.float16)
        bad = np.array([np.nan, np.inf, -np.inf, 65504.0], dtype=np.float16)
        self.k, self.v = (rng.standard_normal((self.blocks, 16, hk, hd)).astype(np.float16) for _ in range(2))
        if stale:
            live = np.zeros((self.blocks, 16), dtype=bool)
            for table, n in [(self.prefix_refs, prefix)] + [(self.refs[b], int(n)) for b, n in enumerate(own)]:
                t = np.arange(n)
                live[table[t // 16], t % 16] = True
            for p in (self.k, self.v):
                p[~live] = bad[rng.integers(0, 4, p[~live].shape)]
        self.prefix_refs[::2] |= 1 << 31  # masked
        self.dq, self.dk, self.dv = dev(self.q), dev(self.k), dev(self.v)
        self.drefs, self.dprefix, self.down = dev(self.refs), dev(self.prefix_refs), dev(self.own)

    def desc(self, **kw):
        import torch
        from aether_nexus_amd import ops as O
        batch, queries, hq, hk, hd = self.shape
        self.out = torch.full((batch, queries, hq, hd), float("nan"), dtype=torch.float16, device="cuda:0")
        base = dict(batch=batch, queries=queries, q_heads=hq, kv_heads=hk, head_dim=hd, prefix_tokens=self.prefix, q=self.dq,
                    out=self.out, hot_k=self.dk, hot_v=self.dv, prefix_refs=self.dprefix if self.prefix else None,
                    own_count=self.count, refs=self.drefs if self.count else None, seq_own=self.down, causal=self.causal)
        return O.make_prefix_desc(**{**base, **kw})

    def want(self, own=None, scale=None, values=None, refs=None, prefix_refs=None):
        scale = self.shape[4] ** -0.5 if scale is None else scale
        a = (self.prefix_refs if prefix_refs is None else prefix_refs, self.prefix, self.refs if refs is None else refs,
             self.own if own is None else own, scale, self.causal)
        v = self.v if values is None else values
        with np.errstate(all="ignore"):
            return (P.shared_prefix_attention(self.q, self.k, v, *a), P.shared_prefix_attention(self.q, self.k, np.abs(v), *a))

    def check(self, what, **kw):
        want, absolute = self.want(**kw)
        got = host(self.out).astype(np.float64)
        n = self.prefix + int(self.own.max(initial=0))
        tol = 2.0 ** -11 * np.abs(want) + 1.5 * 2.0 ** -11 * absolute + (n * 6.0 + 1) * 2.0 ** -25
        d = np.abs(got - want)
        print(f"{what}: worst error over tolerance {float((d / tol).max()):.3f}, rel {np.linalg.norm(d) / max(np.linalg.norm(want), 1e-30):.2e}",
              flush=True)
        assert np.isfinite(got).all() and np.all(d <= tol), what


# batch, queries, q heads, kv heads, head_dim, prefix, own tokens of each sequence
CASES = [
    (1, 1, 1, 1, 64, 1, [1]), (1, 1, 4, 1, 128, 0, [1]), (2, 1, 14, 2, 64, 117, [9, 1]), (3, 1, 32, 8, 128, 16, [16, 17, 15]),
    (4, 1, 32, 8, 128, 1000, [1, 33, 64, 200]), (2, 2, 8, 2, 64, 33, [2, 40]), (3, 8, 32, 8, 64, 515, [8, 100, 47]),
    (2, 5, 12, 2, 128, 64, [300, 5]), (5, 1, 8, 8, 128, 257, [0, 1, 0, 31, 32]), (1, 40, 14, 2, 64, 77, [53]),
    (2, 70, 4, 2, 128, 130, [70, 150]), (33, 1, 32, 8, 128, 300, list(range(33))), (1, 1, 32, 8, 128, 5000, [1]),
    (130, 1, 12, 2, 128, 95, [7] * 130), (1, 3, 70, 1, 64, 31, [4]), (2, 1, 4, 2, 128, 48, [1000, 2]), (7, 1, 2, 1, 64, 0, [0, 5, 0, 16, 3, 0, 1]),
    (3, 2, 6, 3, 128, 63, [0, 1, 2]), (16, 8, 32, 8, 64, 640, [8 + i for i in range(16)]), (1, 1, 2, 2, 64, 20000, [0]),
]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c[:6])) for c in CASES])
def test_against_float64(ops, engine, case, causal):
    c = Case(sum(case[:6]), *case, causal=causal)
    ops.shared_prefix_attention(c.desc())
    engine.check_device_errors()
    c.check(f"{case[:6]}")


def test_own_pages_only_and_prefix_only(ops, engine):
    c = Case(1, 3, 2, 8, 2, 128, 0, [5, 40, 17])
    ops.shared_prefix_attention(c.desc(prefix_refs=None))
    c.check("own pages only")
    c = Case(2, 3, 2, 8, 2, 128, 70, [0, 0, 0])
    ops.shared_prefix_attention(c.desc(own_count=0, refs=None, seq_own=None))
    c.check("prefix only")
    c = Case(3, 2, 1, 8, 2, 64, 10, [32, 32])  # every own row is taken without counts
    ops.shared_prefix_attention(c.desc(seq_own=None))
    c.check("without counts")
    c = Case(4, 3, 2, 8, 2, 128, 0, [0, 0, 0])
    ops.shared_prefix_attention(c.desc(own_count=0, refs=None))
    assert not host(c.out).any()  # nothing to see
    engine.check_device_errors()


@pytest.mark.parametrize("case", [(3, 2, 8, 2, 128, 100, [5, 40, 17]), (40, 1, 8, 2, 64, 5000, [3] * 40)], ids=["small", "tiles"])
def test_output_in_place_of_the_queries(ops, case):
    c = Case(12, *case)
    out = c.dq.clone()
    ops.shared_prefix_attention(c.desc(q=out, out=out))
    c.out = out
    c.check("in place")


def test_keys_that_are_the_values(ops):
    c = Case(5, 3, 1, 8, 2, 128, 100, [5, 40, 17])
    ops.shared_prefix_attention(c.desc(hot_v=None))
    c.check("K rows as values", values=c.k)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 2.0 ** -30])
def test_scales(ops, scale):
    """A negative scale turns the order of the scores round; a scale of 0 weighs every token that is seen alike."""
    for batch in (2, 20):
        c = Case(50, batch, 2, 8, 2, 128, 100, [5, 40] + [3] * (batch - 2))
        ops.shared_prefix_attention(c.desc(scale=scale))
        c.check(f"scale {scale}", scale=scale)


def test_peaked_and_flat_scores(ops):
    """Scores so far apart that one token takes all of the weight, the largest in the last part; equal scores."""
    c = Case(6, 2, 1, 8, 2, 128, 900, [40, 8], qscale=40.0)
    ops.shared_prefix_attention(c.desc(scale=0.25))
    want, _ = c.want(scale=0.25)
    got = host(c.out).astype(np.float64)
    # scores are off by at most 128 2^-24 scale sum |q k| < 128 2^-24 0.25 128 40 6.25 = 0.061 where they are largest; but sums
    # of random signs are far from that bound, and rows whose two best scores are closer than 0.1 are left out
    k = np.concatenate([c.k[c.prefix_refs & P.REF_MASK].reshape(-1, 2, 128)[:900], c.k[c.refs[0, :3]].reshape(-1, 2, 128)[:40]])
    s = np.einsum("hd,nhd->hn", c.q[0, 0].astype(np.float64), np.repeat(k, 4, axis=1).astype(np.float64)) * 0.25
    top = np.sort(s, axis=1)
    rows = top[:, -1] - top[:, -2] > 12.0  # the next weights are below e^-12: 900 of them under 2^-7... of the largest
    assert rows.sum() >= 4
    v = np.concatenate([c.v[c.prefix_refs & P.REF_MASK].reshape(-1, 2, 128)[:900], c.v[c.refs[0, :3]].reshape(-1, 2, 128)[:40]])
    best = np.take_along_axis(np.repeat(v, 4, axis=1).astype(np.float64), s.argmax(1)[None, :, None], 0)[0]
    assert np.all(np.abs(got[0, 0][rows] - best[rows]) <= 900 * np.exp(-11.9) * 12 + 2.0 ** -11 * np.abs(best[rows]))
    assert np.isfinite(got).all()
    c = Case(7, 2, 1, 8, 2, 128, 900, [40, 8], qscale=0.0)
    ops.shared_prefix_attention(c.desc())
    c.check("equal scores")


@pytest.mark.parametrize("hd", [64, 128])
def test_infinities_reach_only_the_rows_that_see_them(ops, hd):
    """Draft tokens whose values hold infinities and NaNs are hidden from earlier drafts; those that see them get
    them in those dims alone.  The same in the prefix, which every row sees."""
    for queries, prefix in ((4, 50), (9, 0), (1, 200)):
        c = Case(8 + queries, 2, queries, 8, 2, hd, prefix, [queries + 10, queries])
        values = c.v.copy()

        def put(b, token, g, dim, x):
            values[c.refs[b, token // 16], token % 16, g, dim] = x
        put(0, queries + 9, 0, 3, np.inf)            # the last draft: only the last row sees it
        put(1, queries - 1, 1, hd - 1, np.nan)
        if queries > 2:
            put(0, queries + 7, 1, 17, -np.inf)      # the third last
        if prefix:
            at = c.prefix_refs[2] & P.REF_MASK
            values[at, 5, 0, 9] = np.inf             # every row of head 0
        c.v, c.dv = values, dev(values)
        ops.shared_prefix_attention(c.desc())
        got = host(c.out).astype(np.float64)
        finite = np.where(np.isfinite(values), values, 0).astype(np.float16)
        want, absolute = c.want(values=finite)
        bad = np.zeros(got.shape, dtype=bool)
        bad[0, queries - 1, :4, 3] = bad[1, queries - 1, 4:, hd - 1] = True
        if queries > 2:
            bad[0, queries - 3:, 4:, 17] = True
        if prefix:
            bad[:, :, :4, 9] = True
        assert np.array_equal(~np.isfinite(got), bad), (queries, prefix)
        assert np.all(np.isposinf(got[0, queries - 1, :4, 3])) and np.all(np.isnan(got[1, queries - 1, 4:, hd - 1]))
        tol = 2.0 ** -11 * np.abs(want) + 1.5 * 2.0 ** -11 * absolute + 1500 * 2.0 ** -25
        assert np.all((np.abs(got - want) <= tol)[~bad])


# Requests whose prefix is read by work-groups of 128 rows: parts of one step and of several, both widths, partial last pages
TILES = [(33, 1, 8, 2, 128, 1700), (20, 2, 16, 16, 64, 1030), (9, 16, 4, 2, 64, 3500), (40, 1, 32, 32, 128, 777),
         (70, 1, 64, 64, 64, 389), (12, 8, 24, 8, 128, 3001), (33, 1, 16, 16, 64, 2900), (40, 1, 32, 32, 128, 2000),
         (18, 2, 32, 32, 128, 2500), (40, 1, 64, 64, 64, 1500)]


@pytest.mark.parametrize("case", TILES, ids=["-".join(map(str, c)) for c in TILES])
def test_many_rows_behind_a_prefix(ops, engine, case):
    """Stale rows of the last page, keys as the values, scales of either sign, infinities and NaNs in keys and values."""
    batch, queries, hq, hk, hd, prefix = case
    own = [queries + b % 5 for b in range(batch)]
    c = Case(60, *case, own)
    p = plan(c)
    assert p.row_tile == 128 and p.prefix_splits > 1
    ops.shared_prefix_attention(c.desc())
    c.check("random")
    ops.shared_prefix_attention(c.desc(scale=-0.05))
    c.check("a negative scale", scale=-0.05)
    ops.shared_prefix_attention(c.desc(hot_v=None))
    c.check("K rows as values", values=c.k)
    # values: an inf and a NaN in the prefix, each in one dim of one head, in a full page and in the last row of all
    at, last = c.prefix_refs[(prefix - 1) // 32] & P.REF_MASK, c.prefix_refs[(prefix - 1) // 16] & P.REF_MASK
    values = c.v.copy()
    values[at, 7, 0, 9], values[last, (prefix - 1) % 16, hk - 1, hd - 1] = -np.inf, np.nan
    c.v, c.dv = values, dev(values)
    ops.shared_prefix_attention(c.desc())
    engine.check_device_errors()
    got = host(c.out).astype(np.float64)
    want, absolute = c.want(values=np.where(np.isfinite(values), values, 0).astype(np.float16))
    bad = np.zeros(got.shape, dtype=bool)
    g = hq // hk
    bad[:, :, :g, 9] = bad[:, :, hq - g:, hd - 1] = True
    assert np.array_equal(~np.isfinite(got), bad)
    assert np.all(np.isneginf(got[:, :, :g, 9])) and np.all(np.isnan(got[:, :, hq - g:, hd - 1]))
    tol = 2.0 ** -11 * np.abs(want) + 1.5 * 2.0 ** -11 * absolute + (prefix + 40) * 6 * 2.0 ** -25
    assert np.all((np.abs(got - want) <= tol)[~bad])
    k = c.k.copy()  # a NaN in a key: every row of its head
    k[at, 7, 0, 5] = np.nan
    c.dk = dev(k)
    ops.shared_prefix_attention(c.desc())
    nan = np.zeros(got.shape, dtype=bool)
    nan[:, :, :g] = nan[:, :, hq - g:, hd - 1] = True
    assert np.array_equal(np.isnan(host(c.out)), nan)


@pytest.mark.parametrize("case,tile,parts", [
    ((2, 1, 8, 2, 128, 100), 16, False), ((1, 1, 8, 2, 64, 480), 16, False), ((2, 1, 8, 2, 64, 1500), 16, True),
    ((33, 1, 8, 2, 128, 1700), 128, True)], ids=["waves-128", "waves-64", "merged-pages", "merged-tiles"])
def test_infinities_whose_weight_is_below_fp32(ops, engine, case, tile, parts):
    """A token that every row sees, whose weight 2^-240 is 0 in fp32, holds an inf in one dim: that dim is not finite
    (0 times inf, as in any fp32 softmax), wherever the token and the one that takes all of the weight lie."""
    batch, queries, hq, hk, hd, prefix = case
    own = [queries + b % 5 for b in range(batch)]
    for heavy, far in ((3, 17), (3, prefix - 1), (prefix - 1, 3), (prefix - 1, prefix // 2)):
        c = Case(62, *case, own, stale=False)
        p = plan(c)
        assert (p.prefix_splits > 1) == parts and p.row_tile == tile
        at = lambda t: (c.prefix_refs[t // 16] & P.REF_MASK, t % 16)  # noqa: E731
        c.k[:] = 0
        c.q[..., 0] = 8.0
        c.k[at(heavy)][:, 0] = 240.0 / 8.0 / np.log2(np.e) * hd ** 0.5
        c.v[at(far)][:, 9] = np.inf
        c.dq, c.dk, c.dv = dev(c.q), dev(c.k), dev(c.v)
        ops.shared_prefix_attention(c.desc())
        engine.check_device_errors()
        got = host(c.out)
        bad = np.zeros(got.shape, dtype=bool)
        bad[..., 9] = True
        assert np.array_equal(~np.isfinite(got), bad), (heavy, far)
        want = np.broadcast_to(c.v[at(heavy)].repeat(hq // hk, axis=0), got.shape)
        # the other weights together are below prefix 2^-240
        assert np.array_equal(got[~bad], want[~bad]), (heavy, far)


def test_rising_scores_beside_many_rows(ops, engine):
    """Scores that rise along the prefix, by steps below and above what the running maximum lets pass (2^8), up to
    weights that span far more than f16 does."""
    batch, hq, hk, hd, prefix = 40, 8, 2, 128, 4100
    for slope in (0.01, 0.2, -0.2):
        c = Case(61, batch, 1, hq, hk, hd, prefix, [2] * batch, stale=False, qscale=0.5)
        c.q[..., 0] = 1.0
        t = np.arange(prefix)
        c.k[c.prefix_refs[t // 16] & P.REF_MASK, t % 16, :, 0] = (slope * t)[:, None].astype(np.float16)
        c.dq, c.dk = dev(c.q), dev(c.k)
        assert plan(c).row_tile == 128
        ops.shared_prefix_attention(c.desc(scale=1.0))
        # scores up to 820 + 12 6: fp32 sums off by 128 2^-24 900 = 0.007 in an exponent at most, 14 2^-11 in a weight
        want, absolute = c.want(scale=1.0)
        d = np.abs(host(c.out).astype(np.float64) - want)
        assert np.all(d <= 2.0 ** -11 * np.abs(want) + 30 * 2.0 ** -11 * absolute + prefix * 6 * 2.0 ** -25), slope
    engine.check_device_errors()


def test_nan_keys_make_nan_rows(ops):
    """A NaN in a key that a row sees makes the row NaN, whichever part it lies in; other rows and heads stay."""
    for where in ("prefix", "own"):
        c = Case(20, 2, 1, 8, 2, 128, 1500, [40, 17])
        k = c.k.copy()
        at = (c.prefix_refs[70] & P.REF_MASK) if where == "prefix" else c.refs[0, 1]
        k[at, 3, 1, 5] = np.nan
        c.dk = dev(k)
        ops.shared_prefix_attention(c.desc())
        got = host(c.out)
        nan = np.zeros(got.shape, dtype=bool)
        nan[(slice(None) if where == "prefix" else 0), :, 4:] = True
        assert np.array_equal(np.isnan(got), nan), where


def test_bad_refs_and_counts(ops, engine):
    from aether_nexus_amd.types import AW_E_OOB
    from aether_nexus_amd.weaver import WeaverError

    def error(word):
        with pytest.raises(WeaverError) as e:
            engine.check_device_errors()
        assert e.value.status == AW_E_OOB and word in str(e.value)
        engine.check_device_errors()

    c = Case(30, 3, 2, 8, 2, 128, 150, [20, 40, 3])
    c.prefix_refs[4] = c.blocks
    c.dprefix = dev(c.prefix_refs)
    ops.shared_prefix_attention(c.desc())
    error("hot block ref")
    c.check("bad prefix page")
    c = Case(31, 3, 2, 8, 2, 64, 150, [20, 40, 3])
    c.refs[1, 0] = 0x7FFFFFFE
    c.drefs = dev(c.refs)
    ops.shared_prefix_attention(c.desc())
    error("hot block ref")
    c.check("bad own page")
    c = Case(32, 2, 1, 8, 2, 64, 15, [32, 32])  # two pages each, all rows live
    ops.shared_prefix_attention(c.desc(seq_own=dev(np.array([33, 32]))))
    error("sequence length")
    c.check("count past the table")


@pytest.mark.parametrize("page", [5, 70, 93])
def test_bad_ref_beside_many_rows(ops, engine, page):
    """A bad ref anywhere in a long prefix that many rows read: reported, its tokens hidden, whatever page 0 holds."""
    from aether_nexus_amd.types import AW_E_OOB
    from aether_nexus_amd.weaver import WeaverError
    c = Case(33, 40, 1, 8, 2, 128, 2600, [3] * 40)
    c.prefix_refs[page] = c.blocks + 7
    for table in (c.prefix_refs, c.refs):  # no one's page 0: its stale rows, NaNs among them, are what a bad ref could show
        table[(table & P.REF_MASK) == 0] = c.blocks - 1
    c.k[0], c.v[0] = np.nan, np.inf
    c.k[c.blocks - 1], c.v[c.blocks - 1] = 0.5, 0.25
    c.dk, c.dv, c.drefs, c.dprefix = dev(c.k), dev(c.v), dev(c.refs), dev(c.prefix_refs)
    assert plan(c).row_tile == 128
    ops.shared_prefix_attention(c.desc())
    with pytest.raises(WeaverError) as e:
        engine.check_device_errors()
    assert e.value.status == AW_E_OOB and "hot block ref" in str(e.value)
    c.check(f"bad page {page}")


# batch, queries, q heads, kv heads, head_dim, prefix, own tokens, rows to a tile, least tokens of a part of (prefix, own)
LONG = [(20, 1, 2, 2, 64, 70001, [1] * 20, 128, (1024, 0)), (1, 2, 4, 1, 64, 300007, [2], 16, (4096, 0)),
        (2, 2, 2, 1, 64, 3, [300003, 40], 16, (0, 4096))]


@pytest.mark.parametrize("case", LONG, ids=["many-rows", "few-rows", "own"])
def test_parts_of_many_pages(ops, engine, case):
    """Parts longer than the 64 pages whose refs a wave holds at once: random scores; and equal ones, where every
    token counts once: the output's dim d is 60000 / n for the one token t[d] that holds 60000 there (60000 and the
    count n < 2^24 are sums that fp32 holds)."""
    *shape, tile, (least_prefix, least_own) = case
    c = Case(34, *shape)
    p = plan(c)
    assert p.row_tile == tile and p.prefix_tokens_per_split > least_prefix and p.own_tokens_per_split > least_own
    ops.shared_prefix_attention(c.desc())
    c.check("random scores")
    queries, hd, prefix = shape[1], shape[4], shape[5]
    c = Case(35, *shape, qscale=0.0, causal=False)
    c.v[:] = 0
    n = prefix + int(c.own[0])
    table = np.concatenate([(c.prefix_refs & P.REF_MASK)[t // 16:t // 16 + 1] * 16 + t % 16 if t < prefix else
                            c.refs[0, (t - prefix) // 16:(t - prefix) // 16 + 1] * 16 + (t - prefix) % 16
                            for t in np.linspace(0, n - 1, hd).astype(int)])
    c.v.reshape(-1, shape[3], hd)[table, :, np.arange(hd)] = 60000.0
    c.dv = dev(c.v)
    ops.shared_prefix_attention(c.desc())
    engine.check_device_errors()
    got = host(c.out).astype(np.float64)[0]
    want = 60000.0 / n
    assert np.all(np.abs(got - want) <= want * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25), (got.min(), got.max(), want)


@pytest.mark.parametrize("shape", LONG_PREFIXES, ids=["many-rows", "few-rows", "own"])
def test_no_page_of_a_long_prefix_is_lost(ops, engine, shape):
    """Scores of standard deviation 1 / 4 over the same long parts, so that every page counts: within bounds that a
    single page left out exceeds (test_the_bounds_of_long_prefixes_see_what_is_lost)."""
    c = Case(48, *shape, qscale=0.25)
    assert max(plan(c).prefix_tokens_per_split, plan(c).own_tokens_per_split) > 1024
    ops.shared_prefix_attention(c.desc())
    engine.check_device_errors()
    want, absolute = c.want()
    total = P.shared_prefix_weight_sums(c.q, c.k, c.prefix_refs, c.prefix, c.refs, c.own, c.shape[4] ** -0.5, c.causal)
    got = host(c.out)
    largest = float(np.abs(c.v[np.isfinite(c.v) & (np.abs(c.v) < 65504)]).max())
    worst, rel = prefix_errors(got, want, absolute, total, c.prefix + int(c.own.max()), largest)
    print(f"{shape[:6]}: worst error over tolerance {worst:.3f}, worst rel-L2 of a sequence {rel:.2e}", flush=True)
    assert np.isfinite(got).all() and worst <= 1.0 and rel <= PREFIX_REL_L2


@pytest.mark.parametrize("shape", [(2, 1100, 32, 8, 128, 300, [1400, 4096]), (1, 2600, 14, 2, 64, 1000, [2700])], ids=["two", "one"])
def test_many_queries(ops, engine, shape):
    """Prompt pieces behind a prefix, whose parts' sums are bounded: against float64 on the GPU, causal, over each
    sequence's tokens end to end."""
    import torch
    batch, queries, hq, hk, hd, prefix, own = shape
    c = Case(36, *shape, stale=False, spare=300)
    p = plan(c)
    assert p.own_tokens_per_split > 512 and p.workspace_bytes <= 133 << 20
    ops.shared_prefix_attention(c.desc())
    engine.check_device_errors()
    got, group = c.out.double(), hq // hk
    worst = 0.0
    for b in range(batch):
        at = torch.from_numpy(np.concatenate([c.prefix_refs & P.REF_MASK, c.refs[b, :-(-own[b] // 16)]])).cuda()
        n0 = -(-prefix // 16) * 16
        rows = torch.cat([torch.arange(prefix), n0 + torch.arange(own[b])]).cuda()
        last = prefix + own[b] - queries + torch.arange(queries, device="cuda:0").repeat_interleave(group)
        hidden = torch.arange(len(rows), device="cuda:0") > last[:, None]
        for g in range(hk):
            k, v = (x[at][:, :, g].flatten(0, 1)[rows].double() for x in (c.dk, c.dv))
            q = c.dq[b, :, g * group:(g + 1) * group].double().flatten(0, 1)
            s = (q @ k.t().contiguous() * hd ** -0.5).masked_fill(hidden, -float("inf"))
            w = (s - s.amax(1, keepdim=True)).exp()
            total = w.sum(1, keepdim=True)
            want, absolute = w @ v / total, w @ v.abs() / total
            # the head's tolerance, its subnormal weights over the row's sum of weights (its largest is 1)
            tol = 2.0 ** -11 * want.abs() + 1.5 * 2.0 ** -11 * absolute + len(rows) * 6.0 * 2.0 ** -25 / total + 2.0 ** -25
            d = (got[b, :, g * group:(g + 1) * group].flatten(0, 1) - want).abs()
            worst = max(worst, float((d / tol).max()))
    print(f"many queries: worst error over tolerance {worst:.3f}", flush=True)
    assert worst <= 1.0


def test_pages_past_32_bits(ops, engine):
    """Pages whose addresses lie more than 2^32 bytes into the pool, written by append_paged and read back."""
    import torch
    from aether_nexus_amd import ops as O
    hk, hd, blocks = 8, 128, 140000  # 4.6 GB
    pool = torch.empty(blocks, 16, hk, hd, dtype=torch.float16, device="cuda:0")
    assert pool.numel() * 2 > 2 ** 32
    for batch, prefix in ((1, 40), (40, 900)):  # read by few rows, and by many
        c = Case(37, batch, 1, 8, hk, hd, prefix, [5] * batch, stale=False)
        assert plan(c).row_tile == (128 if batch > 1 else 16)
        high = c.blocks
        rows = torch.arange(blocks - high, blocks, device="cuda:0")
        pool[rows] = 0
        x = dev(c.k.reshape(-1, hk, hd))
        ops.append_paged(O.make_append_desc(
            batch=1, num_tokens=high * 16, q_heads=0, kv_heads=hk, head_dim=hd, k=x, v=None, hot_k=pool, hot_v=None,
            refs=rows.to(torch.int32).view(1, -1), seq_hot=torch.tensor([high * 16], dtype=torch.int32, device="cuda:0")))
        engine.check_device_errors()
        assert torch.equal(pool[rows].view(torch.int16), c.dk.view(torch.int16).view(high, 16, hk, hd))
        up = lambda t: dev(np.where((t & P.REF_MASK) == P.REF_MASK, t, (t & P.REF_MASK) + blocks - high))  # noqa: E731
        ops.shared_prefix_attention(c.desc(hot_k=pool, hot_v=None, prefix_refs=up(c.prefix_refs), refs=up(c.refs)))
        engine.check_device_errors()
        c.check(f"high pages, {batch} sequences", values=c.k)


def test_results_do_not_depend_on_the_batch_order_or_run(ops):
    c = Case(40, 6, 2, 8, 2, 128, 700, [2, 30, 17, 90, 2, 5])
    ops.shared_prefix_attention(c.desc())
    first = host(c.out).copy()
    for _ in range(3):
        ops.shared_prefix_attention(c.desc())
        assert np.array_equal(host(c.out).view(np.int16), first.view(np.int16))


@pytest.mark.parametrize("growth", [3.0, 7.75])
@pytest.mark.parametrize("case", [(64, 1, 16, 4, 128, 8192), (40, 2, 12, 4, 64, 6000), (5, 1, 8, 2, 128, 1104)],
                         ids=["tiles-128", "tiles-64", "pages"])
def test_peaked_rows_beside_the_decode(ops, engine, case, growth):
    """Rows whose maximum grows in a later step, by a token that then takes most of the weight: every 64th token has
    2^0, one in the second half of the second step and one in the first half of the last 2^growth, the others 2^-14.
    The error against 64 bits is no larger than aw_decode_device's over the same tokens (its rounding of the weights
    is the reference: a row's largest is exactly 1); 5% for the two orders of sums, whose effect on the root mean
    square of thousands of values is below 1%."""
    import torch
    from aether_nexus_amd.weaver import make_desc
    batch, queries, hq, hk, hd, prefix = case
    c = Case(47, *case, [queries + b % 20 for b in range(batch)], stale=False)
    assert plan(c).row_tile == (128 if batch > 8 else 16)
    scores = np.full(prefix, -14.0)
    scores[::64] = 0.0
    for i, at in enumerate((64 + 45, 64 * (prefix // 64 - 1) + 10)):
        scores[at] = growth - 0.25 * i
    t, unit = np.arange(prefix), np.sqrt(hd) / (8.0 * np.log2(np.e))
    c.q[..., 0] = 8.0
    c.k[..., 1:] *= np.float16(0.01)
    c.k[..., 0] = -14.0 * unit
    c.k[c.prefix_refs[t // 16] & P.REF_MASK, t % 16, :, 0] = (scores * unit)[:, None].astype(np.float16)
    c.dq, c.dk = dev(c.q), dev(c.k)
    ops.shared_prefix_attention(c.desc())
    count = prefix // 16 + c.count  # the prefix fills its pages: a sequence's tokens are one table's
    table = np.concatenate([np.repeat(c.prefix_refs[None] & P.REF_MASK, batch, 0), np.where(c.refs < c.blocks, c.refs, 0)], axis=1)
    few = torch.empty_like(c.out)
    engine.decode_device(make_desc(layers=1, batch=batch, queries=queries, q_heads=hq, kv_heads=hk, head_dim=hd, dict_size=0,
                                   dict_heads=1, hot_count=count, cold_count=0, refs_stride=count, hot_blocks=c.blocks,
                                   cold_blocks=0, q=c.dq, out=few, hot_k=c.dk, hot_v=c.dv, refs=dev(table),
                                   seq_hot=dev(prefix + c.own), seq_hot_tokens=True, causal=True, scale=hd ** -0.5))
    engine.check_device_errors()
    want = P.shared_prefix_attention(c.q, c.k, c.v, c.prefix_refs, prefix, c.refs, c.own, hd ** -0.5, True)
    rel = [float(np.linalg.norm(host(x).astype(np.float64) - want) / np.linalg.norm(want)) for x in (c.out, few)]
    print(f"peaked rows {case} growth {growth}: rel-L2 {rel[0]:.3e}, decode {rel[1]:.3e}", flush=True)
    c.check("peaked rows")
    assert rel[0] <= 1.05 * rel[1], rel


@pytest.mark.parametrize("case", [(64, 1, 32, 8, 128, 2600), (33, 2, 32, 8, 64, 1500)], ids=["128", "64"])
def test_results_do_not_depend_on_the_neighbours(ops, case):
    """Rows of many sequences share a work-group's wave; each keeps its bits when the sequences change places, and when
    the others' queries change.  Scores of standard deviation 9: their maxima keep growing, by less and by more than 2^8,
    in other steps for each row."""
    batch, queries = case[:2]
    c = Case(46, *case, [queries + b % 40 for b in range(batch)], qscale=9.0)
    p = plan(c)
    assert p.row_tile == 128 and p.prefix_tokens_per_split > 2 * 64 and p.prefix_splits > 1
    ops.shared_prefix_attention(c.desc())
    first = host(c.out).view(np.int16).copy()
    assert np.isfinite(first.view(np.float16)).all()
    q, refs, own = c.q.copy(), c.refs.copy(), c.own.copy()
    for turn in range(3):
        order = c.rng.permutation(batch)
        c.dq, c.drefs, c.down = dev(q[order]), dev(refs[order]), dev(own[order])
        ops.shared_prefix_attention(c.desc())
        assert np.array_equal(host(c.out).view(np.int16), first[order]), f"order {turn}"
    c.drefs, c.down = dev(refs), dev(own)
    for keep in (0, batch // 2, batch - 1):
        other = (c.rng.standard_normal(q.shape) * 3.0).astype(np.float16)
        other[keep] = q[keep]
        c.dq = dev(other)
        ops.shared_prefix_attention(c.desc())
        assert np.array_equal(host(c.out)[keep].view(np.int16), first[keep]), f"sequence {keep}"


def test_another_stream_and_graph_replays(ops, engine):
    """Captured once, replayed while counts grow in device memory, with eager calls of another shape between:
    every replay gives the eager call's bits."""
    import torch
    c, other = Case(41, 3, 1, 8, 2, 128, 700, [20, 40, 3], spare=1), Case(42, 2, 3, 8, 2, 128, 300, [9, 3])
    down = c.down.clone()
    d, d2 = c.desc(seq_own=down), other.desc()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.shared_prefix_attention(d)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.shared_prefix_attention(d, stream=torch.cuda.current_stream().cuda_stream)
        for step, own in enumerate(([20, 40, 3], [19, 39, 2], [1, 1, 1], [20, 40, 3])):
            down.copy_(torch.tensor(own, dtype=torch.int32))
            ops.shared_prefix_attention(d)
            eager = c.out.clone()
            c.out.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(c.out.view(torch.int16), eager.view(torch.int16)), step
            c.own = np.array(own)
            c.check(f"replay {step}")
            ops.shared_prefix_attention(d2)
            _ = (other.out.float() * 2).sum()
            torch.cuda.synchronize()
    other.check("the other shape")
    engine.check_device_errors(s.cuda_stream)
    del g


def test_capture_refuses_workspace_growth():
    import torch
    from aether_nexus_amd.ops import OpsEngine
    from aether_nexus_amd.types import AW_E_UNSUPPORTED
    from aether_nexus_amd.weaver import WeaverError
    fresh = OpsEngine()
    try:
        c = Case(43, 2, 1, 8, 2, 64, 1000, [20, 3])
        d = c.desc()
        small = Case(45, 2, 1, 8, 2, 64, 100, [20, 3])  # in one part: no workspace
        d2 = small.desc()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with pytest.raises(WeaverError) as e:
                with torch.cuda.graph(g, stream=s):
                    fresh.shared_prefix_attention(d, stream=torch.cuda.current_stream().cuda_stream)
            assert e.value.status == AW_E_UNSUPPORTED and "eager" in str(e.value)
            del g
            torch.cuda.synchronize()
            assert np.isnan(host(c.out)).all()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                fresh.shared_prefix_attention(d2, stream=torch.cuda.current_stream().cuda_stream)
            for _ in range(2):
                small.out.fill_(float("nan"))
                g.replay()
                small.check("a small request captured at once")
            del g
            fresh.shared_prefix_attention(d)
        c.check("after the refusal")
    finally:
        torch.cuda.synchronize()
        fresh.close()


def test_a_decode_loop_of_all_of_them(ops, engine):
    """Three steps of four conversations behind one instruction: head norms and rotation on the way into the pages
    (the prefix first, then each conversation's tokens), then attention; against float64 over the tokens end to end."""
    import torch
    from aether_nexus_amd import ops as O
    rng = np.random.default_rng(44)
    batch, hq, hk, hd, prefix, count = 4, 8, 2, 128, 43, 4
    rotary = O.Rotary(hd, 10000.0, scaling="parts", factor=4.0, original_length=2048.0)
    f = rotary.inv_freq.cpu().numpy()
    wq, wk = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    blocks = 3 + batch * count
    pool_k, pool_v = (torch.full((blocks, 16, hk, hd), float("nan"), dtype=torch.float16, device="cuda:0") for _ in range(2))
    order = rng.permutation(blocks)
    prefix_refs, refs = dev(order[:3]), dev(order[3:].reshape(batch, count))
    keys, values = [[] for _ in range(batch + 1)], [[] for _ in range(batch + 1)]

    def feed(new, held, table, seqs, start):
        """New rows of the sequences through append_paged; returns their turned q."""
        x = (rng.standard_normal((sum(new), hq + 2 * hk, hd)) * 1.5).astype(np.float16)
        d = dev(x)
        q_out = torch.empty(sum(new), hq, hd, dtype=torch.float16, device="cuda:0")
        ops.append_paged(O.make_append_desc(
            batch=len(new), num_tokens=sum(new), q_heads=hq, kv_heads=hk, head_dim=hd, q=d[:, :hq], q_out=q_out, k=d[:, hq:hq + hk],
            v=d[:, hq + hk:], hot_k=pool_k, hot_v=pool_v, refs=table, seq_hot=dev(np.array(held) + np.array(new)),
            token_offsets=dev(np.concatenate([[0], np.cumsum(new)])), rotary=rotary, q_norm=dev(wq), k_norm=dev(wk),
            start_position=start))
        at = 0
        for i, n, h in zip(seqs, new, held):
            pos = start + h + np.arange(n)
            k = P.rotary(P.head_norm(x[at:at + n, hq:hq + hk], wk, 1e-5), pos, f)
            keys[i].append(k.astype(np.float16).astype(np.float64))
            values[i].append(x[at:at + n, hq + hk:].astype(np.float64))
            at += n
        return q_out
    feed([prefix], [0], prefix_refs.view(1, 3), [batch], 0)
    held = [0] * batch
    for queries in (20, 1, 3):
        q = feed([queries] * batch, held, refs, range(batch), prefix)
        held = [h + queries for h in held]
        out = torch.empty(batch, queries, hq, hd, dtype=torch.float16, device="cuda:0")
        ops.shared_prefix_attention(O.make_prefix_desc(
            batch=batch, queries=queries, q_heads=hq, kv_heads=hk, head_dim=hd, prefix_tokens=prefix, q=q.view_as(out), out=out,
            hot_k=pool_k, hot_v=pool_v, prefix_refs=prefix_refs, own_count=count, refs=refs, seq_own=dev(np.array(held))))
        engine.check_device_errors()
        got, qs = host(out).astype(np.float64), host(q).astype(np.float64).reshape(batch, queries, hq, hd)
        for b in range(batch):
            k, v = (np.concatenate(x[batch] + x[b]) for x in (keys, values))
            for i in range(queries):
                n = prefix + held[b] - queries + 1 + i
                for h in range(hq):
                    s = k[:n, h // 4] @ qs[b, i, h] * hd ** -0.5
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    want, a = w @ v[:n, h // 4], w @ np.abs(v[:n, h // 4])
                    # besides the kernel's own errors, the oracle's keys are rounded to f16 from 64 bits and may differ by a
                    # step from the kernel's: 2^-10 of each product, in weights and sum
                    grow = 2 * 2.0 ** -10 * np.abs(k[:n, h // 4] * qs[b, i, h]).sum(1).max() * hd ** -0.5
                    assert np.all(np.abs(got[b, i, h] - want) <= 2.0 ** -11 * np.abs(want) + (1.5 * 2.0 ** -11 + grow) * a + 2.0 ** -20)
