"""Rotary positions, head norms and paged appends on cuda:0 through the C ABI against
the float64 oracle (oracle/paged_oracle.py).

Tolerance of a value y of pair (x0, x1): half a step of the f16 store (2^-11 |y|, or
2^-25 among the subnormals), and fp32 roundings on the way, 2^-24 of what they round:
the products and their sum 3, cosine and sine 5 (their own 2, the angle's 2 pi 2^-25 of
a turn, the magnitude), the norm 22 (the sum of at most 1024 squares: 16 in a lane and 6
joins; mean, root, division, two products) -- 32 (|x0| + |x1|) 2^-24 m covers them all."""
from __future__ import annotations

import numpy as np
import pytest

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
    return torch.from_numpy(a.astype(np.int32)).cuda() if a.dtype != np.float64 else torch.from_numpy(a).cuda()


def bits(t):
    import torch
    torch.cuda.synchronize()
    return t.contiguous().cpu().view(torch.int16).numpy()


def host(t):
    return bits(t).view(np.float16)


def f16(rng, *shape, scale=1.5):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


def close(got, want, scale, what):
    got, tol = got.astype(np.float64), 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 32 * 2.0 ** -24 * scale
    d = np.abs(got - want)
    print(f"{what}: worst error over tolerance {float((d / tol).max()) if d.size else 0:.3f}", flush=True)
    assert np.isfinite(got).all() and np.all(d <= tol), what


def turned(x, positions, r, norm=None, eps=1e-5):
    """(value, scale) of rows in float64."""
    x = np.asarray(x, dtype=np.float64) if norm is None else P.head_norm(x, norm, eps)
    f = r.inv_freq.cpu().numpy()
    return (P.rotary(x, positions, f, r.interleaved, r.magnitude),
            max(1.0, abs(r.magnitude)) * P.rotary_scale(x, r.rotary_dim, r.interleaved))


def token_rows(rng, kind, tokens, hq, hk, hd):
    """(rows, q, k, v views of them on the GPU, the same on the host): 'plain' contiguous, 'fused' views of
    [tokens][hq + 2 hk][hd], 'odd' views of rows with one value between them, 2 bytes off 16-byte alignment."""
    import torch
    if kind == "plain":
        h = [f16(rng, tokens, n, hd) for n in (hq, hk, hk)]
        return [dev(x) for x in h], h
    heads = hq + 2 * hk
    if kind == "fused":
        x = f16(rng, tokens, heads, hd)
        d = dev(x)
        cut = [slice(0, hq), slice(hq, hq + hk), slice(hq + hk, heads)]
        return [d[:, c] for c in cut], [x[:, c] for c in cut]
    x = f16(rng, tokens, heads * hd + 1)
    d = torch.zeros(x.size + 1, dtype=torch.float16, device="cuda:0")
    d[1:] = dev(x).flatten()
    d = d[1:].view(tokens, heads * hd + 1)
    cut = [(0, hq), (hq, hk), (hq + hk, hk)]
    return ([d[:, a * hd:(a + n) * hd] for a, n in cut],
            [np.ascontiguousarray(x[:, a * hd:(a + n) * hd]).reshape(tokens, n, hd) for a, n in cut])


# (tokens, q heads, kv heads, head_dim, rotary_dim)
SHAPES = [(1, 14, 2, 64, 64), (1, 32, 8, 128, 128), (3, 32, 8, 128, 64), (16, 4, 4, 80, 20), (37, 12, 2, 128, 128),
          (5, 1, 0, 128, 32), (5, 0, 3, 64, 48), (7, 3, 2, 6, 6), (2, 5, 1, 256, 256), (4, 2, 2, 1024, 1024), (9, 7, 1, 96, 96),
          (6, 3, 1, 112, 62), (130, 8, 2, 192, 128), (11, 2, 1, 2, 2), (3, 2, 2, 48, 16), (700, 5, 3, 32, 32), (8, 2, 1, 512, 96)]


# Fewer than 16 turned dims, 1 to 7 passing ones, both, heads of fewer than 16
SHAPES += [(300, 5, 3, 64, 2), (9, 4, 2, 128, 14), (5, 3, 1, 16, 8), (6, 3, 1, 16, 2), (7, 2, 2, 17, 12), (3, 2, 1, 23, 6), (4, 2, 2, 24, 10),
           (9, 3, 2, 65, 64), (5, 32, 8, 128, 122), (8, 2, 1, 67, 60), (3, 2, 1, 17, 16), (2, 3, 2, 15, 14), (4, 1, 1, 12, 4), (3, 2, 2, 39, 32),
           (2, 2, 1, 1023, 4), (2, 1, 2, 1024, 1018), (2, 2, 1, 1024, 1000), (2, 2, 1, 1023, 1010), (2, 2, 1, 1024, 1008)]


@pytest.mark.parametrize("rows", ["plain", "fused", "odd"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True], ids=["rotary", "norm"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_rows(ops, shape, norm, interleaved, rows):
    import torch
    from aether_nexus_amd import ops as O
    tokens, hq, hk, hd, n = shape
    rng = np.random.default_rng(sum(shape) + 7 * norm)
    (q, k, _), (hq_, hk_, _) = token_rows(rng, rows, tokens, hq, hk, hd)
    r = O.Rotary(n, 10000.0, interleaved=interleaved, magnitude=1.25)
    w = [f16(rng, hd, scale=1.0) for _ in range(2)] if norm else [None, None]
    start = 4097
    out = [torch.full((tokens, h, hd), 7.0, dtype=torch.float16, device="cuda:0") for h in (hq, hk)]
    d = O.make_rotary_desc(num_tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=hd, rotary=r, q=q, k=k, q_out=out[0],
                           k_out=out[1], start_position=start, q_norm=dev(w[0]) if norm else None,
                           k_norm=dev(w[1]) if norm else None)
    call = ops.qk_norm_rotary if norm else ops.rotary
    call(d)
    positions = start + np.arange(tokens)
    for got, x, wt, what in ((out[0], hq_, w[0], "q"), (out[1], hk_, w[1], "k")):
        close(host(got), *turned(x, positions, r, wt), f"{what} {shape} {rows}")
    assert np.array_equal(host(q).reshape(tokens, hq, hd).view(np.int16), np.ascontiguousarray(hq_).view(np.int16))
    # in place: the same bits, and nothing between the rows changes
    before = [bits(o) for o in out]
    d = O.make_rotary_desc(num_tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=hd, rotary=r, q=q, k=k,
                           start_position=start, q_norm=dev(w[0]) if norm else None, k_norm=dev(w[1]) if norm else None)
    call(d)
    assert np.array_equal(bits(q).reshape(before[0].shape), before[0])
    assert np.array_equal(bits(k).reshape(before[1].shape), before[1])


@pytest.mark.parametrize("tokens", [1 << 20, (1 << 20) + 1, 1 << 24])
def test_as_many_tokens_as_a_call_takes(ops, engine, tokens):
    """Heads of 2 dims, a work-group a token: more of them than one row of a grid takes, up to the most that is
    accepted; turned alone, and into pages in the opposite order."""
    import torch
    from aether_nexus_amd import ops as O
    rng = np.random.default_rng(3)
    x = f16(rng, tokens, 1, 2)
    r = O.Rotary(2, 10000.0)
    q, out = dev(x), torch.full((tokens, 1, 2), 7.0, dtype=torch.float16, device="cuda:0")
    ops.rotary(O.make_rotary_desc(num_tokens=tokens, q_heads=1, kv_heads=0, head_dim=2, rotary=r, q=q, q_out=out, k=None))
    want = turned(x, np.arange(tokens), r)
    close(host(out), *want, f"{tokens} tokens")
    pages = -(-tokens // 16)
    pool = torch.full((pages, 16, 1, 2), 7.0, dtype=torch.float16, device="cuda:0")
    refs = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda:0").view(1, pages)
    ops.append_paged(O.make_append_desc(batch=1, num_tokens=tokens, q_heads=0, kv_heads=1, head_dim=2, rotary=r, k=q, v=None,
                                        hot_k=pool, hot_v=None, refs=refs,
                                        seq_hot=torch.tensor([tokens], dtype=torch.int32, device="cuda:0")))
    engine.check_device_errors()
    assert np.array_equal(bits(pool)[::-1].reshape(-1, 1, 2)[:tokens], bits(out))


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("hd,n", [(64, 2), (16, 14), (23, 6), (65, 64), (128, 122), (128, 32), (12, 4)])
def test_passing_dims_keep_their_bits(ops, hd, n, interleaved):
    """Infinities and NaNs of any payload in dims that pass, none of which reach the turned ones."""
    import torch
    from aether_nexus_amd import ops as O
    rng = np.random.default_rng(hd + n)
    x = f16(rng, 5, 3, hd)
    x[..., n:] = rng.choice(np.array([0x7C00, 0xFC00, 0x7E00, 0x7D01, 0xFC05, 0x0001, 0x8000], dtype=np.uint16), x[..., n:].shape).view(np.float16)
    q, r = dev(x), O.Rotary(n, 10000.0, interleaved=interleaved)
    out = torch.zeros_like(q)
    ops.rotary(O.make_rotary_desc(num_tokens=5, q_heads=3, kv_heads=0, head_dim=hd, rotary=r, q=q, k=None, q_out=out, start_position=9))
    got = host(out).reshape(5, 3, hd)
    assert np.array_equal(got[..., n:].view(np.uint16), x[..., n:].view(np.uint16))
    want, scale = turned(np.where(np.arange(hd) < n, x, 0).astype(np.float16), 9 + np.arange(5), r, None)
    close(got[..., :n], want[..., :n], scale[..., :n], f"{hd} {n}")


def test_positions_of_their_own(ops):
    """Far, repeated, descending positions, the largest 32-bit one among them, one token per position and heads of zeros."""
    import torch
    from aether_nexus_amd import ops as O
    rng = np.random.default_rng(5)
    positions = np.array([0, 1, 131071, 131071, 5, 1 << 20, (1 << 31) + 12345, (1 << 32) - 1], dtype=np.uint32)
    x = f16(rng, 8, 3, 64)
    x[4] = 0
    for scaling in ({}, dict(scaling="linear", factor=7.5), dict(scaling="ntk", factor=8.0),
                    dict(scaling="parts", factor=16.0, original_length=8192.0, magnitude=1.27)):
        r = O.Rotary(64, 500000.0, **scaling)
        q, out = dev(x), torch.empty(8, 3, 64, dtype=torch.float16, device="cuda:0")
        d = O.make_rotary_desc(num_tokens=8, q_heads=3, kv_heads=0, head_dim=64, rotary=r, q=q, k=None, q_out=out,
                               positions=dev(positions.view(np.int32)))
        ops.rotary(d)
        close(host(out), *turned(x, positions, r), f"positions {scaling}")
        assert not host(out)[4].any()


def test_infinities_stay_in_their_pairs(ops):
    import torch
    from aether_nexus_amd import ops as O
    x = np.ones((2, 2, 64), dtype=np.float16)
    x[0, 1, 3], x[1, 0, 40] = np.inf, np.nan
    for interleaved in (False, True):
        r = O.Rotary(64, 10000.0, interleaved=interleaved)
        q = dev(x)
        ops.rotary(O.make_rotary_desc(num_tokens=2, q_heads=2, kv_heads=0, head_dim=64, rotary=r, q=q, k=None, start_position=1))
        bad = ~np.isfinite(host(q))
        want = np.zeros_like(bad)
        for t, h, i in ((0, 1, 3), (1, 0, 40)):
            want[t, h, [i, i ^ 1] if interleaved else [i, (i + 32) % 64]] = True
        assert np.array_equal(bad, want)


def test_norms_alone_and_small_heads(ops):
    import torch
    from aether_nexus_amd import ops as O
    rng = np.random.default_rng(6)
    for hd in (64, 7, 1):
        x, w = f16(rng, 9, 4, hd), f16(rng, hd, scale=1.0)
        x[3] = 0
        x[5] *= np.float16(2.0 ** -14)
        out = torch.empty(9, 4, hd, dtype=torch.float16, device="cuda:0")
        ops.qk_norm_rotary(O.make_rotary_desc(num_tokens=9, q_heads=0, kv_heads=4, head_dim=hd, rotary=None, q=None, k=dev(x),
                                              k_out=out, k_norm=dev(w), eps=1e-6))
        want = P.head_norm(x, w, 1e-6)
        close(host(out), want, np.abs(want), f"norm {hd}")
        assert not host(out)[3].any()


def test_zero_counts_and_refusals(ops):
    import torch
    from aether_nexus_amd import ops as O
    from aether_nexus_amd.types import AW_E_INVALID_ARG
    from aether_nexus_amd.weaver import WeaverError
    r = O.Rotary(64, 10000.0)
    x = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda:0")
    common = dict(head_dim=64, rotary=r, k=None, kv_heads=0)
    ops.rotary(O.make_rotary_desc(num_tokens=0, q_heads=2, q=x, **common))
    ops.rotary(O.make_rotary_desc(num_tokens=3, q_heads=0, q=None, **common))
    assert bool((x == 1).all())
    bad = [dict(num_tokens=4, q_heads=2, q=x), dict(num_tokens=3, q_heads=2, q=x.float()),
           dict(num_tokens=3, q_heads=2, q=x.transpose(1, 2)), dict(num_tokens=3, q_heads=2, q=x[:1].expand(3, 2, 64)),
           dict(num_tokens=3, q_heads=2, q=x, positions=torch.zeros(2, dtype=torch.int32, device="cuda:0")),
           dict(num_tokens=3, q_heads=2, q=x, positions=torch.zeros(3, device="cuda:0"))]
    for kw in bad:
        with pytest.raises(WeaverError) as e:
            O.make_rotary_desc(**{**common, **kw})
        assert e.value.status == AW_E_INVALID_ARG, kw
    d = O.make_rotary_desc(num_tokens=3, q_heads=2, q=x, **common)
    with pytest.raises(WeaverError):
        ops.qk_norm_rotary(d)  # no weights
    d._device = 1
    with pytest.raises(WeaverError) as e:
        ops.rotary(d)
    assert "GPU 1" in str(e.value)
    assert bool((x == 1).all())


# ---------------------------------------------------------------- appends


class Batch:
    """A ragged batch and its pages: lengths after the append, new tokens, padded rows behind them."""

    def __init__(self, seed, held, new, hq, hk, hd, *, rows="plain", pad=0, values=True, offsets=True):
        self.rng = rng = np.random.default_rng(seed)
        self.batch, self.hq, self.hk, self.hd = len(new), hq, hk, hd
        self.tokens = sum(new) + pad
        self.seq = np.array([h + n for h, n in zip(held, new)])
        self.offsets = np.concatenate([[0], np.cumsum(new)]) if offsets else None
        (self.q, self.k, self.v), (self.hq_, self.hk_, self.hv_) = token_rows(rng, rows, self.tokens, hq, hk, hd)
        pages = [-(-int(n) // 16) for n in self.seq]
        self.blocks = sum(pages) + 2
        order = rng.permutation(self.blocks)
        self.count = max(max(pages), 1)
        self.refs = np.full((self.batch, self.count + 1), 0x7FFFFFFF, dtype=np.int64)
        at = 0
        for b, n in enumerate(pages):
            self.refs[b, :n] = order[at:at + n]
            at += n
        self.refs[:, ::2] |= 1 << 31  # bit 31 is masked
        self.pool_k, self.pool_v = f16(rng, self.blocks, 16, hk, hd), f16(rng, self.blocks, 16, hk, hd)
        self.dk, self.dv = dev(self.pool_k), dev(self.pool_v) if values else None
        self.q_out = f16(rng, self.tokens, hq, hd)
        self.dq = dev(self.q_out)

    def desc(self, rotary, **kw):
        from aether_nexus_amd import ops as O
        base = dict(batch=self.batch, num_tokens=self.tokens, q_heads=self.hq, kv_heads=self.hk, head_dim=self.hd, k=self.k,
                    v=self.v if self.dv is not None else None, hot_k=self.dk, hot_v=self.dv,
                    refs=dev(self.refs.astype(np.uint32).view(np.int32)), hot_count=self.count, seq_hot=dev(self.seq),
                    token_offsets=None if self.offsets is None else dev(self.offsets), rotary=rotary,
                    q=self.q if self.hq else None, q_out=self.dq if self.hq else None)
        return O.make_append_desc(**{**base, **kw})

    def check(self, rotary, what, start=0, positions=None, q_norm=None, k_norm=None, seq=None, refs=None, offsets=None):
        """Every value of q_out and of the pools, those that the call leaves alone to the bit."""
        offsets = self.offsets if offsets is None else offsets
        s, place, row = P.places(self.tokens, self.batch, self.seq if seq is None else seq, offsets,
                                 self.refs if refs is None else refs, self.count, self.blocks)
        positions = place + start if positions is None else positions

        def made(x, norm):
            if rotary is not None:
                return turned(x, positions, rotary, norm)
            y = np.asarray(x, dtype=np.float64) if norm is None else P.head_norm(x, norm, 1e-5)
            return y, np.abs(y)
        if self.hq:
            got, (want, scale) = host(self.dq), made(self.hq_, q_norm)
            close(got[s >= 0], want[s >= 0], scale[s >= 0], what + " q")
            assert np.array_equal(got[s < 0].view(np.int16), self.q_out[s < 0].view(np.int16)), "padded q rows"
        want, scale = made(self.hk_, k_norm)
        got, pool = host(self.dk).reshape(-1, self.hk, self.hd), self.pool_k.reshape(-1, self.hk, self.hd)
        w = row >= 0
        close(got[row[w]], want[w], scale[w], what + " k")
        rest = np.setdiff1d(np.arange(len(pool)), row[w])
        assert np.array_equal(got[rest].view(np.int16), pool[rest].view(np.int16)), "other rows of the k pool"
        if self.dv is not None:
            pool = self.pool_v.reshape(-1, self.hk, self.hd).copy()
            pool[row[w]] = self.hv_[w]
            assert np.array_equal(bits(self.dv).reshape(pool.shape), pool.view(np.int16)), "v pool"


APPENDS = [  # held, new
    ([0], [1]), ([15], [1]), ([16], [1]), ([0, 31, 700], [1, 1, 1]), ([5, 0, 40, 15], [3, 0, 17, 2]), ([0, 0], [0, 33]),
    ([100], [530]), ([3] * 70, [1] * 70), ([7] * 131, [i % 3 for i in range(131)]),
]


@pytest.mark.parametrize("rows", ["plain", "fused", "odd"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (3, 1, 80), (0, 2, 64)], ids=str)
@pytest.mark.parametrize("held,new", APPENDS, ids=[f"{len(n)}x{sum(n)}" for _, n in APPENDS])
def test_append(ops, engine, held, new, heads, rows):
    from aether_nexus_amd import ops as O
    b = Batch(len(new) + sum(new), held, new, *heads, rows=rows, pad=len(new) % 3)
    r = O.Rotary(heads[2] - 16, 10000.0, interleaved=len(new) % 2 == 1)
    ops.append_paged(b.desc(r, start_position=11))
    engine.check_device_errors()
    b.check(r, f"append {len(new)} sequences", start=11)


def test_no_tokens(ops, engine):
    """Empty tensors, whose address is null: nothing happens."""
    import torch
    from aether_nexus_amd import ops as O
    q, k = (torch.empty(0, h, 64, dtype=torch.float16, device="cuda:0") for h in (4, 2))
    pool = torch.full((3, 16, 2, 64), 5.0, dtype=torch.float16, device="cuda:0")
    r = O.Rotary(64)
    ops.rotary(O.make_rotary_desc(num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, rotary=r, q=q, k=k))
    for batch in (0, 2):
        ops.append_paged(O.make_append_desc(
            batch=batch, num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, q=q, k=k, v=k, hot_k=pool, hot_v=pool.clone(), rotary=r,
            refs=torch.zeros(batch, 3, dtype=torch.int32, device="cuda:0"), seq_hot=torch.zeros(batch, dtype=torch.int32, device="cuda:0")))
    engine.check_device_errors()
    assert bool((pool == 5).all())


@pytest.mark.parametrize("norms", ["none", "k", "both"])
@pytest.mark.parametrize("hd,n", [(64, 10), (128, 2), (72, 66), (31, 30), (33, 14), (13, 6)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_append_of_few_turned_or_passing_dims(ops, engine, hd, n, norms, interleaved):
    from aether_nexus_amd import ops as O
    b = Batch(hd + n, [5, 0, 40, 15], [3, 0, 17, 2], 6, 3, hd, rows="fused", pad=1)
    r = O.Rotary(n, 10000.0, interleaved=interleaved)
    qw, kw = f16(b.rng, hd, scale=1.0) if norms == "both" else None, f16(b.rng, hd, scale=1.0) if norms != "none" else None
    ops.append_paged(b.desc(r, start_position=3, q_norm=None if qw is None else dev(qw), k_norm=None if kw is None else dev(kw)))
    engine.check_device_errors()
    b.check(r, f"append {hd} {n} {norms}", start=3, q_norm=qw, k_norm=kw)


def test_append_forms(ops, engine):
    """Equal shares without offsets, positions of their own, norms, no rotation, keys that are the values too."""
    from aether_nexus_amd import ops as O
    r = O.Rotary(64, 10000.0)
    b = Batch(1, [3, 20, 0], [4, 4, 4], 4, 2, 64, offsets=False)
    ops.append_paged(b.desc(r))
    b.check(r, "equal shares")
    b = Batch(2, [3, 20], [5, 2], 4, 2, 64)
    positions = np.array([9, 8, 7, 100000, 3, 2, 1])
    ops.append_paged(b.desc(r, positions=dev(positions), start_position=55))
    b.check(r, "positions", positions=positions)
    b = Batch(3, [3, 20], [5, 2], 4, 2, 64)
    wq, wk = f16(b.rng, 64), f16(b.rng, 64)
    ops.append_paged(b.desc(r, q_norm=dev(wq), k_norm=dev(wk)))
    b.check(r, "both norms", q_norm=wq, k_norm=wk)
    b = Batch(4, [3, 20], [5, 2], 4, 2, 64)
    ops.append_paged(b.desc(r, k_norm=dev(wk)))
    b.check(r, "the keys' norm", k_norm=wk)
    b = Batch(5, [3, 20], [5, 2], 4, 2, 64, pad=2)
    ops.append_paged(b.desc(None))
    b.check(None, "no rotation")
    b = Batch(6, [3, 20], [5, 2], 4, 2, 64, values=False)
    ops.append_paged(b.desc(r))
    b.check(r, "one pool")
    b = Batch(7, [3, 20], [5, 2], 4, 2, 64)  # q in place
    ops.append_paged(b.desc(r, q_out=None))
    b.dq = b.q
    b.check(r, "q in place")
    engine.check_device_errors()


@pytest.mark.parametrize("batch", [64, 65, 128, 4096, 4097, 5000, 70000])
def test_append_of_many_sequences(ops, engine, batch):
    """Each token finds its sequence among any number of them: sequences without new tokens wherever a search of 64
    stretches at a time cuts the batch, at both ends, and in runs longer than a stretch; rows behind the last one."""
    from aether_nexus_amd import ops as O
    r = O.Rotary(16, 10000.0)
    rng = np.random.default_rng(batch)
    new, held = rng.integers(0, 3, batch), rng.integers(0, 20, batch)
    n = batch
    while n > 1:
        stretch = -(-n // 64)
        for cut in range(0, batch, stretch if stretch > 1 else 7):
            new[cut:cut + 2] = 0
        n = stretch
    new[batch // 3:batch // 3 + batch // 50 + 2] = new[-3:] = 0
    new[batch // 2] = 40
    assert 0 < np.count_nonzero(new) < batch
    b = Batch(9, held.tolist(), new.tolist(), 1, 1, 16, pad=3)
    ops.append_paged(b.desc(r))
    engine.check_device_errors()
    b.check(r, f"{batch} sequences")


def test_append_bad_pages_and_lengths(ops, engine):
    """A ref past the pool, a page past the table, a sequence with more new tokens than it has, offsets that
    descend: the tokens are left out as described, everything else is written, and the error is reported."""
    from aether_nexus_amd import ops as O
    from aether_nexus_amd.types import AW_E_OOB
    from aether_nexus_amd.weaver import WeaverError
    r = O.Rotary(64, 10000.0)

    def run(word, change, **kw):
        b = Batch(8, [3, 20, 30], [5, 14, 4], 4, 2, 64, pad=1)
        change(b)
        ops.append_paged(b.desc(r, **kw))
        with pytest.raises(WeaverError) as e:
            engine.check_device_errors()
        assert e.value.status == AW_E_OOB and word in str(e.value), str(e.value)
        engine.check_device_errors()  # cleared
        return b

    def bad_ref(b):
        b.refs[1, 1] = b.blocks
    run("hot block ref", bad_ref).check(r, "ref past the pool")

    def short_table(b):
        b.count = 2
    run("hot block ref", short_table).check(r, "page past the table")

    def too_short(b):
        b.seq[0] = 4
    run("sequence length", too_short).check(r, "more new tokens than the sequence has")

    def empty(b):
        b.seq[2] = 0
    run("sequence length", empty).check(r, "a sequence of no tokens")

    def descending(b):
        b.offsets = np.array([0, 19, 5, 23])
    b = Batch(8, [3, 20, 30], [5, 14, 4], 4, 2, 64, pad=1)
    descending(b)
    ops.append_paged(b.desc(r))  # which rows are left out is not said: nothing out of range is touched
    with pytest.raises(WeaverError) as e:
        engine.check_device_errors()
    assert "sequence length" in str(e.value)


def test_append_graph_replays(ops, engine):
    """Captured once, replayed as the lengths grow in device memory, with eager work between: each replay's pools
    are those of eager calls."""
    import torch
    from aether_nexus_amd import ops as O
    r = O.Rotary(64, 10000.0)
    a, e = (Batch(9, [24, 0, 33], [1, 1, 1], 4, 2, 64) for _ in range(2))  # pages for what they grow to
    a.seq = e.seq = np.array([15, 1, 34])
    seq_a, seq_e = dev(a.seq), dev(e.seq)
    da, de = a.desc(r, seq_hot=seq_a), e.desc(r, seq_hot=seq_e)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.append_paged(da)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.append_paged(da, stream=torch.cuda.current_stream().cuda_stream)
        for step in range(4):
            x = torch.randn_like(a.k)
            a.k.copy_(x)
            e.k.copy_(x)
            g.replay()
            ops.append_paged(de)
            _ = x.sum()
            torch.cuda.synchronize()
            assert torch.equal(a.dk.view(torch.int16), e.dk.view(torch.int16)), step
            assert torch.equal(a.dq.view(torch.int16), e.dq.view(torch.int16)), step
            seq_a += torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda:0")
            seq_e += torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda:0")
    engine.check_device_errors(s.cuda_stream)
    del g


def test_append_then_decode(ops, engine):
    """The table and counts of an append serve the decode behind it: three steps of a batch equal attention over
    the rows laid end to end."""
    import torch
    from aether_nexus_amd import ops as O
    from aether_nexus_amd.weaver import make_desc
    from oracle.attention_oracle import multihead_attention_f64
    from helpers import assert_close
    rng = np.random.default_rng(10)
    hq, hk, hd, batch, count = 8, 2, 64, 3, 3
    r = O.Rotary(hd, 10000.0)
    f = r.inv_freq.cpu().numpy()
    pool_k, pool_v = (torch.full((batch * count, 16, hk, hd), float("nan"), dtype=torch.float16, device="cuda:0") for _ in range(2))
    refs = dev(rng.permutation(batch * count).reshape(batch, count))
    held = np.zeros(batch, dtype=np.int64)
    keys, values = [np.zeros((0, hk, hd)) for _ in range(batch)], [np.zeros((0, hk, hd)) for _ in range(batch)]
    for new in ([17, 1, 30], [1, 1, 1], [14, 16, 1]):
        b = Batch(int(held.sum()) + 11, held, new, hq, hk, hd, rows="fused")
        held = held + new
        seq = dev(held)
        d = b.desc(r, hot_k=pool_k, hot_v=pool_v, refs=refs, hot_count=count, seq_hot=seq)
        ops.append_paged(d)
        _, place, _ = P.places(b.tokens, batch, held, b.offsets, refs.cpu().numpy(), count, batch * count)
        for i in range(batch):
            rows = slice(b.offsets[i], b.offsets[i + 1])
            keys[i] = np.concatenate([keys[i], P.rotary(b.hk_[rows], place[rows], f).astype(np.float16).astype(np.float64)])
            values[i] = np.concatenate([values[i], b.hv_[rows].astype(np.float64)])
        # the newest token of each sequence
        last = torch.tensor([b.offsets[i + 1] - 1 for i in range(batch)], device="cuda:0")
        q = b.dq[last].contiguous()
        out = torch.empty_like(q)
        engine.decode_device(make_desc(layers=1, batch=batch, queries=1, q_heads=hq, kv_heads=hk, head_dim=hd, dict_size=0,
                                       dict_heads=1, hot_count=count, cold_count=0, refs_stride=count, hot_blocks=batch * count,
                                       cold_blocks=0, q=q, out=out, hot_k=pool_k, hot_v=pool_v, refs=refs, seq_hot=seq,
                                       seq_hot_tokens=True, scale=hd ** -0.5))
        engine.check_device_errors()
        hq_rows, got = host(q), host(out)
        for i in range(batch):
            want = multihead_attention_f64(hq_rows[i:i + 1], keys[i], values[i], int(held[i]), 1)
            assert_close(got[i], want[0], f"sequence {i} of {held[i]} tokens")
