"""The float64 oracle of the operators around a batch over pages, against other forms of the same mathematics."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import LONG_PREFIXES, PREFIX_REL_L2, prefix_errors
from oracle import paged_oracle as P


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,n", [(8, 8), (12, 6), (6, 2)])
def test_rotary_is_a_complex_multiplication(interleaved, hd, n):
    rng = np.random.default_rng(hd * 10 + n)
    x = rng.standard_normal((5, 3, hd))
    positions = np.array([0, 1, 77, 100000, -1], dtype=np.int32)  # -1: the largest unsigned position
    f = 10.0 ** -np.arange(n // 2)
    got = P.rotary(x, positions, f, interleaved, 1.25)
    for t in range(5):
        turn = 1.25 * np.exp(1j * (int(positions[t]) % 2 ** 32) * f)
        z = x[t, :, 0:n:2] + 1j * x[t, :, 1:n:2] if interleaved else x[t, :, :n // 2] + 1j * x[t, :, n // 2:n]
        z = z * turn
        want = np.stack([z.real, z.imag], -1).reshape(3, n) if interleaved else np.concatenate([z.real, z.imag], -1)
        np.testing.assert_allclose(got[t, :, :n], want, rtol=0, atol=1e-9)  # angles of 2^32 keep 2^-20 turns in 64 bits
        assert np.array_equal(got[t, :, n:], x[t, :, n:])
    s = P.rotary_scale(x, n, interleaved)
    assert np.all(s >= np.abs(x)) and np.array_equal(s[..., n:], np.abs(x[..., n:]))


def test_head_norm():
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((4, 2, 10)), rng.standard_normal(10)
    want = np.empty_like(x)
    for t in range(4):
        for h in range(2):
            want[t, h] = x[t, h] * w * np.sqrt(10) / np.sqrt(np.linalg.norm(x[t, h]) ** 2 + 10 * 1e-3)
    np.testing.assert_allclose(P.head_norm(x, w, 1e-3), want, rtol=1e-12)


def test_places():
    refs = np.array([[4, 2 | 1 << 31], [0, 9], [1, 3]], dtype=np.uint32)
    # sequence 0: 2 new, 17 after: places 15 and 16; 1: 3 new, 17 after, its second page's ref 9 of 8 blocks;
    # 2: more new tokens than it has; one padded row behind
    seq, place, row = P.places(9, 3, [17, 17, 2], [0, 2, 5, 8], refs, 2, 8)
    assert seq.tolist() == [0, 0, 1, 1, 1, -1, -1, -1, -1]
    assert place.tolist() == [15, 16, 14, 15, 16, -1, -1, -1, -1]
    assert row.tolist() == [4 * 16 + 15, 2 * 16, 14, 15, -1, -1, -1, -1, -1]
    seq, place, row = P.places(3, 3, [33, 1, 16], None, refs, 2, 8)  # a third page of a table of two
    assert seq.tolist() == [0, 1, 2] and place.tolist() == [32, 0, 15] and row.tolist() == [-1, 0, 31]


@pytest.mark.parametrize("causal", [False, True])
def test_shared_prefix_attention_is_attention_over_each_sequence(causal):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(5)
    pools = rng.standard_normal((2, 7, 16, 2, 8))
    prefix_refs, refs, own, prefix = [5, 1], np.array([[0, 2], [6, 3], [4, 4]]), [20, 3, 1], 19
    q = rng.standard_normal((3, 2, 4, 8))
    got = P.shared_prefix_attention(q, pools[0], pools[1], prefix_refs, prefix, refs, own, 0.3, causal)
    for b in range(3):
        pages = [np.concatenate([p[prefix_refs].reshape(-1, 2, 8)[:prefix], p[refs[b]].reshape(-1, 2, 8)[:own[b]]]) for p in pools]
        k, v = (torch.from_numpy(np.repeat(x.transpose(1, 0, 2), 2, axis=0)) for x in pages)
        n = prefix + own[b]
        mask = torch.arange(n)[None, :] < (torch.tensor([[n - 1], [n]]) if causal else torch.tensor([[n], [n]]))
        want = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q[b]).transpose(0, 1).contiguous(), k, v,
                                                                attn_mask=mask, scale=0.3)
        np.testing.assert_allclose(got[b], want.transpose(0, 1).numpy(), rtol=0, atol=1e-12)


def test_weight_sums():
    rng = np.random.default_rng(6)
    pools = rng.standard_normal((2, 4, 16, 1, 8))
    q = rng.standard_normal((2, 1, 2, 8))
    got = P.shared_prefix_weight_sums(q, pools[0], [2], 5, [[1], [0]], [4, 0], 0.5, True)
    for b, n in ((0, 4), (1, 0)):
        k = np.concatenate([pools[0][2, :5, 0], pools[0][1 - b, :n, 0]])
        s = q[b, 0] @ k.T * 0.5
        np.testing.assert_allclose(got[b, 0], [sum(np.exp(x - max(row)) for x in row) for row in s], rtol=1e-12)
    assert not P.shared_prefix_weight_sums(q, pools[0], [], 0, [[1], [0]], [0, 0], 0.5, True).any()


@pytest.mark.parametrize("shape", LONG_PREFIXES, ids=["many-rows", "few-rows", "own"])
def test_the_bounds_of_long_prefixes_see_what_is_lost(shape):
    """Zeros, half of the tokens, and any single page left out miss the bounds that the GPU's outputs over these many
    tokens are held to."""
    batch, queries, hq, hk, hd, prefix, own = shape
    rng = np.random.default_rng(34)
    pages = [-(-n // 16) for n in own]
    shared = -(-prefix // 16)
    blocks = shared + sum(pages)
    order = rng.permutation(blocks)
    refs = np.full((batch, max(pages)), blocks)
    for b, n in enumerate(pages):
        refs[b, :n] = order[shared + sum(pages[:b]):][:n]
    q = (rng.standard_normal((batch, queries, hq, hd)) * 0.25).astype(np.float16)
    k, v = (rng.standard_normal((blocks, 16, hk, hd)).astype(np.float16) for _ in range(2))
    shape = (batch, queries, hq, hd)
    want, absolute, half, total = np.zeros(shape), np.zeros(shape), np.zeros(shape), np.zeros(shape[:3])
    lost = [0.0] * batch  # squared error of a sequence for each page left out
    for at, w, x in P._seen_scores(q, k, v, order[:shared], prefix, refs, own, hd ** -0.5, True):
        tokens = w.shape[1]
        total[at] = w.sum(1)
        want[at], absolute[at] = w @ x / total[at][:, None], w @ np.abs(x) / total[at][:, None]
        half[at] = w[:, :tokens // 2] @ x[:tokens // 2] / w[:, :tokens // 2].sum(1, keepdims=True)
        first = np.concatenate([np.arange(0, prefix, 16), np.arange(prefix, tokens, 16)])
        for h in range(w.shape[0]):
            sums = np.add.reduceat(w[h][:, None] * x, first, axis=0)
            rest = total[at][h] - np.add.reduceat(w[h], first)
            lost[at[0]] = lost[at[0]] + (((want[at][h] * total[at][h] - sums) / rest[:, None] - want[at][h]) ** 2).sum(1)
    n, largest = prefix + max(own), float(np.abs(v).max())
    for what, got in (("zeros", np.zeros(shape)), ("half", half)):
        worst, rel = prefix_errors(got, want, absolute, total, n, largest)
        assert worst > 1.0 and rel > 2 * PREFIX_REL_L2, what
    assert prefix_errors(want.astype(np.float16), want, absolute, total, n, largest)[0] < 1.0
    for b in range(batch):
        rel = np.sqrt(lost[b]) / np.linalg.norm(want[b])
        print(f"sequence {b}: a page left out is {rel.min():.2e} to {rel.max():.2e} of the output", flush=True)
        assert rel.min() > 2 * PREFIX_REL_L2


def test_shared_prefix_rows_that_see_nothing_are_zeros():
    pools = np.ones((2, 1, 16, 1, 8))
    out = P.shared_prefix_attention(np.ones((1, 3, 1, 8)), pools[0], pools[1], [], 0, [[0]], [1], 1.0, True)
    assert np.array_equal(out[0, :2], np.zeros((2, 1, 8))) and np.array_equal(out[0, 2], np.ones((1, 8)))
