"""Pins of oracle/step_oracle.py, the restatement that the GPU tests of a step over trees compare with."""
from __future__ import annotations

import itertools

import numpy as np
import pytest

from oracle import step_oracle as S


def tree(rng, n):
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)] if n else []


@pytest.mark.parametrize("n", [0, 1, 2, 33, 70])
def test_masks_against_reachability(n):
    rng = np.random.default_rng(n)
    parents = tree(rng, n)
    a = np.eye(n, dtype=np.int64)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i, p] = 1
    reach = np.linalg.matrix_power(a.astype(object), max(n, 1)) > 0 if n else np.zeros((0, 0), dtype=bool)
    words = -(-max(n, 1) // 32)
    mask = S.mask_of([parents], n + 2, words)
    got = np.array([[int(mask[i, j // 32]) >> (j % 32) & 1 for j in range(n)] for i in range(n)], dtype=bool).reshape(n, n)
    assert np.array_equal(got, reach.astype(bool)) and not mask[n:].any()
    assert [d for _, d in S.sees_of(parents)] == [int(r.sum()) - 1 for r in reach]


def test_tables_against_a_pool_that_hands_out_pages_token_by_token():
    rng = np.random.default_rng(0)
    held, new = [0, 1, 15, 16, 17, 40, 0, 33], [3, 15, 1, 1, 0, 30, 0, 16]
    extra = [0, 1, 0, 0, 0, 2, 3, 0]
    pages = [-(-h // 16) + x for h, x in zip(held, extra)]
    order = rng.permutation(60)
    refs = np.full((8, 9), S.REF_MASK, dtype=np.int64)
    at = 0
    for b, p in enumerate(pages):
        refs[b, :p] = order[at:at + p]
        at += p
    free = order[at:]
    got = S.page_tables(refs, held, new, pages, free, 2, sum(new) + 3, 9)
    take, table, slots = iter(free[2:]), refs.copy(), []
    for b in range(8):
        have = pages[b]
        for i in range(new[b]):
            place = held[b] + i
            if place // 16 == have:
                table[b, have] = next(take)
                have += 1
            slots.append(table[b, place // 16] * 16 + place % 16)
        assert got["pages_out"][b] == have and got["seq_hot"][b] == held[b] + new[b]
    assert np.array_equal(got["refs"], table) and got["slots"].tolist() == slots + [-1] * 3 and not got["errors"]
    assert int(free[got["free_next"]]) == next(take)
    assert S.page_tables(refs, held, new, pages, free[:3], 2, sum(new), 9)["errors"] == {"free pages"}
    assert S.page_tables(refs, held, new, pages, free, 2, sum(new) - 1, 9)["errors"] == {"sequence length"}


def test_attention_against_one_softmax_with_a_dense_mask():
    rng = np.random.default_rng(1)
    held, n, hq, hk, hd = [19, 0], [5, 3], 4, 2, 8
    hot = [rng.standard_normal((6, 16, hk, hd)) for _ in range(2)]
    refs = np.array([[4 | 1 << 31, 1], [0, 0]])
    q, k, v = (rng.standard_normal((9, h, hd)) for h in (hq, hk, hk))
    trees = [tree(rng, x) for x in n]
    mask = S.mask_of(trees, 9, 1)
    mask[6] = 0
    out, absolute, total = S.tree_attention(q, k, v, *hot, refs, held, S.offsets_of(n), mask, 0.3)
    assert np.isnan(out[8]).all() and (out[6] == 0).all() and (total[6] == 0).all()
    for r in range(8):
        b, first = (0, 0) if r < 5 else (1, 5)
        keys = np.concatenate([hot[0][[4, 1]].reshape(32, hk, hd)[:held[b]], k[first:first + n[b]]])
        vals = np.concatenate([hot[1][[4, 1]].reshape(32, hk, hd)[:held[b]], v[first:first + n[b]]])
        hide = np.zeros(len(keys))
        for j in range(n[b]):
            if not int(mask[r, 0]) >> j & 1:
                hide[held[b] + j] = -np.inf
        if r == 6:
            continue
        for h in range(hq):
            s = keys[:, h // 2] @ q[r, h] * 0.3 + hide
            w = np.exp(s) / np.exp(s).sum()
            assert np.allclose(out[r, h], w @ vals[:, h // 2]) and np.allclose(absolute[r, h], w @ np.abs(vals[:, h // 2]))
            assert np.isclose(total[r, h], np.exp(s).sum() / np.exp(s).max())


def test_logits_against_counts():
    rng = np.random.default_rng(2)
    vocab, n = 50, 4
    x = rng.standard_normal((n, vocab)).astype(np.float32)
    history = rng.integers(0, vocab, (1, 40))
    nodes, mask = np.array([7, 7, 3, 9]), S.mask_of([[-1, 0, 1, 0]], n, 1)
    got, best = S.adjust_logits(x, [0, n], history, [30], [12], [1.5], [0.25], [0.5], nodes, mask, np.array([[3, 8, 3]]),
                                np.array([[9.0, 1.0, -2.0]]))
    for r, mine in enumerate([[7], [7, 7], [7, 7, 3], [7, 9]]):
        made = np.bincount(np.concatenate([history[0, 12:30], mine]).astype(int), minlength=vocab)
        seen = made + np.bincount(history[0, :12], minlength=vocab) > 0
        want = np.where(seen, np.where(x[r] > 0, x[r] / 1.5, x[r] * 1.5), x[r]) - 0.25 * made - 0.5 * (made > 0)
        want[3] += -2.0
        want[8] += 1.0
        assert np.allclose(got[r], want, rtol=1e-6, atol=1e-6) and best[r] == int(np.argmax(got[r]))
    words = np.zeros((2, 2), dtype=np.uint32)
    words[1, 1] = 1 << 5
    got, best = S.adjust_logits(x, allowed=words, allowed_index=[0, 1, -1, 2])
    assert (got[0] == -np.inf).all() and got[1, 37] == x[1, 37] and np.array_equal(got[2], x[2]) and (got[3] == -np.inf).all()
    assert best.tolist() == [-1, 37, int(x[2].argmax()), -1]


def test_acceptance_against_all_paths():
    rng = np.random.default_rng(3)
    for n, _ in itertools.product([1, 2, 6, 40], range(5)):
        parents, tokens, targets = tree(rng, n), rng.integers(0, 3, n), rng.integers(0, 3, n)
        path = S.accept_tree(parents, tokens, targets, [0, n])[0]
        good = [0]  # every node whose whole path was the lowest match at each step
        for i in range(1, n):
            p = parents[i]
            rivals = [j for j in range(1, i) if parents[j] == p and tokens[j] == targets[p]]
            if p in good and tokens[i] == targets[p] and not rivals:
                good.append(i)
        assert path == good
    assert S.accept_tree([], [], [], [0, 0]) == [[]]


def test_tables_after_a_list_that_ended():
    """What a step found no page for is not a page that a sequence has: the next step takes it."""
    free, none = np.array([7, 8, 9]), np.array([], dtype=np.int64)
    first = S.page_tables([[3, 0, 0]], [16], [4], [1], none, 0, 4, 3)
    assert first["errors"] == {"free pages"} and first["pages_out"].tolist() == [1] and (first["slots"] < 0).all()
    assert first["refs"].tolist() == [[3, S.REF_MASK, 0]]
    again = S.page_tables(first["refs"], [16], [4], first["pages_out"], free, 0, 4, 3)
    assert not again["errors"] and again["pages_out"].tolist() == [2] and again["slots"].tolist() == [7 * 16 + i for i in range(4)]
    assert again["refs"].tolist() == [[3, 7, 0]] and again["free_next"] == 1
    held = S.page_tables(first["refs"], [20], [14], first["pages_out"], free, 0, 14, 3)  # held without a page: none is taken behind it
    assert held["errors"] == {"sequence length"} and held["pages_out"].tolist() == [1] and (held["slots"] < 0).all() and held["free_next"] == 0
    hole = S.page_tables(first["refs"], [20], [14], [2], free, 0, 14, 3)  # counted as a page although it names none
    assert hole["errors"] == {"free pages"} and hole["pages_out"].tolist() == [3] and (hole["slots"] < 0).sum() == 12


def test_acceptance_before_a_row_without_a_slot():
    parents, tokens = [-1, 0, 1, 2, -1, 0], [5, 6, 7, 8, 3, 4]
    targets, offsets = [6, 7, 8, 9, 4, 2], [0, 4, 6]
    assert S.accept_tree(parents, tokens, targets, offsets, [9, -1, 2, 3, 4, 5]) == [[0, 1, 2, 3], [0, 1]]
    assert S.accept_tree(parents, tokens, targets, offsets, [9, -1, S.NO_SLOT, 3, S.NO_SLOT, 5]) == [[0, 1], []]


def test_tables_of_a_sequence_past_its_table_leave_the_others():
    """The second of three sequences fits, is full, or has more nodes than the mask: the rows of the third are the same."""
    parents = [-1, 0, 1, -1, 0, 0, -1, 0, 1]
    args = dict(pages=None, free=np.arange(5, 20), first=0, rows=9, hot_count=3, parents=parents, words=1)
    refs = np.arange(9).reshape(3, 3)
    good, full = S.page_tables(refs, [4, 30, 16], [3, 3, 3], **args), S.page_tables(refs, [4, 47, 16], [3, 3, 3], **args)
    assert not good["errors"] and full["errors"] == {"sequence length"}
    for name in ("positions", "tree_mask"):
        assert np.array_equal(good[name][6:], full[name][6:])
    assert full["token_offsets"].tolist() == [0, 3, 6, 9] and full["slots"][3] >= 0 and (full["slots"][4:6] == S.NO_SLOT).all()
    assert (full["slots"][6:] % 16 == good["slots"][6:] % 16).all() and full["pages_out"].tolist() == [1, 3, 2]
    wide = S.page_tables(refs, [4, 30, 16], [3, 40, 3], **{**args, "rows": 46, "parents": parents[:3] + [-1] * 40 + parents[6:]})
    assert wide["errors"] == {"sequence length"} and (wide["slots"][3:43] == S.NO_SLOT).all() and not wide["tree_mask"][35:43].any()
    assert wide["pages_out"].tolist() == [1, 2, 2] and np.array_equal(wide["tree_mask"][43:], good["tree_mask"][6:])
