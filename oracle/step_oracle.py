"""CPU restatement of a step over trees of drafted tokens.

TEST INFRASTRUCTURE ONLY: imported by tests/ to check aw_ops_page_tables,
aw_ops_adjust_logits, aw_ops_accept_tree (include/aether_ops.h) and
aw_tree_attention_device (include/aether_weaver.h), never by the product package.  numpy;
attention in float64, logits in float32 as their description rounds them, the rest whole
numbers.

Pins (tests/test_step_oracle.py): tables against a pool that hands out pages one token at
a time, masks against reachability by matrix powers, attention against one softmax with a dense mask,
logits against counts by np.bincount, acceptance against a search of all paths.
"""
from __future__ import annotations

import numpy as np

PAGE = 16
REF_MASK = 0x7FFFFFFF
MAX_NODES = 1024
NO_SLOT = -(1 << 63)


def offsets_of(counts) -> list:
    return [0] + np.cumsum(np.asarray(counts, dtype=np.int64)).tolist()


def sees_of(parents) -> list:
    """For each node of one tree the set (as bits) of itself and its ancestors, its depth; a parent that is not
    an earlier node makes a root."""
    out = []
    for i, p in enumerate(parents):
        p = int(p)
        bits, depth = out[p] if 0 <= p < i else (0, -1)
        out.append((bits | 1 << i, depth + 1))
    return out


def mask_of(trees, rows: int, words: int) -> np.ndarray:
    """[rows][words] of the trees' rows one after another; rows behind the last see nothing."""
    out = np.zeros((rows, words), dtype=np.uint32)
    t = 0
    for parents in trees:
        for bits, _ in sees_of(parents):
            for w in range(words):
                out[t, w] = bits >> (32 * w) & 0xFFFFFFFF
            t += 1
    return out


def page_tables(refs, held, new, pages, free, first: int, rows: int, hot_count: int, parents=None, words: int = 0) -> dict:
    """What aw_ops_page_tables writes (refs [batch][>= hot_count] as they were before), and "errors"."""
    refs = np.array(refs, dtype=np.int64)
    batch, errors, t, f = len(held), set(), 0, int(first)
    got = {k: np.zeros(batch, dtype=np.int64) for k in ("seq_hot", "pages_out")}
    offsets, slots, positions = [0], np.full(rows, -1, dtype=np.int64), np.zeros(rows, dtype=np.int64)
    mask = np.zeros((rows, words), dtype=np.uint32)
    for b in range(batch):
        h, n = int(held[b]), min(int(new[b]), rows - t)
        room = hot_count * PAGE
        many = parents is not None and int(new[b]) > 32 * words
        if n < int(new[b]) or int(new[b]) > max(0, room - h) or h > room or many:
            errors.add("sequence length")
        least = -(-h // PAGE)
        p = least if pages is None else int(pages[b])
        lacks = p < least
        if lacks:
            errors.add("sequence length")
        need = max(0, -(-min(h + n, room) // PAGE) - p) if n and h < room and not lacks and not many else 0
        mine = [int(x) & REF_MASK for x in free[f:f + need]]
        if len(mine) < need:
            errors.add("free pages")
        f += need
        tree = None if parents is None else sees_of(parents[t:t + min(n, 32 * words)])
        for i in range(n):
            at, ref = (h + i) // PAGE, REF_MASK
            if h + i < room:
                if at >= p:
                    ref = mine[at - p] if at - p < len(mine) else REF_MASK
                    if i == 0 or (h + i) % PAGE == 0:
                        refs[b, at] = ref
                else:
                    ref = int(refs[b, at]) & REF_MASK
                    if ref == REF_MASK:
                        errors.add("free pages")
                    ref = REF_MASK if many else ref
            slots[t] = NO_SLOT if ref == REF_MASK else ref * PAGE + (h + i) % PAGE
            sees, depth = (0, i) if tree is None else tree[i] if i < len(tree) else (0, 0)
            positions[t] = h + depth
            for w in range(words):
                mask[t, w] = sees >> (32 * w) & 0xFFFFFFFF
            if tree is not None and i < len(tree) and int(parents[t]) >= i:
                errors.add("sequence length")
            t += 1
        got["seq_hot"][b], got["pages_out"][b] = h + n, p + len(mine)
        offsets.append(t)
    return {**got, "refs": refs, "token_offsets": np.array(offsets), "free_next": min(f, max(len(free), int(first))), "slots": slots,
            "positions": positions, "tree_mask": mask, "errors": errors}


def tree_attention(q, k, v, hot_k, hot_v, refs, held, offsets, mask, scale: float):
    """(outputs, the sums A of p |v| / sum p, the sums W of weights whose largest is 1); NaN in the outputs of rows
    behind the last sequence.  q [rows][q_heads][head_dim], k and v [rows][kv_heads][head_dim]."""
    q = np.asarray(q, dtype=np.float64)
    rows, hq, hd = q.shape
    hk = k.shape[1]
    group = hq // hk
    out, absolute, total = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b in range(len(offsets) - 1):
        first, end = int(offsets[b]), int(offsets[b + 1])
        n, h = end - first, int(held[b])
        at = np.asarray([(int(refs[b][p // PAGE]) & REF_MASK, p % PAGE) for p in range(h)], dtype=np.int64).reshape(-1, 2)
        ok = at[:, 0] < (0 if hot_k is None else hot_k.shape[0])
        at = at[ok]
        kk = k[first:end].astype(np.float64)
        vv = v[first:end].astype(np.float64)
        if at.size:
            kk = np.concatenate([hot_k[at[:, 0], at[:, 1]].astype(np.float64), kk])
            vv = np.concatenate([hot_v[at[:, 0], at[:, 1]].astype(np.float64), vv])
        for i in range(n):
            if mask is None:
                sees = np.arange(n) <= i
            else:
                bits = sum(int(w) << (32 * x) for x, w in enumerate(mask[first + i]))
                sees = np.array([bits >> j & 1 for j in range(n)], dtype=bool)
            see = np.concatenate([np.ones(len(at), dtype=bool), sees])
            out[first + i] = 0.0
            if not see.any():
                continue
            for g in range(hk):
                heads = slice(g * group, (g + 1) * group)
                s = q[first + i, heads] @ kk[see, g].T * scale
                w = np.exp(s - s.max(1, keepdims=True))
                total[first + i, heads] = w.sum(1)
                out[first + i, heads] = w / w.sum(1, keepdims=True) @ vv[see, g]
                absolute[first + i, heads] = w / w.sum(1, keepdims=True) @ np.abs(vv[see, g])
    return out, absolute, total


def adjust_logits(logits, offsets=None, history=None, history_count=None, prompt_count=None, repetition=None, frequency=None,
                  presence=None, node_tokens=None, mask=None, bias_ids=None, bias_values=None, bias_count=None, allowed=None,
                  allowed_index=None):
    """(x in float32 before it is rounded to the output's type, best); rows behind the last sequence: NaN, -2."""
    rows, vocab = logits.shape
    one = np.float32
    out, best = np.full((rows, vocab), np.nan, dtype=np.float32), np.full(rows, -2, dtype=np.int64)
    batch = None if offsets is None else len(offsets) - 1
    for r in range(rows):
        b, first, end = None, 0, 0
        if batch is not None:
            b = next((x for x in range(batch) if int(offsets[x]) <= r < int(offsets[x + 1])), None)
            if b is None:
                continue
            first, end = int(offsets[b]), int(offsets[b + 1])
        counts, prompt = {}, set()
        if history is not None:
            n, p = min(int(history_count[b]), history.shape[1]), 0 if prompt_count is None else int(prompt_count[b])
            prompt = {int(t) & 0xFFFFFFFF for t in history[b, :min(n, p)]}
            for t in history[b, p:n]:
                counts[int(t) & 0xFFFFFFFF] = counts.get(int(t) & 0xFFFFFFFF, 0) + 1
        if node_tokens is not None:
            for j in range(min(end - first, 32 * mask.shape[1])):
                if int(mask[r, j // 32]) >> (j % 32) & 1:
                    t = int(node_tokens[first + j]) & 0xFFFFFFFF
                    counts[t] = counts.get(t, 0) + 1
        x = logits[r].astype(np.float32)
        rep = one(1.0) if repetition is None else one(repetition[b])
        freq = one(0.0) if frequency is None else one(frequency[b])
        pres = one(0.0) if presence is None else one(presence[b])
        with np.errstate(all="ignore"):
            for t in prompt | set(counts):
                if t < vocab:
                    x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            for t, c in counts.items():
                if t < vocab:
                    x[t] = one(x[t] - one(freq * one(c)))
                    x[t] = one(x[t] - pres)
            if bias_ids is not None:
                n = bias_ids.shape[1] if bias_count is None else min(int(bias_count[b]), bias_ids.shape[1])
                last = {int(t) & 0xFFFFFFFF: e for e, t in enumerate(bias_ids[b, :n])}
                for t, e in last.items():
                    if t < vocab:
                        x[t] = one(x[t] + one(bias_values[b, e]))
        if allowed is not None:
            a = r if allowed_index is None else int(allowed_index[r])
            if a >= allowed.shape[0]:
                x[:] = -np.inf
            elif a >= 0:
                bits = np.unpackbits(np.ascontiguousarray(allowed[a]).astype("<u4").view(np.uint8), bitorder="little")[:vocab]
                x[bits == 0] = -np.inf
        out[r] = x
        finite = np.where(np.isnan(x), -np.inf, x)
        best[r] = int(np.argmax(finite)) if finite.max() > -np.inf else -1
    return out, best


def accept_tree(parents, tokens, targets, offsets, slots=None) -> list:
    """The kept nodes of each sequence, in order; with slots, those before the first row without one."""
    paths = []
    for b in range(len(offsets) - 1):
        first, n = int(offsets[b]), min(int(offsets[b + 1]) - int(offsets[b]), MAX_NODES)
        path = [0] if n else []
        while path:
            cur = path[-1]
            target = int(targets[first + cur]) & 0xFFFFFFFF
            child = [j for j in range(cur + 1, n) if int(parents[first + j]) == cur and int(tokens[first + j]) & 0xFFFFFFFF == target != 0xFFFFFFFF]
            if not child:
                break
            path.append(child[0])
        if slots is not None:
            path = path[:next((j for j in range(n) if int(slots[first + j]) == NO_SLOT), n)]
        paths.append(path)
    return paths
