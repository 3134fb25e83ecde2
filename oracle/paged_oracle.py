"""CPU restatement, in float64, of the operators around a batch over pages.

TEST INFRASTRUCTURE ONLY: imported by tests/ to check aw_ops_rotary,
aw_ops_qk_norm_rotary, aw_ops_append_paged (include/aether_ops.h) and
aw_shared_prefix_attention_device (include/aether_weaver.h), never by the product
package.  numpy.

Pins (tests/test_paged_oracle.py): the rotation against a complex multiplication by
e^{i angle}, the norm against np.linalg.norm, the append against a loop over tokens in
the words of its description, the attention against one softmax over each sequence's
tokens laid end to end.
"""
from __future__ import annotations

import numpy as np

PAGE = 16
REF_MASK = 0x7FFFFFFF


def head_norm(x, weight, eps: float) -> np.ndarray:
    x = np.asarray(x, dtype=np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)


def rotary(x, positions, inv_freq, interleaved: bool = False, magnitude: float = 1.0) -> np.ndarray:
    """x [tokens][heads][head_dim]; positions are unsigned; dims past 2 * len(inv_freq) pass."""
    x = np.asarray(x, dtype=np.float64)
    angle = np.asarray(positions).astype(np.uint32).astype(np.float64)[:, None, None] * np.asarray(inv_freq, dtype=np.float64)
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    n = 2 * angle.shape[-1]
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def rotary_scale(x, n: int, interleaved: bool = False) -> np.ndarray:
    """|x0| + |x1| of the pair that each value belongs to (|x| where it passes): the scale of a rotation's rounding."""
    x = np.abs(np.asarray(x, dtype=np.float64))
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y = x.copy()
    y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


def places(tokens: int, batch: int, seq_hot, offsets, refs, hot_count: int, hot_blocks: int):
    """For each token of an append: (its sequence or -1, its place or -1, its pool row or -1)."""
    if offsets is None:
        offsets = [tokens // batch * b for b in range(batch + 1)]
    seq, place, row = (np.full(tokens, -1, dtype=np.int64) for _ in range(3))
    for b in range(batch):
        first, end = int(offsets[b]), int(offsets[b + 1])
        if end - first > int(seq_hot[b]):
            continue
        for t in range(first, min(end, tokens)):
            seq[t], place[t] = b, int(seq_hot[b]) - (end - t)
            page = place[t] // PAGE
            ref = int(refs[b][page]) & REF_MASK if page < hot_count else hot_blocks
            if ref < hot_blocks:
                row[t] = ref * PAGE + place[t] % PAGE
    return seq, place, row


def _seen_scores(q, hot_k, hot_v, prefix_refs, prefix_tokens: int, refs, seq_own, scale: float, causal: bool):
    """((sequence, query, kv head), its heads' exp(score - largest), the values), of what each query sees."""
    q = np.asarray(q, dtype=np.float64)
    blocks, _, kv_heads, hd = hot_k.shape
    batch, queries, q_heads, _ = q.shape
    group = q_heads // kv_heads

    def gather(table, tokens):
        at = np.asarray([(int(table[t // PAGE]) & REF_MASK, t % PAGE) for t in range(tokens)], dtype=np.int64).reshape(-1, 2)
        ok = at[:, 0] < blocks
        at = np.where(ok[:, None], at, 0)
        return hot_k[at[:, 0], at[:, 1]].astype(np.float64), hot_v[at[:, 0], at[:, 1]].astype(np.float64), ok

    pk, pv, pok = gather(prefix_refs, prefix_tokens)
    for b in range(batch):
        n = int(seq_own[b])
        ok_, ov, oseen = gather(refs[b], n)
        for i in range(queries):
            lim = max(0, n - queries + 1 + i) if causal else n
            see = np.concatenate([pok, oseen & (np.arange(n) < lim)])
            if not see.any():
                continue
            k, v = np.concatenate([pk, ok_])[see], np.concatenate([pv, ov])[see]
            for g in range(kv_heads):
                s = q[b, i, g * group:(g + 1) * group] @ k[:, g].T * scale
                yield (b, i, slice(g * group, (g + 1) * group)), np.exp(s - s.max(1, keepdims=True)), v[:, g]


def shared_prefix_attention(q, hot_k, hot_v, prefix_refs, prefix_tokens: int, refs, seq_own, scale: float, causal: bool):
    """q [batch][queries][q_heads][head_dim], pools [blocks][16][kv_heads][head_dim]; query i of Q sees
    every prefix token and own tokens p < seq_own - Q + 1 + i (all of them where not causal).  Rows that
    see nothing are zeros.  Out-of-range refs (>= blocks) hide their tokens."""
    out = np.zeros(np.shape(q))
    for at, w, v in _seen_scores(q, hot_k, hot_v, prefix_refs, prefix_tokens, refs, seq_own, scale, causal):
        out[at] = (w / w.sum(1, keepdims=True)) @ v
    return out


def shared_prefix_weight_sums(q, hot_k, prefix_refs, prefix_tokens: int, refs, seq_own, scale: float, causal: bool):
    """[batch][queries][q_heads]: the sum of a row's weights where its largest is 1 (0 for a row that sees nothing)."""
    total = np.zeros(np.shape(q)[:3])
    for at, w, _ in _seen_scores(q, hot_k, hot_k, prefix_refs, prefix_tokens, refs, seq_own, scale, causal):
        total[at] = w.sum(1)
    return total
