"""A step over trees of drafted tokens without a GPU: descriptors at an edge of what their description allows."""
from __future__ import annotations

import pytest
import torch

from aether_nexus_amd import ops as O
from aether_nexus_amd.types import AW_E_INVALID_ARG, AW_E_UNSUPPORTED
from aether_nexus_amd.weaver import WeaverError
from test_step import A, accept, check, tree


@pytest.mark.parametrize("kw", [dict(v_stride=257), dict(v_stride=8), dict(v_stride=1 << 40), dict(k_stride=1536, k=A["q"] + 2 * 1024, q_stride=1536)])
def test_v_stride_is_not_read_without_v(kw):
    assert O.tree_plan(tree(v=0, hot_v=0, **kw)).work_groups


# ---------------------------------------------------------------- tensors of other shapes than the request's

@pytest.fixture
def on_cpu(monkeypatch):
    """Descriptors of CPU tensors: every check of a tensor but that it is on the GPU."""
    def check(t, need, what, dtypes):
        if t is None or isinstance(t, int):
            return
        if t.dtype not in dtypes or not t.is_contiguous() or t.numel() < need:
            raise WeaverError(f"{what}: dtype, contiguity or {t.numel()} < {need}", AW_E_INVALID_ARG)
    monkeypatch.setattr(O, "_check_tensor", check)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refused(make, **kw):
    with pytest.raises(WeaverError) as e:
        make(**kw)
    assert e.value.status == AW_E_INVALID_ARG
    return str(e.value)


def logits_of(rows=3, vocab=1000, **kw):
    return O.make_logits_desc(**{**dict(num_tokens=rows, vocab_size=vocab, logits=torch.zeros(rows, vocab), best=i32(rows)), **kw})


def test_logits_of_a_padded_vocabulary(on_cpu):
    """Rows longer than the vocabulary are a tensor's own, contiguous or sliced; flat tensors are rows of the vocabulary."""
    for wide in (torch.zeros(3, 1024), torch.zeros(3, 1024)[:, :1000], torch.zeros(5, 1024), torch.zeros(1, 3, 1024)):
        d = logits_of(logits=wide, out=wide, allowed=i32(3, 40))
        assert (d.logits_stride, d.out_stride, d.allowed_stride) == (1024, 1024, 40)
    d = logits_of(logits=torch.zeros(3, 1000), out=torch.zeros(3000), allowed=i32(3 * 32), allowed_rows=3)
    assert (d.logits_stride, d.out_stride, d.allowed_stride) == (1000, 1000, 32)
    d = logits_of(allowed=i32(7, 64)[:, :32])
    assert (d.allowed_stride, d.allowed_rows) == (64, 7)
    assert logits_of(rows=1, logits=torch.zeros(1, 1000).expand(1, 1000)).logits_stride >= 1000
    assert logits_of(rows=0, logits=torch.zeros(0, 1000)).num_tokens == 0


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(6, 500)), dict(logits=torch.zeros(1, 3000)), dict(logits=torch.zeros(2, 1024)), dict(logits=torch.zeros(2999)),
    dict(logits=torch.zeros(3, 999)), dict(logits=torch.zeros(1, 1000).expand(3, 1000)), dict(logits=torch.zeros(1000, 3).t()),
    dict(logits=torch.zeros(3, 2, 1000)[:, 0], out=torch.zeros(3, 1, 2, 1000)[:, :, 0]), dict(out=torch.zeros(3, 2000)[:, ::2]),
    dict(allowed=i32(3, 31)), dict(allowed=i32(2, 40), allowed_rows=3), dict(allowed=i32(6, 16), allowed_rows=3)], ids=lambda d: None)
def test_rows_of_another_shape_are_refused(on_cpu, kw):
    refused(logits_of, **kw)


def test_row_lengths_that_differ_from_their_tensors_are_refused(on_cpu):
    own = dict(batch=2, bias_count=i32(2), token_offsets=i32(3))
    f32 = torch.zeros(2, 16)
    assert logits_of(**own, bias_ids=i32(2, 16), bias_values=f32).bias_stride == 16
    assert logits_of(**own, bias_ids=i32(2, 8), bias_values=torch.zeros(16)).bias_stride == 8  # flat: rows of the ids' length
    assert "bias_values" in refused(logits_of, **own, bias_ids=i32(2, 8), bias_values=f32)
    assert "bias_ids" in refused(logits_of, **own, bias_ids=i32(2, 16), bias_values=f32, bias_stride=8)
    assert "history" in refused(logits_of, **own, history=i32(2, 64), history_count=i32(2), history_stride=32)
    assert "tree_mask" in refused(logits_of, **own, node_tokens=i32(3), tree_mask=i32(3, 4), mask_words=1)
    tables = dict(batch=2, num_tokens=3, seq_held=i32(2), seq_new=i32(2), refs=i32(2, 4), seq_hot=i32(2), token_offsets=i32(3), parents=i32(3))
    assert O.make_tables_desc(**tables, tree_mask=i32(3, 2), mask_words=2).mask_words == 2
    assert "tree_mask" in refused(O.make_tables_desc, **tables, tree_mask=i32(3, 2), mask_words=1)


def accept_of(layers=3, tokens=6, **kw):
    own = {n: A[n] for n in ("parents", "node_tokens", "targets", "seq_held", "accepted", "next_token", "seq_hot", "path", "slots", "hot_k", "hot_v")}
    return O.make_accept_desc(**{**dict(batch=2, num_tokens=tokens, layers=layers, kv_heads=2, head_dim=64, hot_blocks=9, v=A["v"], **own), **kw})


def f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def test_expanded_rows_are_refused(on_cpu):
    """A stride of 0 would be taken for contiguous rows, layers or tokens times the memory that is there."""
    refused(accept_of, k=f16(1, 6, 2, 64).expand(3, 6, 2, 64))
    refused(accept_of, k=f16(3, 1, 2, 64).expand(3, 6, 2, 64))
    refused(accept_of, k=f16(3, 6, 2, 64), v=f16(1, 6, 2, 64).expand(3, 6, 2, 64))
    d = accept_of(k=f16(6, 3, 9, 64).transpose(0, 1)[:, :, 5:7])
    assert (d.k_layer_stride, d.k_stride) == (9 * 64, 27 * 64)
    d = accept_of(layers=1, k=f16(6, 9, 64)[None, :, 5:7])  # one layer, one token: no stride is taken
    assert (d.k_layer_stride, d.k_stride) == (0, 9 * 64)
    d = accept_of(tokens=1, k=f16(3, 1, 9, 64)[:, :, 5:7])
    assert (d.k_layer_stride, d.k_stride) == (9 * 64, 0)


def test_rows_of_a_larger_buffer(on_cpu):
    """k and v of more tokens or layers than the step's: the buffer's own strides, contiguous or not."""
    for k in (f16(3, 10, 2, 64), f16(5, 10, 2, 64), f16(3, 10, 128)):
        d = accept_of(k=k, v=f16(3, 6, 2, 64))
        assert (d.k_layer_stride, d.k_stride, d.v_layer_stride, d.v_stride) == (1280, 128, 768, 128)
    for k in (f16(2, 64).expand(18, 2, 64).contiguous(), f16(20, 128), f16(3 * 6 * 128)):  # layers one after another
        assert (lambda d: (d.k_layer_stride, d.k_stride))(accept_of(k=k)) == (0, 0)
    for k in (f16(9, 2, 64), f16(9, 128), f16(1, 9, 2, 64), f16(7, 9, 2, 64)):
        assert (lambda d: (d.k_layer_stride, d.k_stride))(accept_of(layers=1, k=k)) == (0, 128)
    d = accept_of(layers=1, k=f16(9, 6, 64)[:, 2:4])
    assert (d.k_layer_stride, d.k_stride) == (0, 384)
    assert accept_of(layers=0, k=None, v=None, hot_k=None, hot_v=None).k_stride == 0


@pytest.mark.parametrize("shape", [(3, 6, 3, 64), (3, 6, 2, 128), (3, 5, 2, 64), (2, 9, 2, 64), (2, 18, 2, 64), (17, 2, 64), (6, 3, 64), (3 * 6 * 128 - 1,),
                                   (18, 64, 2), (1, 3, 6, 2, 64), (9, 256)])
def test_rows_of_other_heads_are_refused(on_cpu, shape):
    refused(accept_of, k=f16(*shape))


def test_pools_of_more_layers_or_blocks(on_cpu):
    """A pool's own layers: not the elements of all of them shared out over the step's."""
    def of(d):
        return d.hot_blocks, d.hot_layer_stride
    page, flat = 16 * 128, f16(3, 6, 2, 64)
    kw = dict(k=flat, v=flat, hot_blocks=None)
    for pool, want in ((f16(3, 9, 16, 2, 64), (9, 0)), (f16(5, 9, 16, 2, 64), (9, 0)), (f16(3 * 9 * page), (9, 0)), (f16(27, 16, 2, 64), (9, 0))):
        assert of(accept_of(**kw, hot_k=pool, hot_v=pool)) == want
    pool = f16(3, 12, 16, 2, 64)
    assert of(accept_of(**{**kw, "hot_blocks": 9}, hot_k=pool, hot_v=pool)) == (9, 12 * page)
    for layers in (1, 2):
        d = accept_of(layers=layers, k=flat, v=flat, hot_k=pool, hot_v=pool, hot_blocks=None)
        assert of(d) == (12, 0)
    assert of(accept_of(layers=1, k=flat, v=flat, hot_k=f16(9, 16, 2, 64), hot_v=f16(1, 9, 16, 2, 64), hot_blocks=None)) == (9, 0)


@pytest.mark.parametrize("kw", [
    dict(hot_k=f16(2, 30, 16, 2, 64)), dict(hot_k=f16(3, 9, 16, 3, 64)), dict(hot_k=f16(3, 9, 16, 1, 128)), dict(hot_k=f16(27, 16, 4, 32)),
    dict(hot_k=f16(3, 9, 16, 2, 64), hot_blocks=10), dict(hot_k=f16(3, 9, 16, 2, 64), hot_v=f16(3, 8, 16, 2, 64)),
    dict(hot_k=f16(3, 9, 16, 2, 64), hot_v=f16(3, 10, 16, 2, 64)), dict(hot_k=f16(3 * 9 * 16 * 128 - 1), hot_blocks=9)], ids=lambda d: None)
def test_pools_of_other_pages_are_refused(on_cpu, kw):
    rows = f16(3, 6, 2, 64)
    refused(accept_of, **{**dict(k=rows, v=rows, hot_v=kw["hot_k"], hot_blocks=None), **kw})


def tree_of(rows=6, **kw):
    return O.make_tree_desc(**{**dict(batch=2, num_tokens=rows, q_heads=4, kv_heads=2, head_dim=64, q=f16(rows, 4, 64), k=f16(rows, 2, 64),
                                      v=f16(rows, 2, 64), out=f16(rows, 4, 64)), **kw})


def test_tree_rows_of_other_heads_are_refused(on_cpu):
    """A whole fused row, or a pool of other heads, where its part is asked for: no flat memory of the request's rows."""
    for kw in (dict(q=f16(6, 8, 64)), dict(k=f16(6, 4, 64)), dict(v=f16(6, 3, 64)), dict(out=f16(6, 512)),
               dict(hot_k=f16(9, 16, 4, 64), hot_v=A["hot_v"]), dict(hot_k=A["hot_k"], hot_v=f16(9, 16, 1, 128), hot_blocks=9)):
        refused(tree_of, **kw)
    for kw in (dict(q=f16(6, 256), k=f16(8, 128)), dict(q=f16(6, 2, 64, 2, 2)), dict(q=f16(6 * 256), out=f16(2, 3, 4, 64)), dict(k=f16(6, 8, 64)[:, 4:6]),
               dict(hot_k=f16(9, 16, 2, 64), hot_v=f16(3, 3, 16, 2, 64)), dict(rows=0, q=f16(0, 8, 64)), dict(q=f16(1, 6, 4, 64))):
        assert tree_of(**kw).q_stride == 256
    one = dict(kv_heads=1, q_heads=4)
    assert tree_of(**one, k=f16(6, 1, 64), v=f16(6, 64)).k_stride == 64


def test_tree_plan_of_equal_parts():
    """Rows that the sequences share equally are counted as that, not as if each had all of them."""
    none = dict(tree_mask=0, mask_words=0, hot_count=0, refs=0, seq_held=0, hot_k=0, hot_v=0, q_heads=32, kv_heads=8)
    p = O.tree_plan(tree(batch=1 << 18, num_tokens=1 << 18, token_offsets=0, **none))
    assert p.work_groups
    with pytest.raises(WeaverError) as e:  # offsets that the device alone knows
        O.tree_plan(tree(batch=1 << 18, num_tokens=1 << 18, **none))
    assert e.value.status == AW_E_UNSUPPORTED
    few = dict(batch=64, num_tokens=512, tree_mask=0, mask_words=0, q_heads=8, kv_heads=2)  # 8 nodes each behind up to 48 tokens
    assert O.tree_plan(tree(**few, token_offsets=0)).workspace_bytes == 0


def test_pools_whose_layers_lie_between_each_other():
    """K and V of a layer side by side in one buffer: no element of one is the other's."""
    layer = 50 * 16 * 128
    assert check(accept(hot_layer_stride=2 * layer, hot_v=A["hot_k"] + 2 * layer)) == (0, "")
    assert check(accept(hot_layer_stride=3 * layer, hot_v=A["hot_k"] + 4 * layer)) == (0, "")
    for kw in (dict(hot_v=A["hot_k"]), dict(hot_v=A["hot_k"] + 2 * layer - 2), dict(hot_v=A["hot_k"] + 2 * layer + 2), dict(hot_v=A["hot_k"] + 4 * layer),
               dict(hot_v=A["hot_k"] + 2 * layer, path=A["hot_k"] + 2 * layer), dict(hot_v=A["hot_k"] + 2 * layer, k=A["hot_k"] + 6 * layer)):
        rc, msg = check(accept(hot_layer_stride=2 * layer, **kw))
        assert rc == AW_E_INVALID_ARG and "overlap" in msg


def test_pools_in_one_buffer(on_cpu):
    rows, both = f16(3, 6, 2, 64), f16(3, 2, 9, 16, 2, 64)
    d = accept_of(k=rows, v=rows, hot_k=both[:, 0], hot_v=both[:, 1], hot_blocks=None)
    assert (d.hot_blocks, d.hot_layer_stride) == (9, 2 * 9 * 16 * 128)
    d = accept_of(k=rows, v=rows, hot_k=both[:, 0, :5], hot_v=both[:, 1, :5], hot_blocks=None)
    assert (d.hot_blocks, d.hot_layer_stride) == (5, 2 * 9 * 16 * 128)
    for pool in (both[:, 0, ::2], both[:1, 0].expand(3, 9, 16, 2, 64), f16(3, 9, 16, 2, 128)[..., ::2], f16(3, 9, 32, 2, 64)[:, :, ::2]):
        refused(accept_of, k=rows, v=rows, hot_k=pool, hot_v=pool, hot_blocks=None)


def test_steps_of_no_rows_take_empty_tensors(on_cpu):
    """A batch without a new token, whose tensors of no elements have no address."""
    d = O.make_tables_desc(batch=2, num_tokens=0, seq_held=i32(2), seq_new=i32(2), refs=i32(2, 3), seq_hot=i32(2), token_offsets=i32(3),
                           parents=i32(0), tree_mask=i32(0, 2), slots=torch.zeros(0, dtype=torch.int64), positions=i32(0))
    assert check(d) == (0, "")
    d = O.make_tree_desc(batch=2, num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, q=f16(0, 4, 64), k=f16(0, 2, 64), v=f16(0, 2, 64),
                         out=f16(0, 4, 64), token_offsets=i32(3), tree_mask=i32(0, 2))
    O.tree_plan(d)
    none = dict(rows=0, logits=torch.zeros(0, 1000), best=i32(0), out=torch.zeros(0, 1000), batch=2, token_offsets=i32(3))
    assert check(logits_of(**none)) == (0, "")
    assert check(logits_of(**none, node_tokens=i32(0), tree_mask=i32(0, 2), allowed=i32(3, 32), allowed_index=i32(0))) == (0, "")
    own = {n: i32(2) for n in ("seq_held", "accepted", "next_token", "seq_hot")}
    d = O.make_accept_desc(batch=2, num_tokens=0, layers=3, kv_heads=2, head_dim=64, parents=i32(0), node_tokens=i32(0), targets=i32(0), path=i32(0),
                           token_offsets=i32(3), slots=torch.zeros(0, dtype=torch.int64), k=torch.empty_strided((3, 0, 2, 64), (0, 0, 0, 0), dtype=torch.float16), v=f16(3, 0, 2, 64),
                           hot_k=f16(3, 9, 16, 2, 64), hot_v=f16(3, 9, 16, 2, 64), **own)
    assert check(d) == (0, "")


def test_lists_of_no_entries_take_empty_tensors(on_cpu):
    """No history, biases or grammar states yet: the counts beside them and an index of -1 stay."""
    own = dict(batch=2, token_offsets=i32(3))
    assert check(logits_of(**own, history=i32(2, 0), history_count=i32(2), prompt_count=i32(2))) == (0, "")
    assert check(logits_of(**own, bias_ids=i32(2, 0), bias_values=torch.zeros(2, 0), bias_count=i32(2))) == (0, "")
    assert check(logits_of(**own, allowed=i32(0, 32), allowed_index=i32(3))) == (0, "")
    assert "allowed" in refused(logits_of, **own, allowed=i32(0, 32))
