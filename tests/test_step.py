"""A step over trees of drafted tokens without a GPU: the descriptors' layouts, what the host refuses, the attention's plan."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from aether_nexus_amd import _lib
from aether_nexus_amd import ops as O
from aether_nexus_amd.types import (AW_E_ALIGN, AW_E_INVALID_ARG, AW_E_UNSUPPORTED, AcceptDesc, LogitsDesc, TablesDesc, TreeDesc,
                                    TreePlanInfo)
from aether_nexus_amd.weaver import WeaverError

NAMES = ("seq_held seq_new seq_pages free_pages free_first parents refs seq_hot pages_out token_offsets free_next slots positions "
         "tree_mask logits out best history history_count prompt_count repetition frequency presence node_tokens bias_ids "
         "bias_values bias_count allowed allowed_index targets k v hot_k hot_v accepted next_token path history_count_out q").split()
A = {n: (i + 1) << 38 for i, n in enumerate(NAMES)}


def fill(cls, numbers, **kw):
    d = cls(**numbers)
    for n, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(d, n, A[n])
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def tables(**kw):
    return fill(TablesDesc, dict(batch=4, num_tokens=100, hot_count=9, refs_stride=10, free_count=50, mask_words=1), **kw)


def logits(**kw):
    return fill(LogitsDesc, dict(num_tokens=12, vocab_size=1000, batch=4, mask_words=1, history_stride=64, bias_stride=8, allowed_rows=5), **kw)


def accept(**kw):
    return fill(AcceptDesc, dict(batch=4, num_tokens=20, layers=3, kv_heads=2, head_dim=64, history_stride=100, hot_blocks=50), **kw)


def tree(**kw):
    return fill(TreeDesc, dict(batch=4, num_tokens=20, q_heads=8, kv_heads=2, head_dim=128, hot_count=3, refs_stride=4, mask_words=1,
                               scale=0.1, hot_blocks=50), **kw)


def check(d):
    name = {TablesDesc: "tables", LogitsDesc: "logits", AcceptDesc: "accept"}[type(d)]
    msg = ctypes.create_string_buffer(256)
    rc = getattr(_lib.load(), f"aw_ops_check_{name}")(ctypes.byref(d), msg, 256)
    return rc, msg.value.decode()


def test_struct_sizes_match():
    sizes = (ctypes.c_size_t * 3)()
    _lib.load().aw_abi_step_desc_sizes(sizes)
    assert tuple(sizes) == tuple(map(ctypes.sizeof, (TablesDesc, LogitsDesc, AcceptDesc)))
    sizes = (ctypes.c_size_t * 2)()
    _lib.load().aw_abi_tree_sizes(sizes)
    assert tuple(sizes) == (ctypes.sizeof(TreeDesc), ctypes.sizeof(TreePlanInfo))


def test_null_descriptors():
    for name in ("tables", "logits", "accept"):
        assert getattr(_lib.load(), f"aw_ops_check_{name}")(None, None, 0) == AW_E_INVALID_ARG
    assert _lib.load().aw_tree_plan(None, 0, None, None, 0) == AW_E_INVALID_ARG


# ---------------------------------------------------------------- accepted

@pytest.mark.parametrize("d", [
    tables(), tables(parents=0, mask_words=0, tree_mask=0), tables(seq_pages=0, free_first=0, pages_out=0, free_next=0, slots=0, positions=0),
    tables(batch=0), tables(num_tokens=0), tables(free_count=0, free_pages=0), tables(hot_count=0, refs_stride=0, refs=0),
    tables(refs=A["refs"], refs_stride=9), tables(mask_words=32), tables(token_offsets=A["seq_hot"] + 16)], ids=lambda d: None)
def test_tables_accepted(d):
    assert check(d) == (0, "")


@pytest.mark.parametrize("d", [
    logits(), logits(flags=1), logits(out=A["logits"]), logits(out=0), logits(best=0), logits(history=0, history_count=0, prompt_count=0),
    logits(node_tokens=0, tree_mask=0, mask_words=0), logits(bias_ids=0, bias_values=0, bias_count=0, bias_stride=0),
    logits(allowed=0, allowed_index=0, allowed_rows=0), logits(allowed_index=0, allowed_rows=12), logits(token_offsets=0),
    logits(num_tokens=0), logits(logits_stride=1003, out_stride=1001),
    logits(flags=1, logits=A["logits"] + 2, out=A["out"] + 6)], ids=lambda d: None)
def test_logits_accepted(d):
    assert check(d) == (0, "")


@pytest.mark.parametrize("d", [
    accept(), accept(v=0, hot_v=0), accept(layers=0, k=0, v=0, hot_k=0, hot_v=0, slots=0), accept(history=0, history_count=0, history_count_out=0),
    accept(seq_hot=A["seq_held"]), accept(history_count_out=A["history_count"]), accept(batch=0), accept(token_offsets=0),
    accept(k_stride=4 * 128, v_stride=4 * 128, v=A["k"] + 2 * 128), accept(hot_layer_stride=1 << 30)], ids=lambda d: None)
def test_accept_accepted(d):
    assert check(d) == (0, "")


@pytest.mark.parametrize("kw", [
    dict(), dict(v=0, hot_v=0), dict(tree_mask=0, mask_words=0), dict(token_offsets=0), dict(hot_count=0, refs=0, seq_held=0, hot_k=0, hot_v=0),
    dict(num_tokens=0), dict(out=A["q"]), dict(q_stride=1024 + 512, k_stride=1536, v_stride=1536, k=A["q"] + 2 * 1024, v=A["q"] + 2 * 1280),
    dict(scale=0.0), dict(scale=-1.0), dict(head_dim=64), dict(hot_blocks=1 << 31, hot_v=1 << 50), dict(batch=1 << 20, num_tokens=1 << 20),
    dict(mask_words=32), dict(q_heads=2 * 70)])
@pytest.mark.parametrize("cus", [0, 1, 64, 304])
def test_tree_accepted(kw, cus):
    p = O.tree_plan(tree(**kw), cus)
    assert p.workspace_bytes <= 160 << 20


# ---------------------------------------------------------------- refused

@pytest.mark.parametrize("kw,word", [
    (dict(refs_stride=8), "refs_stride"), (dict(parents=0), "go together"), (dict(tree_mask=0), "go together"), (dict(mask_words=0), "go together"),
    (dict(seq_held=0), "null"), (dict(seq_new=0), "null"), (dict(refs=0), "null"), (dict(seq_hot=0), "null"), (dict(token_offsets=0), "null"),
    (dict(free_pages=0), "null"), (dict(seq_hot=A["seq_held"]), "overlap"), (dict(seq_hot=A["seq_held"] + 12), "overlap"),
    (dict(pages_out=A["seq_pages"]), "overlap"), (dict(free_next=A["free_first"]), "overlap"), (dict(slots=A["positions"] + 396), "overlap"),
    (dict(refs=A["free_pages"] - 4 * 38), "overlap"), (dict(tree_mask=A["parents"]), "overlap"), (dict(token_offsets=A["seq_hot"] + 12), "overlap")])
def test_tables_refused(kw, word):
    rc, msg = check(tables(**kw))
    assert rc == AW_E_INVALID_ARG and word in msg and msg.startswith("page_tables"), msg


@pytest.mark.parametrize("kw,word", [
    (dict(flags=2), "flags"), (dict(vocab_size=0), "vocab_size"), (dict(out=0, best=0), "neither"), (dict(logits=0), "null"),
    (dict(batch=0), "batch"), (dict(history_count=0), "history_count"), (dict(history=0), "prompt_count"), (dict(tree_mask=0), "go together"),
    (dict(node_tokens=0), "go together"), (dict(mask_words=0), "go together"), (dict(bias_values=0), "go together"), (dict(bias_ids=0), "go together"),
    (dict(allowed=0), "allowed"), (dict(allowed_index=0), "fewer"), (dict(logits_stride=999), "stride"), (dict(out_stride=999), "stride"),
    (dict(allowed_stride=31), "stride"), (dict(num_tokens=13, token_offsets=0), "token_offsets"), (dict(out=A["logits"], out_stride=1004), "overlap"),
    (dict(out=A["logits"] + 4), "overlap"), (dict(best=A["logits"] + 4 * 11999), "overlap"), (dict(best=A["out"]), "overlap"),
    (dict(out=A["allowed"]), "overlap"), (dict(best=A["history"] + 4 * 255), "overlap")])
def test_logits_refused(kw, word):
    rc, msg = check(logits(**kw))
    assert rc == AW_E_INVALID_ARG and word in msg and msg.startswith("adjust_logits"), msg


@pytest.mark.parametrize("kw,word", [
    (dict(seq_held=0), "null"), (dict(accepted=0), "null"), (dict(next_token=0), "null"), (dict(seq_hot=0), "null"), (dict(parents=0), "null"),
    (dict(node_tokens=0), "null"), (dict(targets=0), "null"), (dict(path=0), "null"), (dict(history=0), "go together"),
    (dict(history_count=0), "go together"), (dict(k=0), "null"), (dict(hot_k=0), "null"), (dict(slots=0), "null"), (dict(v=0), "go together"),
    (dict(hot_v=0), "go together"), (dict(kv_heads=0), "kv_heads"), (dict(head_dim=0), "head_dim"), (dict(hot_blocks=0), "hot_blocks"),
    (dict(hot_blocks=(1 << 31) + 1), "2^31"), (dict(k_stride=127), "stride"), (dict(hot_layer_stride=50 * 16 * 128 - 1), "stride"),
    (dict(num_tokens=21, token_offsets=0), "token_offsets"), (dict(hot_v=A["hot_k"]), "overlap"), (dict(hot_k=A["k"] - 64), "overlap"),
    (dict(hot_v=A["v"] + 2), "overlap"), (dict(seq_hot=A["seq_held"] + 4), "overlap"), (dict(history_count_out=A["history_count"] + 4), "overlap"),
    (dict(accepted=A["seq_held"]), "overlap"), (dict(accepted=A["seq_held"], seq_hot=A["seq_held"]), "overlap"), (dict(path=A["targets"]), "overlap"),
    (dict(next_token=A["seq_held"], seq_hot=A["seq_held"] + 64), "overlap"), (dict(history=A["slots"]), "overlap")])
def test_accept_refused(kw, word):
    rc, msg = check(accept(**kw))
    assert rc == AW_E_INVALID_ARG and word in msg and msg.startswith("accept_tree"), msg


@pytest.mark.parametrize("d", [
    tables(batch=(1 << 20) + 1), tables(num_tokens=(1 << 24) + 1), tables(hot_count=(1 << 26) + 1, refs_stride=1 << 27), tables(free_count=(1 << 30) + 1),
    tables(mask_words=33), logits(num_tokens=(1 << 24) + 1, token_offsets=0), logits(vocab_size=(1 << 24) + 1), logits(history_stride=(1 << 20) + 1),
    logits(bias_stride=1024), logits(mask_words=33), logits(batch=(1 << 20) + 1), logits(logits_stride=(1 << 30) + 1), accept(layers=65536),
    accept(batch=(1 << 20) + 1), accept(num_tokens=(1 << 24) + 1), accept(kv_heads=1 << 20, head_dim=2), accept(history_stride=(1 << 30) + 1),
    accept(k_stride=(1 << 30) + 1)], ids=lambda d: None)
def test_unsupported(d):
    assert check(d)[0] == AW_E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(logits=A["logits"] + 2), dict(out=A["out"] + 2), dict(flags=1, logits=A["logits"] + 1)])
def test_logits_misaligned(kw):
    assert check(logits(**kw))[0] == AW_E_ALIGN


@pytest.mark.parametrize("kw", [
    dict(reserved=1), dict(batch=0), dict(kv_heads=0), dict(q_heads=7), dict(q_heads=0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=3e38),
    dict(refs_stride=2), dict(tree_mask=0), dict(mask_words=0), dict(num_tokens=21, token_offsets=0), dict(q=0), dict(k=0), dict(out=0), dict(refs=0),
    dict(seq_held=0), dict(hot_k=0), dict(hot_blocks=0), dict(hot_v=0), dict(v=0), dict(hot_blocks=(1 << 31) + 1), dict(q_stride=1016),
    dict(k_stride=248), dict(out_stride=1020), dict(out=A["q"] + 16), dict(out=A["q"], out_stride=2048), dict(out=A["k"]), dict(out=A["v"] - 64),
    dict(out=A["hot_k"] + 64), dict(out=A["hot_v"] - 64), dict(out=A["refs"] + 8), dict(out=A["tree_mask"]), dict(out=A["seq_held"] - 1024)])
def test_tree_invalid(kw):
    with pytest.raises(WeaverError) as e:
        O.tree_plan(tree(**kw))
    assert e.value.status == AW_E_INVALID_ARG and "tree_attention" in str(e.value)


@pytest.mark.parametrize("kw", [
    dict(head_dim=96), dict(hot_count=(1 << 18) + 1, refs_stride=1 << 19), dict(kv_heads=1024, q_heads=1024), dict(num_tokens=1 << 23),
    dict(batch=(1 << 20) + 1), dict(mask_words=33), dict(q_stride=(1 << 30) + 8), dict(num_tokens=(1 << 24) + 1, q_heads=2),
    dict(num_tokens=1 << 20, hot_count=1 << 16, refs_stride=1 << 16)])
def test_tree_unsupported(kw):
    with pytest.raises(WeaverError) as e:
        O.tree_plan(tree(**kw))
    assert e.value.status == AW_E_UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(q=A["q"] + 8), dict(k=A["k"] + 2), dict(v=A["v"] + 8), dict(hot_k=A["hot_k"] + 8), dict(hot_v=A["hot_v"] + 2), dict(out=A["out"] + 4),
    dict(q_stride=1028), dict(k_stride=260), dict(v_stride=257), dict(out_stride=1026)])
def test_tree_misaligned(kw):
    with pytest.raises(WeaverError) as e:
        O.tree_plan(tree(**kw))
    assert e.value.status == AW_E_ALIGN


# ---------------------------------------------------------------- from Python

def test_descriptors_take_gpu_tensors_only():
    t = torch.zeros(8, dtype=torch.int32)
    raw = {n: A[n] for n in ("seq_held", "seq_new", "refs", "seq_hot", "token_offsets")}
    for kw in (dict(seq_held=t), dict(slots=t.long()), dict(free_pages=t, free_count=8)):
        with pytest.raises(WeaverError) as e:
            O.make_tables_desc(batch=2, num_tokens=3, hot_count=2, **{**raw, **kw})
        assert "GPU" in str(e.value)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(WeaverError) as e:
        O.make_tree_desc(batch=1, num_tokens=3, q_heads=4, kv_heads=2, head_dim=64, q=q, k=A["k"], out=A["out"])
    assert "GPU" in str(e.value)
    with pytest.raises(WeaverError) as e:
        O.make_logits_desc(num_tokens=3, vocab_size=8, logits=torch.zeros(3, 8), out=A["out"])
    assert "GPU" in str(e.value)
    with pytest.raises(WeaverError) as e:
        O.make_accept_desc(batch=1, num_tokens=8, parents=t, **{n: A[n] for n in ("node_tokens", "targets", "seq_held", "accepted", "next_token",
                                                                                  "seq_hot", "path")})
    assert "GPU" in str(e.value)


def test_lengths_of_raw_pointers_are_required():
    raw = {n: A[n] for n in ("seq_held", "seq_new", "refs", "seq_hot", "token_offsets")}
    for make, kw, word in (
            (O.make_tables_desc, dict(batch=2, num_tokens=3, **raw), "hot_count"),
            (O.make_tables_desc, dict(batch=2, num_tokens=3, hot_count=1, free_pages=A["free_pages"], **raw), "free_count"),
            (O.make_tables_desc, dict(batch=2, num_tokens=3, hot_count=1, parents=A["parents"], tree_mask=A["tree_mask"], **raw), "row length"),
            (O.make_tree_desc, dict(batch=1, num_tokens=3, q_heads=4, kv_heads=2, head_dim=64, q=A["q"], k=A["k"], out=A["out"], refs=A["refs"]), "hot_count"),
            (O.make_tree_desc, dict(batch=1, num_tokens=3, q_heads=4, kv_heads=2, head_dim=64, q=A["q"], k=A["k"], out=A["out"], hot_k=A["hot_k"]), "hot_blocks"),
            (O.make_logits_desc, dict(num_tokens=3, vocab_size=8, logits=A["logits"], out=A["out"], allowed=A["allowed"]), "allowed_rows"),
            (O.make_logits_desc, dict(num_tokens=3, vocab_size=8, logits=A["logits"], out=A["out"], history=A["history"], batch=3), "row length")):
        with pytest.raises(WeaverError) as e:
            make(**kw)
        assert e.value.status == AW_E_INVALID_ARG and word in str(e.value)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(num_tokens=-1), dict(hot_count=1 << 32), dict(free_count=-1, free_pages=A["free_pages"]),
                                dict(mask_words=-1, tree_mask=A["tree_mask"])])
def test_numbers_that_do_not_fit_are_refused(kw):
    raw = {n: A[n] for n in ("seq_held", "seq_new", "refs", "seq_hot", "token_offsets")}
    with pytest.raises(WeaverError) as e:
        O.make_tables_desc(**{**dict(batch=2, num_tokens=3, hot_count=1, **raw), **kw})
    assert e.value.status == AW_E_INVALID_ARG and "within" in str(e.value)


def test_raw_descriptors_are_those_of_the_header():
    d = O.make_tree_desc(batch=2, num_tokens=6, q_heads=4, kv_heads=2, head_dim=64, q=A["q"], k=A["k"], v=A["v"], out=A["out"], hot_k=A["hot_k"],
                         hot_v=A["hot_v"], hot_blocks=9, refs=A["refs"], hot_count=3, refs_stride=5, seq_held=A["seq_held"])
    assert (d.scale, d.refs_stride, d.q_stride, d.k_stride) == (0.125, 5, 256, 128)
    O.tree_plan(d)
    raw = {n: A[n] for n in ("parents", "node_tokens", "targets", "seq_held", "accepted", "next_token", "seq_hot", "path")}
    assert check(O.make_accept_desc(batch=2, num_tokens=6, **raw)) == (0, "")
