"""Rotary positions, head norms and paged appends without a GPU: the frequencies,
the descriptors' layouts, and every call that the host refuses (through the host
checks of the C ABI, which the calls themselves make)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from aether_nexus_amd import _lib
from aether_nexus_amd import ops as O
from aether_nexus_amd.types import AW_E_INVALID_ARG, AW_E_UNSUPPORTED, AppendDesc, RotaryDesc, RotaryScaling
from aether_nexus_amd.weaver import WeaverError


def test_struct_sizes_match():
    sizes = (ctypes.c_size_t * 3)()
    _lib.load().aw_abi_ops_desc_sizes(sizes)
    assert tuple(sizes) == tuple(ctypes.sizeof(t) for t in (RotaryScaling, RotaryDesc, AppendDesc))


@pytest.mark.parametrize("n,theta", [(2, 10000.0), (20, 10000.0), (64, 500000.0), (128, 1e6)])
def test_frequencies(n, theta):
    """pow in double is within 2 ulp of the value in either library; 8 leave room for the few operations around it."""
    tol = 8 * 2.0 ** -52
    base = np.array([theta ** (-2.0 * p / n) for p in range(n // 2)])
    np.testing.assert_allclose(O.rotary_frequencies(n, theta), base, rtol=tol)
    np.testing.assert_allclose(O.rotary_frequencies(n, theta, "linear", 4.0), base / 4.0, rtol=tol)
    if n > 2:
        # theta's own rounding is raised to a power of at most 1
        ntk = np.array([(theta * 8.0 ** (n / (n - 2))) ** (-2.0 * p / n) for p in range(n // 2)])
        np.testing.assert_allclose(O.rotary_frequencies(n, theta, "ntk", 8.0), ntk, rtol=tol)
    got = O.rotary_frequencies(n, theta, "parts", 8.0, original_length=4096.0, low=1.0, high=4.0)
    for p, f in enumerate(base):
        turns = 4096.0 * f / (2 * math.pi)
        if turns >= 4.0 * (1 + 1e-9):
            assert abs(got[p] - f) <= tol * f
        elif turns <= 1.0 * (1 - 1e-9):
            assert abs(got[p] - f / 8.0) <= tol * f / 8.0
        else:
            g = (turns - 1.0) / 3.0
            # g's error is about 4 ulp of turns over 3, times f
            assert abs(got[p] - ((1 - g) * f / 8.0 + g * f)) <= 4 * tol * f
    assert got[0] == 1.0  # many turns: kept


def test_ntk_keeps_the_fastest_pair_and_stretches_the_slowest():
    n, factor = 64, 16.0
    base, got = O.rotary_frequencies(n, 10000.0), O.rotary_frequencies(n, 10000.0, "ntk", factor)
    assert got[0] == base[0] == 1.0
    assert abs(got[-1] - base[-1] / factor) <= 1e-12 * base[-1]


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(theta=0.0), dict(theta=-1.0), dict(theta=math.inf),
                                dict(theta=math.nan), dict(scaling="linear", factor=0.0), dict(scaling="linear", factor=math.nan),
                                dict(scaling="ntk", rotary_dim=2, factor=2.0), dict(scaling="parts", factor=2.0),
                                dict(scaling="parts", factor=2.0, original_length=4096.0, low=4.0, high=4.0),
                                dict(scaling="parts", factor=2.0, original_length=4096.0, low=-1.0), dict(scaling="other")])
def test_frequencies_refused(kw):
    with pytest.raises(WeaverError) as e:
        O.rotary_frequencies(**{"rotary_dim": 64, "theta": 10000.0, **kw})
    assert e.value.status == AW_E_INVALID_ARG


def test_rotary_takes_given_frequencies():
    r = O.Rotary(8, inv_freq=[1.0, 0.5, 0.25, 0.0], interleaved=True, magnitude=1.5, device="cpu")
    assert r.inv_freq.dtype == torch.float64 and r.inv_freq.tolist() == [1.0, 0.5, 0.25, 0.0]
    assert (r.rotary_dim, r.interleaved, r.magnitude) == (8, True, 1.5)
    for dim, f in ((8, [1.0]), (3, [1.0]), (0, [])):
        with pytest.raises(WeaverError):
            O.Rotary(dim, inv_freq=f, device="cpu")


# Addresses of buffers that no refused call touches: 1 MiB apart.
A = {n: 0x100000 * (i + 1) for i, n in enumerate(("q", "k", "v", "q_out", "k_out", "w", "freq", "hot_k", "hot_v", "refs", "seq", "off"))}


def rows(**kw):
    d = RotaryDesc(num_tokens=5, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64, layout=0, magnitude=1.0, eps=1e-5,
                   q=A["q"], k=A["k"], q_out=A["q_out"], k_out=A["k_out"], inv_freq=A["freq"])
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def check_rows(d, norms=0):
    msg = ctypes.create_string_buffer(256)
    rc = _lib.load().aw_ops_check_rotary(None if d is None else ctypes.byref(d), norms, msg, 256)
    return rc, msg.value.decode()


def test_rows_accepted():
    for kw in ({}, dict(rotary_dim=2), dict(layout=1), dict(q_heads=0, q=0, q_out=0), dict(kv_heads=0, k=0, k_out=0),
               dict(q_out=A["q"], k_out=A["k"]), dict(q_stride=1000, q_out_stride=257), dict(num_tokens=0),
               dict(q_out=A["q"] + 2 * 256, num_tokens=1), dict(head_dim=1024, rotary_dim=1024, num_tokens=1)):
        assert check_rows(rows(**kw))[0] == 0, (kw, check_rows(rows(**kw)))
    n = dict(q_norm=A["w"], k_norm=A["w"])
    assert check_rows(rows(**n), 1)[0] == 0
    assert check_rows(rows(**n, rotary_dim=0, inv_freq=0, magnitude=math.nan), 1)[0] == 0  # norms alone


@pytest.mark.parametrize("kw,word", [
    (dict(head_dim=0), "head_dim"), (dict(rotary_dim=63), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(layout=2), "layout"), (dict(inv_freq=0), "inv_freq"),
    (dict(magnitude=math.inf), "magnitude"), (dict(magnitude=math.nan), "magnitude"), (dict(reserved=1), "reserved"),
    (dict(q=0), "null"), (dict(k=0), "null"), (dict(q_out=0), "null"), (dict(k_out=0), "null"),
    (dict(q_stride=255), "stride"), (dict(k_stride=127), "stride"), (dict(q_out_stride=255), "stride"),
    (dict(k_out_stride=1), "stride"), (dict(q_norm=A["w"]), "norm"), (dict(k_norm=A["w"]), "norm"),
    (dict(q_out=A["q"] + 2), "overlaps"), (dict(q_out=A["q"], q_stride=512), "overlaps"),
    (dict(k_out=A["k"] + 2 * (4 * 128 + 127)), "overlaps"), (dict(k=A["k"] + 2 * 639, k_out=A["k"]), "overlaps"),
    (dict(k_out=A["q"] + 2 * 500), "overlap"), (dict(q_out=A["k"] + 2 * 100), "overlap"), (dict(k_out=A["q_out"]), "overlap"),
    (dict(q=A["q"], k=A["q"] + 2 * 255, q_out=A["q"], k_out=A["k_out"], q_stride=500, k_stride=500, q_out_stride=500), "overlap"),
])
def test_rows_refused(kw, word):
    rc, msg = check_rows(rows(**kw))
    assert rc == AW_E_INVALID_ARG and word in msg, msg


def test_no_tokens_need_no_rows():
    """An empty tensor's address is null."""
    assert check_rows(rows(num_tokens=0, q=0, k=0, q_out=0, k_out=0))[0] == 0
    assert check_append(append(dict(num_tokens=0, q=0, k=0, q_out=0), v=0))[0] == 0
    assert check_append(append(dict(num_tokens=0, q=0, k=0, q_out=0), v=0, batch=0, refs=0, seq_hot=0, token_offsets=0))[0] == 0
    assert check_append(append(dict(num_tokens=0), hot_k=0))[0] == AW_E_INVALID_ARG


def test_parts_of_one_buffer_are_accepted():
    """q, k and both outputs side by side in rows of one buffer: no element twice."""
    part = dict(q=A["q"], k=A["q"] + 2 * 256, q_out=A["q"] + 2 * 384, k_out=A["q"] + 2 * 640,
                q_stride=768, k_stride=768, q_out_stride=768, k_out_stride=768)
    assert check_rows(rows(**part))[0] == 0, check_rows(rows(**part))
    assert check_rows(rows(**{**part, "q_out": part["q"], "k_out": part["k"]}))[0] == 0  # in place
    assert check_rows(rows(**{**part, "q_out": part["q_out"] + 2 * 768}))[0] == 0  # a row further
    for n, by in (("q_out", -2), ("k_out", -2), ("k_out", 2), ("k_out", 2 * 768 - 2), ("k_out", 2 * 768 + 2)):
        assert check_rows(rows(**{**part, n: part[n] + by}))[0] == AW_E_INVALID_ARG, (n, by)


def test_rows_unsupported():
    for kw in (dict(head_dim=1026), dict(num_tokens=1 << 31), dict(num_tokens=(1 << 24) + 1), dict(q_heads=1 << 16), dict(q_stride=(1 << 30) + 1)):
        assert check_rows(rows(**kw))[0] == AW_E_UNSUPPORTED, kw
    assert check_rows(None)[0] == AW_E_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(), dict(q_norm=A["w"]), dict(k_norm=A["w"]),
                                dict(q_norm=A["w"], k_norm=A["w"], eps=-1.0), dict(q_norm=A["w"], k_norm=A["w"], eps=math.nan)])
def test_norm_rows_refused(kw):
    assert check_rows(rows(**kw), 1)[0] == AW_E_INVALID_ARG


def append(rows_kw=None, **kw):
    d = AppendDesc(rows=rows(k_out=0, **(rows_kw or {})), batch=2, hot_count=3, refs_stride=4, hot_blocks=7, v=A["v"],
                   hot_k=A["hot_k"], hot_v=A["hot_v"], refs=A["refs"], seq_hot=A["seq"], token_offsets=A["off"])
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def check_append(d):
    msg = ctypes.create_string_buffer(256)
    rc = _lib.load().aw_ops_check_append(None if d is None else ctypes.byref(d), msg, 256)
    return rc, msg.value.decode()


def test_append_accepted():
    for d in (append(), append(dict(rotary_dim=0, inv_freq=0)), append(dict(q_heads=0, q=0, q_out=0)),
              append(v=0, hot_v=0), append(dict(num_tokens=6), token_offsets=0), append(batch=0),
              append(dict(k_norm=A["w"])), append(hot_blocks=1 << 31, hot_v=1 << 50)):
        assert check_append(d)[0] == 0, check_append(d)


@pytest.mark.parametrize("rows_kw,kw,word", [
    (dict(kv_heads=0), {}, "kv_heads"), (dict(q_norm=A["w"], eps=-1.0), {}, "eps"), (dict(rotary_dim=3), {}, "rotary_dim"),
    ({}, dict(reserved=1), "reserved"), ({}, dict(v=0), "null"), ({}, dict(hot_v=0), "hot_v"), ({}, dict(hot_k=0), "null"),
    ({}, dict(refs=0), "null"), ({}, dict(seq_hot=0), "null"), ({}, dict(hot_blocks=0), "hot_blocks"),
    ({}, dict(hot_blocks=(1 << 31) + 1), "hot_blocks"), ({}, dict(hot_count=0), "hot_count"),
    ({}, dict(refs_stride=2), "refs_stride"), ({}, dict(token_offsets=0), "token_offsets"), ({}, dict(v_stride=127), "stride"),
    ({}, dict(hot_v=A["hot_k"]), "overlap"), ({}, dict(hot_v=A["hot_k"] + 7 * 16 * 128 * 2 - 2), "overlap"),
    ({}, dict(hot_k=A["k"] - 2), "overlaps"), ({}, dict(hot_v=A["v"] + 2 * 639), "overlaps"), ({}, dict(hot_k=A["q_out"] - 64), "overlaps"),
    (dict(q_out=A["v"]), {}, "overlap"),
])
def test_append_refused(rows_kw, kw, word):
    rc, msg = check_append(append(rows_kw, **kw))
    assert rc == AW_E_INVALID_ARG and word in msg, msg


@pytest.mark.parametrize("batch", [(1 << 24) + 1, (1 << 32) - 63, (1 << 32) - 1])
def test_append_of_too_many_sequences(batch):
    """The search of the offsets counts them in 32 bits: a batch near 2^32 is refused, not searched."""
    rc, msg = check_append(append(batch=batch))
    assert rc == AW_E_UNSUPPORTED and "batch" in msg
    assert check_append(append(batch=1 << 24))[0] == 0


def test_append_refuses_k_out():
    d = append()
    d.rows.k_out = A["k_out"]
    assert check_append(d)[0] == AW_E_INVALID_ARG
    assert check_append(None)[0] == AW_E_INVALID_ARG


def test_descriptors_take_gpu_tensors_only():
    q = torch.zeros(5, 4, 64, dtype=torch.float16)
    with pytest.raises(WeaverError) as e:
        O.make_rotary_desc(num_tokens=5, q_heads=4, kv_heads=0, head_dim=64, rotary=None, q=q, k=None)
    assert e.value.status == AW_E_INVALID_ARG and "GPU" in str(e.value)
    with pytest.raises(WeaverError):  # q_heads without q
        O.make_append_desc(batch=1, num_tokens=5, q_heads=4, kv_heads=2, head_dim=64, k=A["k"], v=A["v"], hot_k=A["hot_k"],
                           hot_v=A["hot_v"], hot_blocks=4, hot_count=1, refs=A["refs"], seq_hot=A["seq"])
    with pytest.raises(WeaverError):  # hot_count unknown
        O.make_append_desc(batch=1, num_tokens=5, q_heads=0, kv_heads=2, head_dim=64, k=A["k"], v=A["v"], hot_k=A["hot_k"],
                           hot_v=A["hot_v"], hot_blocks=4, refs=A["refs"], seq_hot=A["seq"])
    d = O.make_append_desc(batch=1, num_tokens=5, q_heads=0, kv_heads=2, head_dim=64, k=A["k"], v=A["v"], hot_k=A["hot_k"],
                           hot_v=A["hot_v"], hot_blocks=4, hot_count=1, refs=A["refs"], seq_hot=A["seq"])
    assert check_append(d)[0] == 0


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(num_tokens=-5), dict(q_heads=-1), dict(start_position=-1),
                                dict(start_position=1 << 32), dict(hot_count=-1), dict(hot_blocks=-1), dict(refs_stride=-4)])
def test_numbers_that_do_not_fit_are_refused(kw):
    base = dict(batch=1, num_tokens=5, q_heads=0, kv_heads=2, head_dim=64, k=A["k"], v=A["v"], hot_k=A["hot_k"], hot_v=A["hot_v"],
                hot_blocks=4, hot_count=1, refs=A["refs"], seq_hot=A["seq"], token_offsets=A["off"], q=A["q"])
    with pytest.raises(WeaverError) as e:
        O.make_append_desc(**{**base, **kw})
    assert e.value.status == AW_E_INVALID_ARG and "within" in str(e.value)
