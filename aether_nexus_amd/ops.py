"""The dense transformer ops on the gfx950 library (include/aether_ops.h).

``OpsEngine`` mirrors the reference's ``Ops`` (nexus-core/src/ops.rs:21-462):
the same method names, argument order and meaning, over device tensors (or
raw device pointers) instead of Metal buffers.  Every call is asynchronous on a
HIP stream, torch's current stream by default: the reference's batch mode
(``begin_batch`` / ``end_batch``, ops.rs:88-101, one command buffer per
forward pass) is the stream itself, and ``end_batch`` waits for it.  With
tensors the wrapper also checks their dtype, device and element counts before
anything is enqueued (the C ABI takes raw pointers).

Beside them, without a counterpart in the reference, what a batch over pages needs:
``rotary``, ``qk_norm_rotary``, ``append_paged`` and ``shared_prefix_attention``, each
of a descriptor (``make_rotary_desc``, ``make_append_desc``, ``make_prefix_desc``) that
is checked once and may be used again.
"""
from __future__ import annotations

import ctypes
import sys
from typing import Optional

import numpy as np

from . import _lib
from .types import (AW_F_CAUSAL, BLOCK_SIZE, ROTARY_SCALINGS, AppendDesc, PrefixDesc, PrefixPlanInfo, RotaryDesc,
                    RotaryScaling)
from .weaver import WeaverEngine, WeaverError, _ptr, _stream

AW_E_INVALID_ARG = -1


def _check_tensor(t, need: int, what: str, dtypes) -> None:
    """Element count, dtype and device of a tensor argument (raw ints pass)."""
    if t is None or isinstance(t, int):
        return
    import torch
    if not isinstance(t, torch.Tensor):
        raise WeaverError(f"{what}: expected a device tensor or a device pointer", AW_E_INVALID_ARG)
    if t.device.type != "cuda":
        raise WeaverError(f"{what}: tensor is on {t.device}, not the GPU", AW_E_INVALID_ARG)
    if t.dtype not in dtypes:
        raise WeaverError(f"{what}: dtype {t.dtype} (want {' or '.join(map(str, dtypes))})", AW_E_INVALID_ARG)
    if not t.is_contiguous():
        raise WeaverError(f"{what}: tensor is not contiguous", AW_E_INVALID_ARG)
    if t.numel() < need:
        raise WeaverError(f"{what}: {t.numel()} elements, the call reads or writes {need}", AW_E_INVALID_ARG)


def _checker(*names):
    """check(t, need, what) of tensors of the named torch dtypes: one expression for
    a tensor that passes (about 0.4 us of every call's host time), _check_tensor
    for everything else.  torch is looked up at the first tensor, not at import."""
    tensor, dtypes = None, ()

    def check(t, need, what):
        nonlocal tensor, dtypes
        if t.__class__ is tensor and t.is_cuda and t.dtype in dtypes and t.is_contiguous() and t.numel() >= need:
            return
        if tensor is None and t is not None and not isinstance(t, int):
            import torch
            dtypes = tuple(getattr(torch, n) for n in names)
            tensor = torch.Tensor  # last: another thread that sees it sees the dtypes
        _check_tensor(t, need, what, dtypes)
    return check


_f16 = _checker("float16", "int16")  # f16 values or their bit patterns
_f32 = _checker("float32")
_u32 = _checker("int32")
_f64 = _checker("float64")


def _counts(**values) -> None:
    """Numbers that a descriptor holds in 32 unsigned bits."""
    for name, v in values.items():
        if not 0 <= v < 2 ** 32:
            raise WeaverError(f"{name} {v} is not within [0, 2^32)", AW_E_INVALID_ARG)


def _token_rows(t, tokens: int, heads: int, head_dim: int, what: str) -> int:
    """Token stride (elements) of rows [tokens][heads][head_dim]: a contiguous tensor, a
    raw pointer to one, or a view with contiguous heads whose rows lie further apart
    (the q, k or v part of a fused product's output)."""
    row = heads * head_dim
    if t is None or isinstance(t, int) or not hasattr(t, "is_contiguous") or t.is_contiguous():
        _f16(t, tokens * row, what)
        return row
    inner = ((heads, head_dim), (head_dim, 1)) if t.dim() == 3 else ((row,), (1,))
    if t.dim() not in (2, 3) or tuple(t.shape[1:]) != inner[0] or t.shape[0] < tokens or \
            any(n > 1 and s != w for n, s, w in zip(inner[0], t.stride()[1:], inner[1])) or t.stride(0) < row:
        raise WeaverError(f"{what}: a view must be [tokens][{heads}][{head_dim}] (or flat rows) with contiguous heads "
                          f"and rows apart, got shape {tuple(t.shape)}, strides {tuple(t.stride())}", AW_E_INVALID_ARG)
    _f16(t[:0].contiguous(), 0, what)  # dtype and device
    return t.stride(0)


def _one_device(desc, tensors) -> None:
    """Records the tensors' GPU in the descriptor (raw pointers have none); the call compares it with the engine's."""
    where = {t.device.index for t in tensors if hasattr(t, "device")}
    if len(where) > 1:
        raise WeaverError(f"tensors on several GPUs: {sorted(where)}", AW_E_INVALID_ARG)
    desc._device = where.pop() if where else None
    desc._keep = tensors


def rotary_frequencies(rotary_dim: int, theta: float, scaling: str = "none", factor: float = 1.0,
                       original_length: float = 0.0, low: float = 1.0, high: float = 32.0, lib_path=None) -> np.ndarray:
    """The rotary_dim / 2 frequencies (radians per position, float64) of aw_rotary_frequencies:
    theta^(-2p / rotary_dim), scaled for contexts longer than a model was trained on.
    ``scaling``: "none"; "linear" (divided by ``factor``); "ntk" (theta raised by
    factor^(d / (d - 2))); "parts" (pairs that turn more than ``high`` times over
    ``original_length`` kept, fewer than ``low`` times divided, a ramp over the turns between; for a
    ramp over the pair's index pass ``Rotary`` an ``inv_freq`` of its own).  No GPU needed."""
    if scaling not in ROTARY_SCALINGS:
        raise WeaverError(f"rotary scaling {scaling!r} (one of {', '.join(ROTARY_SCALINGS)})", AW_E_INVALID_ARG)
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim >= 2 ** 32:
        raise WeaverError(f"rotary_dim {rotary_dim} must be even and at least 2", AW_E_INVALID_ARG)
    out = np.empty(rotary_dim // 2, dtype=np.float64)
    s = RotaryScaling(rotary_dim, ROTARY_SCALINGS[scaling], theta, factor, original_length, low, high)
    if _lib.load(lib_path).aw_rotary_frequencies(ctypes.byref(s), out.ctypes.data):
        raise WeaverError("rotary_frequencies: theta and factor must be positive, rotary_dim > 2 for ntk, and for parts "
                          "original_length > 0 and 0 <= low < high", AW_E_INVALID_ARG)
    return out


class Rotary:
    """A rotation: which dims turn, in which pairs, and the frequencies on the device.

    ``rotary_dim`` dims of each head turn (the others pass), in pairs (p, p +
    rotary_dim / 2) or, ``interleaved``, (2p, 2p + 1).  Frequencies are those of
    ``rotary_frequencies``, or ``inv_freq`` (rotary_dim / 2 values in radians per
    position) as given.  ``magnitude`` multiplies cosines and sines (some long-context
    scalings sharpen the scores so)."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, *, interleaved: bool = False, scaling: str = "none",
                 factor: float = 1.0, original_length: float = 0.0, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 1.0, inv_freq=None, device="cuda:0"):
        import torch
        if inv_freq is None:
            inv_freq = rotary_frequencies(rotary_dim, theta, scaling, factor, original_length, low, high)
        self.inv_freq = torch.as_tensor(inv_freq, dtype=torch.float64).to(device).contiguous()
        if rotary_dim < 2 or rotary_dim % 2 or self.inv_freq.numel() != rotary_dim // 2:
            raise WeaverError(f"rotary_dim {rotary_dim} must be even, with half as many frequencies "
                              f"({self.inv_freq.numel()})", AW_E_INVALID_ARG)
        self.rotary_dim, self.interleaved, self.magnitude = rotary_dim, interleaved, magnitude


def _rotary_rows(r: RotaryDesc, *, num_tokens, q_heads, kv_heads, head_dim, rotary, q, k, q_out, k_out, positions,
                 start_position, q_norm, k_norm, eps) -> list:
    """Fills the descriptor of the rows; returns the tensors behind it."""
    _counts(num_tokens=num_tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, start_position=start_position)
    r.num_tokens, r.q_heads, r.kv_heads, r.head_dim = num_tokens, q_heads, kv_heads, head_dim
    r.start_position, r.eps, r.magnitude = start_position, eps, 1.0
    for t, heads, name in ((q, q_heads, "q"), (k, kv_heads, "k"), (q_out, q_heads, "q_out"), (k_out, kv_heads, "k_out")):
        setattr(r, name, _ptr(t))
        setattr(r, name + "_stride", _token_rows(t, num_tokens, heads, head_dim, name))
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        _f16(t, head_dim, name)
        setattr(r, name, _ptr(t))
    _u32(positions, num_tokens, "positions")
    r.positions = _ptr(positions)
    if rotary is not None:
        _f64(rotary.inv_freq, rotary.rotary_dim // 2, "inv_freq")
        r.rotary_dim, r.layout, r.magnitude = rotary.rotary_dim, int(rotary.interleaved), rotary.magnitude
        r.inv_freq = _ptr(rotary.inv_freq)
    return [q, k, q_out, k_out, q_norm, k_norm, positions] + ([rotary.inv_freq] if rotary is not None else [])


def make_rotary_desc(*, num_tokens: int, q_heads: int, kv_heads: int, head_dim: int, rotary: Optional[Rotary], q, k,
                     q_out=None, k_out=None, positions=None, start_position: int = 0, q_norm=None, k_norm=None,
                     eps: float = 1e-5) -> RotaryDesc:
    """An ``aw_rotary_desc`` from device tensors (or raw device pointers to contiguous
    rows), for ``rotary`` and ``qk_norm_rotary``.  q_out and k_out default to q and k
    (in place); ``positions`` is an int32 tensor of one (unsigned) position per token."""
    d = RotaryDesc()
    keep = _rotary_rows(d, num_tokens=num_tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary,
                        q=q, k=k, q_out=q if q_out is None else q_out, k_out=k if k_out is None else k_out,
                        positions=positions, start_position=start_position, q_norm=q_norm, k_norm=k_norm, eps=eps)
    _one_device(d, keep)
    return d


def _table(refs, batch: int, count: int, stride: Optional[int], what: str) -> int:
    """Row stride of a block table [batch][>= count]."""
    if hasattr(refs, "dim") and refs.dim() == 2:
        if refs.shape[0] < batch or refs.shape[1] < count or (refs.shape[1] > 1 and refs.stride(1) != 1) or \
                (batch > 1 and refs.stride(0) < count):
            raise WeaverError(f"{what}: a table of [{batch}][{count}] entries is read, got shape {tuple(refs.shape)}, "
                              f"strides {tuple(refs.stride())}", AW_E_INVALID_ARG)
        _u32(refs[:0].contiguous(), 0, what)
        return refs.stride(0) if batch > 1 else max(refs.stride(0), count)
    stride = count if stride is None else stride
    _u32(refs, (batch - 1) * stride + count if batch else 0, what)
    return stride


def make_append_desc(*, batch: int, num_tokens: int, q_heads: int, kv_heads: int, head_dim: int, k, v, hot_k, hot_v,
                     refs, seq_hot, hot_count: Optional[int] = None, hot_blocks: Optional[int] = None,
                     refs_stride: Optional[int] = None, token_offsets=None, rotary: Optional[Rotary] = None, q=None,
                     q_out=None, positions=None, start_position: int = 0, q_norm=None, k_norm=None,
                     eps: float = 1e-5) -> AppendDesc:
    """An ``aw_append_desc`` from device tensors (or raw device pointers), for ``append_paged``.
    ``refs`` [batch][refs_stride] and ``seq_hot`` [batch] (tokens AFTER the append) are the block
    table and counts of the decode that follows; ``hot_count`` (pages of a sequence) defaults to a
    2-D table's columns and ``hot_blocks`` to the pool tensor's pages.  Without ``rotary`` k and q
    keep their positions' angles as they are; without ``q`` (q_heads 0) only k and v move."""
    d = AppendDesc()
    if q is None and q_heads:
        raise WeaverError("append_paged: q_heads without q", AW_E_INVALID_ARG)
    keep = _rotary_rows(d.rows, num_tokens=num_tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                        rotary=rotary, q=q, k=k, q_out=q if q_out is None else q_out, k_out=None, positions=positions,
                        start_position=start_position, q_norm=q_norm, k_norm=k_norm, eps=eps)
    page = BLOCK_SIZE * kv_heads * head_dim
    if hot_count is None:
        if not hasattr(refs, "dim") or refs.dim() != 2:
            raise WeaverError("append_paged: hot_count is required without a 2-D table", AW_E_INVALID_ARG)
        hot_count = refs.shape[1]
    if hot_blocks is None:
        if not hasattr(hot_k, "numel"):
            raise WeaverError("append_paged: hot_blocks is required for a raw pool pointer", AW_E_INVALID_ARG)
        hot_blocks = hot_k.numel() // max(page, 1)
    _counts(batch=batch, hot_count=hot_count, hot_blocks=hot_blocks, refs_stride=refs_stride or 0)
    for t, name in ((hot_k, "hot_k"), (hot_v, "hot_v")):
        _f16(t, hot_blocks * page, name)
        setattr(d, name, _ptr(t))
    d.v_stride = _token_rows(v, num_tokens, kv_heads, head_dim, "v")
    d.batch, d.hot_count, d.hot_blocks, d.v = batch, hot_count, hot_blocks, _ptr(v)
    d.refs_stride = _table(refs, batch, hot_count, refs_stride, "refs")
    _u32(seq_hot, batch, "seq_hot")
    _u32(token_offsets, batch + 1, "token_offsets")
    d.refs, d.seq_hot, d.token_offsets = _ptr(refs), _ptr(seq_hot), _ptr(token_offsets)
    _one_device(d, keep + [v, hot_k, hot_v, refs, seq_hot, token_offsets])
    return d


def make_prefix_desc(*, batch: int, queries: int, q_heads: int, kv_heads: int, head_dim: int, prefix_tokens: int, q, out,
                     hot_k, hot_v=None, prefix_refs=None, own_count: int = 0, refs=None, refs_stride: Optional[int] = None,
                     seq_own=None, hot_blocks: Optional[int] = None, scale: Optional[float] = None,
                     causal: bool = True) -> PrefixDesc:
    """An ``aw_prefix_desc`` from device tensors (or raw device pointers), for
    ``shared_prefix_attention``: q and out [batch][queries][q_heads][head_dim], the prefix'
    pages in ``prefix_refs``, each sequence's own in its row of ``refs`` and their number of
    tokens in ``seq_own`` (``out`` may be q).  ``scale`` defaults to 1 / sqrt(head_dim), ``hot_blocks`` to the
    pool tensor's pages."""
    d = PrefixDesc()
    _counts(batch=batch, queries=queries, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, prefix_tokens=prefix_tokens,
            own_count=own_count, refs_stride=refs_stride or 0, hot_blocks=hot_blocks or 0)
    d.batch, d.queries, d.q_heads, d.kv_heads, d.head_dim = batch, queries, q_heads, kv_heads, head_dim
    d.prefix_tokens, d.own_count, d.flags = prefix_tokens, own_count, AW_F_CAUSAL if causal else 0
    d.scale = head_dim ** -0.5 if scale is None else scale
    page = BLOCK_SIZE * kv_heads * head_dim
    if hot_blocks is None:
        if not hasattr(hot_k, "numel"):
            raise WeaverError("shared_prefix_attention: hot_blocks is required for a raw pool pointer", AW_E_INVALID_ARG)
        hot_blocks = hot_k.numel() // max(page, 1)
    d.hot_blocks = hot_blocks
    for t, need, name in ((q, batch * queries * q_heads * head_dim, "q"), (out, batch * queries * q_heads * head_dim, "out"),
                          (hot_k, hot_blocks * page, "hot_k"), (hot_v, hot_blocks * page, "hot_v")):
        _f16(t, need, name)
        setattr(d, name, _ptr(t))
    _u32(prefix_refs, -(-prefix_tokens // BLOCK_SIZE), "prefix_refs")
    _u32(seq_own, batch, "seq_own")
    d.refs_stride = _table(refs, batch, own_count, refs_stride, "refs") if refs is not None else own_count
    d.prefix_refs, d.refs, d.seq_own = _ptr(prefix_refs), _ptr(refs), _ptr(seq_own)
    _one_device(d, [q, out, hot_k, hot_v, prefix_refs, refs, seq_own])
    return d


def prefix_plan(desc: PrefixDesc, compute_units: int = 0, lib_path=None) -> PrefixPlanInfo:
    """Validate a ``shared_prefix_attention`` request and return how it is split (no GPU needed)."""
    info, msg = PrefixPlanInfo(), ctypes.create_string_buffer(256)
    rc = _lib.load(lib_path).aw_shared_prefix_plan(ctypes.byref(desc), compute_units, ctypes.byref(info), msg, 256)
    if rc:
        raise WeaverError(msg.value.decode(), rc)
    return info


class OpsEngine:
    """``Ops`` (ops.rs:21-462) on MI355X.  Shares a ``WeaverEngine`` (device,
    device error word, last-error text) or creates its own."""

    def __init__(self, engine: Optional[WeaverEngine] = None, lib_path=None, device: int = 0):
        self._own = engine is None
        self.engine = engine if engine is not None else WeaverEngine(lib_path=lib_path, device=device)
        self._lib = self.engine._lib

    def close(self) -> None:
        if self._own:
            self.engine.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _call(self, name: str, *args) -> None:
        rc = getattr(self._lib, name)(self.engine._h, *args)
        if rc:
            self.engine._check(rc, name[len("aw_ops_"):] if name.startswith("aw_ops_") else name)

    # -- batch mode (ops.rs:88-101)
    def begin_batch(self) -> None:
        """Nothing to open: calls are already queued on the stream without waiting."""

    def end_batch(self, stream: Optional[int] = None) -> None:
        """Wait until everything queued on the stream has finished (ops.rs:95-101)."""
        import torch
        s = _stream(stream)
        if s is None:
            torch.cuda.synchronize()
        elif s == 0:  # the null stream (torch.cuda.ExternalStream(0) would make a stream of its own)
            torch.cuda.default_stream().synchronize()
        else:
            torch.cuda.ExternalStream(s).synchronize()

    def check_device_errors(self, stream: Optional[int] = None) -> None:
        """Raise if a kernel saw out-of-range input (an embed token id >= vocab_size)."""
        self.engine.check_device_errors(stream)

    # -- the ops
    def copy_buffer(self, src, dst, count: int, src_off: int, dst_off: int, stream: Optional[int] = None) -> None:
        """ops.rs:166-180: dst[dst_off + i] = src[src_off + i], i < count (f16 elements)."""
        _f16(src, src_off + count, "copy_buffer src")
        _f16(dst, dst_off + count, "copy_buffer dst")
        self._call("aw_ops_copy_buffer", _ptr(src), _ptr(dst), count, src_off, dst_off, _stream(stream))

    def embed_lookup(self, token_ids, embed_table, output, hidden_size: int, seq_len: int,
                     vocab_size: Optional[int] = None, stream: Optional[int] = None) -> None:
        """ops.rs:183-206: output[t] = embed_table[token_ids[t]]; ``vocab_size``
        defaults to the table tensor's rows."""
        if vocab_size is None:
            if not hasattr(embed_table, "numel"):
                raise WeaverError("embed_lookup: vocab_size is required for a raw table pointer", AW_E_INVALID_ARG)
            vocab_size = embed_table.numel() // max(hidden_size, 1)
        _u32(token_ids, seq_len, "embed_lookup token_ids")
        _f16(embed_table, vocab_size * hidden_size, "embed_lookup embed_table")
        _f16(output, seq_len * hidden_size, "embed_lookup output")
        self._call("aw_ops_embed_lookup", _ptr(token_ids), _ptr(embed_table), _ptr(output), hidden_size, seq_len,
                   vocab_size, _stream(stream))

    def rms_norm(self, input, weight, output, hidden_size: int, num_tokens: int, eps: float,
                 stream: Optional[int] = None) -> None:
        """ops.rs:209-231: output = input * rsqrt(mean(input^2) + eps) * weight, per token."""
        _f16(input, hidden_size * num_tokens, "rms_norm input")
        _f16(weight, hidden_size, "rms_norm weight")
        _f16(output, hidden_size * num_tokens, "rms_norm output")
        self._call("aw_ops_rms_norm", _ptr(input), _ptr(weight), _ptr(output), hidden_size, num_tokens, eps,
                   _stream(stream))

    def rope(self, q, k, num_tokens: int, q_heads: int, kv_heads: int, head_dim: int, start_position: int,
             theta: float, stream: Optional[int] = None) -> None:
        """ops.rs:234-263: rotary embedding of q and k in place."""
        _f16(q, num_tokens * q_heads * head_dim, "rope q")
        _f16(k, num_tokens * kv_heads * head_dim, "rope k")
        self._call("aw_ops_rope", _ptr(q), _ptr(k), num_tokens, q_heads, kv_heads, head_dim, start_position, theta,
                   _stream(stream))

    def matmul(self, a, b, output, m: int, n: int, k: int, stream: Optional[int] = None) -> None:
        """ops.rs:266-296: output [m][n] = a [m][k] . b [n][k]^T, f16 out."""
        _f16(a, m * k, "matmul a")
        _f16(b, n * k, "matmul b")
        _f16(output, m * n, "matmul output")
        self._call("aw_ops_matmul", _ptr(a), _ptr(b), _ptr(output), m, n, k, _stream(stream))

    def silu_gate(self, gate, up, output, size: int, stream: Optional[int] = None) -> None:
        """ops.rs:299-312: output = SiLU(gate) * up."""
        for t, w in ((gate, "gate"), (up, "up"), (output, "output")):
            _f16(t, size, f"silu_gate {w}")
        self._call("aw_ops_silu_gate", _ptr(gate), _ptr(up), _ptr(output), size, _stream(stream))

    def add_residual(self, x, residual, size: int, stream: Optional[int] = None) -> None:
        """ops.rs:315-327: x += residual."""
        _f16(x, size, "add_residual x")
        _f16(residual, size, "add_residual residual")
        self._call("aw_ops_add_residual", _ptr(x), _ptr(residual), size, _stream(stream))

    def add_bias(self, x, bias, hidden_size: int, num_tokens: int, stream: Optional[int] = None) -> None:
        """ops.rs:330-343: x[t][d] += bias[d]."""
        _f16(x, hidden_size * num_tokens, "add_bias x")
        _f16(bias, hidden_size, "add_bias bias")
        self._call("aw_ops_add_bias", _ptr(x), _ptr(bias), hidden_size, num_tokens, _stream(stream))

    def scale_f16(self, x, count: int, scale: float, stream: Optional[int] = None) -> None:
        """ops.rs:350-363: x *= scale."""
        _f16(x, count, "scale_f16 x")
        self._call("aw_ops_scale_f16", _ptr(x), count, scale, _stream(stream))

    def matmul_scaled(self, a, b, output, m: int, n: int, k: int, scale: float,
                      stream: Optional[int] = None) -> None:
        """ops.rs:366-406: output [m][n] = (a . b^T) * scale, f32 out."""
        _f16(a, m * k, "matmul_scaled a")
        _f16(b, n * k, "matmul_scaled b")
        _f32(output, m * n, "matmul_scaled output")
        self._call("aw_ops_matmul_scaled", _ptr(a), _ptr(b), _ptr(output), m, n, k, scale, _stream(stream))

    def causal_attention(self, q, k, v, output, kv_len: int, head_dim: int, cache_tokens: Optional[int] = None,
                         stream: Optional[int] = None) -> None:
        """ops.rs:409-430: single-head softmax(q.K^T/sqrt(d)) V over kv_len rows.
        ``cache_tokens`` (rows k and v hold, >= kv_len rounded up to 16) defaults
        to the k tensor's rows."""
        if cache_tokens is None:
            if not hasattr(k, "numel"):
                raise WeaverError("causal_attention: cache_tokens is required for raw pointers", AW_E_INVALID_ARG)
            cache_tokens = k.numel() // head_dim
        _f16(q, head_dim, "causal_attention q")
        for t, w in ((k, "k"), (v, "v")):
            _f16(t, cache_tokens * head_dim, f"causal_attention {w}")
        _f16(output, head_dim, "causal_attention output")
        self._call("aw_ops_causal_attention", _ptr(q), _ptr(k), _ptr(v), _ptr(output), kv_len, head_dim,
                   cache_tokens, _stream(stream))

    # -- fused forms (no reference counterpart): the same output bits as the separate calls
    def matmul_add_residual(self, a, b, x, m: int, n: int, k: int, residual_multiplier: float = 1.0,
                            stream: Optional[int] = None) -> None:
        """matmul, scale_f16 by ``residual_multiplier``, add_residual into x, in one launch
        (forward_batch's o_proj and down_proj steps, inference.rs:564-572,592-600)."""
        _f16(a, m * k, "matmul_add_residual a")
        _f16(b, n * k, "matmul_add_residual b")
        _f16(x, m * n, "matmul_add_residual x")
        self._call("aw_ops_matmul_add_residual", _ptr(a), _ptr(b), _ptr(x), m, n, k, residual_multiplier,
                   _stream(stream))

    def matmul_silu_gate(self, a, b_gate, b_up, output, m: int, n: int, k: int, stream: Optional[int] = None) -> None:
        """The gate and up matmuls and silu_gate in one launch (inference.rs:586-591); m <= 64."""
        _f16(a, m * k, "matmul_silu_gate a")
        _f16(b_gate, n * k, "matmul_silu_gate b_gate")
        _f16(b_up, n * k, "matmul_silu_gate b_up")
        _f16(output, m * n, "matmul_silu_gate output")
        self._call("aw_ops_matmul_silu_gate", _ptr(a), _ptr(b_gate), _ptr(b_up), _ptr(output), m, n, k,
                   _stream(stream))

    def matmul_qkv(self, a, b_q, b_k, b_v, q, k_out, v_out, m: int, n_q: int, n_kv: int, k: int,
                   stream: Optional[int] = None) -> None:
        """The q, k and v matmuls in one launch (inference.rs:518-523)."""
        _f16(a, m * k, "matmul_qkv a")
        for t, n, w in ((b_q, n_q, "b_q"), (b_k, n_kv, "b_k"), (b_v, n_kv, "b_v")):
            _f16(t, n * k, f"matmul_qkv {w}")
        for t, n, w in ((q, n_q, "q"), (k_out, n_kv, "k_out"), (v_out, n_kv, "v_out")):
            _f16(t, m * n, f"matmul_qkv {w}")
        self._call("aw_ops_matmul_qkv", _ptr(a), _ptr(b_q), _ptr(b_k), _ptr(b_v), _ptr(q), _ptr(k_out), _ptr(v_out),
                   m, n_q, n_kv, k, _stream(stream))

    # -- rotary positions, head norms, paged appends (no reference counterpart): a call's descriptor
    # holds its tensors and may be used again for as long as they are the call's
    def _request(self, name: str, desc, stream: Optional[int]) -> None:
        device = desc._device
        if device is not None and device != self.engine.device:
            raise WeaverError(f"{name}: tensors on GPU {device}, the engine on {self.engine.device}", AW_E_INVALID_ARG)
        if stream is None:  # of the tensors' GPU, whichever torch's current one is
            stream = _stream(None) if device is None else \
                sys.modules["torch"]._C._cuda_getCurrentRawStream(device) or None
        rc = getattr(self._lib, name)(self.engine._h, ctypes.byref(desc), stream)
        if rc:
            self.engine._check(rc, name.removeprefix("aw_ops_"))

    def rotary(self, desc: RotaryDesc, stream: Optional[int] = None) -> None:
        """q and k heads turned by their positions (``make_rotary_desc``)."""
        self._request("aw_ops_rotary", desc, stream)

    def qk_norm_rotary(self, desc: RotaryDesc, stream: Optional[int] = None) -> None:
        """q and k heads RMS-normed with weights of their own, then turned (``make_rotary_desc``)."""
        self._request("aw_ops_qk_norm_rotary", desc, stream)

    def append_paged(self, desc: AppendDesc, stream: Optional[int] = None) -> None:
        """A batch's new k and v rows into their sequences' pages, k and q normed and turned
        on the way (``make_append_desc``)."""
        self._request("aw_ops_append_paged", desc, stream)

    def shared_prefix_attention(self, desc: PrefixDesc, stream: Optional[int] = None) -> None:
        """Attention over pages of a batch whose sequences share a prefix, read once for all
        (aw_shared_prefix_attention_device; ``make_prefix_desc``)."""
        self._request("aw_shared_prefix_attention_device", desc, stream)

    def multihead_attention(self, q, k_cache, v_cache, output, kv_len: int, head_dim: int, q_heads: int,
                            kv_heads: int, num_queries: int, cache_tokens: Optional[int] = None,
                            stream: Optional[int] = None) -> None:
        """ops.rs:433-462 (aw_multihead_attention_device)."""
        self.engine.multihead_attention(q, k_cache, v_cache, output, kv_len, head_dim, q_heads, kv_heads,
                                        num_queries, cache_tokens=cache_tokens, stream=stream)
