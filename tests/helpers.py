"""Shared helpers of the parity tests: run a workload on the GPU through the C
ABI and compare with the CPU oracle at the attention tolerance
(max-abs 2e-3, rel-L2 1e-3 against the fp64 brute force)."""
from __future__ import annotations

import numpy as np

MAX_ABS = 2e-3
REL_L2 = 1e-3


def run_gpu(engine, wl, stream, copy: int = 0, q_latent_f32: bool = False):
    import torch
    from aether_nexus_amd import workloads as W
    dev = wl.to("cuda:0")
    out = torch.full(dev.out_shape(), float("nan"), dtype=torch.float16, device="cuda:0")
    engine.decode_device(W.device_desc(dev, out, copy=copy, q_latent_f32=q_latent_f32), stream=stream)
    engine.check_device_errors(stream)
    return out.cpu().numpy()


def errors(got, ref) -> tuple[float, float]:
    got = np.asarray(got, dtype=np.float64)
    ref = np.asarray(ref, dtype=np.float64)
    d = got - ref
    return float(np.abs(d).max()), float(np.linalg.norm(d) / max(np.linalg.norm(ref), 1e-30))


def assert_close(got, ref, what: str = "", max_abs: float = MAX_ABS, rel_l2: float = REL_L2):
    assert np.all(np.isfinite(np.asarray(got, dtype=np.float64))), f"{what}: non-finite output"
    ma, rl = errors(got, ref)
    print(f"{what}: max_abs={ma:.3e} rel_l2={rl:.3e}", flush=True)
    assert ma <= max_abs and rl <= rel_l2, f"{what}: max_abs {ma:.3e} (<= {max_abs}), rel_l2 {rl:.3e} (<= {rel_l2})"


#: Requests of shared-prefix attention whose parts are longer than the 64 pages whose refs a wave holds:
#: batch, queries, q heads, kv heads, head_dim, prefix, own tokens.
LONG_PREFIXES = [(20, 1, 2, 2, 64, 70001, [1] * 20), (1, 2, 4, 1, 64, 300007, [2]), (2, 2, 2, 1, 64, 3, [300003, 40])]

#: Bound of a sequence's rel-L2 error of shared-prefix attention over many tokens with independent values of random
#: signs.  An output o = sum p v / sum p then has a root mean square of r = sqrt(sum p^2 v^2) / sum p.  Each weight's
#: rounding to f16 is within half a step, at most 2^-11 of it and uniform, so of a root mean square of 2^-11 / sqrt(3)
#: of it at most: together 2^-11 / sqrt(3) r; the f16 store likewise; both sqrt(2 / 3) 2^-11 r = 4.0e-4 r.  fp32 scores and
#: sums add a few 2^-24 of sum p |v|, and a mean over 64 values or more is within a quarter of the expectation.
PREFIX_REL_L2 = 5e-4


def prefix_errors(got, want, absolute, total, tokens: int, largest: float):
    """(worst error over tolerance, worst rel-L2 of a sequence) of outputs [batch][queries][heads][dims] over
    ``tokens`` tokens of values up to ``largest``, with the sums A of p |v| / sum p (``absolute``) and W of weights whose
    largest is 1 (``total``): half a step of the f16 store, 2^-11 |o|; the weights as f16 operands and their scores
    1.5 2^-11 A; a weight among f16's subnormals 2^-25 of the largest, together n 2^-25 max |v| / W; 2^-25."""
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want)
    tol = (2.0 ** -11 * np.abs(want) + 1.5 * 2.0 ** -11 * absolute +
           tokens * 2.0 ** -25 * largest / np.maximum(total, 1.0)[..., None] + 2.0 ** -25)
    d = np.abs(got - want)
    rel = [np.linalg.norm(a) / max(np.linalg.norm(b), 1e-30) for a, b in zip(d, want)]
    return float((d / tol).max()), float(max(rel))
