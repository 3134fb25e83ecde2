"""What a served batch does between a layer's q/k/v product and its output product, as cases to time and compare.

A layer of a decode or prompt step takes the rows of q, k and v, turns q and k by
their positions (some models norm each head first), writes k and v into the pages
of each sequence, and attends over the pages.  Kinds of case (the field ``kind``):
  rotary  q and k heads turned by their positions
  norm    q and k heads RMS-normed, then turned
  append  a ragged batch's k and v rows into 16-token pages, q and k turned on the way
  prefix  one attention over pages for a batch whose sequences share a prefix
Each is computed in its plain form, or (``own``) by the framework's operators.
Widths are those of the model presets; pages of 16 tokens are the framework's.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-5
THETA = 500000.0
PAGE = 16

#: (q_heads, kv_heads, head_dim) of the model presets.
WIDTHS = {"llama8b": (32, 8, 128), "granite2b": (32, 8, 64), "qwen05b": (14, 2, 64), "deepseek_r1_1_5b": (12, 2, 128)}


def _heads(model: str) -> dict:
    q_heads, kv_heads, head_dim = WIDTHS[model]
    return {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim}


def _turn(model: str, *, rotary_dim: int = 0, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
          original: int = 8192, magnitude: float = 1.0) -> dict:
    """Heads of a preset and their rotation: ``rotary_dim`` 0 turns whole heads."""
    h = _heads(model)
    return {**h, "rotary_dim": rotary_dim or h["head_dim"], "interleaved": interleaved, "scaling": scaling,
            "factor": factor, "original": original, "magnitude": magnitude}


def _rows(kind: str, turn: dict, tokens: int, *, start: int = 0, far: int = 0, fused: bool = False) -> dict:
    """``far``: each token has a position of its own below it; else start, start + 1, ...
    ``fused``: q and k are views of the rows that one q/k/v product wrote."""
    return {"kind": kind, **turn, "tokens": tokens, "start": start, "far": far, "fused": fused}


def _append(turn: dict, batch: int, new: int, held: int, *, start: int = 0, norm: bool = False,
            fused: bool = True) -> dict:
    """Up to ``new`` new tokens for each sequence behind up to ``held`` that it has."""
    return {"kind": "append", **turn, "batch": batch, "new": new, "held": held, "start": start, "norm": norm,
            "fused": fused}


def _prefix(model: str, batch: int, queries: int, prefix: int, own_tokens: int) -> dict:
    """``own_tokens``: the longest sequence's tokens behind the prefix, the new ones among them."""
    return {"kind": "prefix", **_heads(model), "batch": batch, "queries": queries, "prefix": prefix,
            "own_tokens": own_tokens}


def listed() -> list:
    def named(name: str, case: dict) -> dict:
        return {"name": name, **case}
    return [
        # The newest token of one conversation: a launch's latency.
        named("rotary_step", _rows("rotary", _turn("qwen05b"), 1, start=30011)),
        # A piece of a prompt: neighbouring pairs of half of each head turned, rows read out of the fused product.
        named("rotary_chunk", _rows("rotary", _turn("llama8b", rotary_dim=64, interleaved=True), 509, start=1022, fused=True)),
        # Packed prompts in a long context: a position for each token, frequencies stretched by parts, cosines scaled.
        named("rotary_prompt", _rows("rotary", _turn("llama8b", scaling="parts", factor=16.0, magnitude=1.2772588722239782),
                                     8192, far=131072)),
        # A batch of draft tokens to verify.
        named("norm_step", _rows("norm", _turn("granite2b"), 16, start=4095)),
        # A prompt, heads normed, rows of the fused product.
        named("norm_prompt", _rows("norm", _turn("deepseek_r1_1_5b", scaling="linear", factor=4.0), 6000, start=0, fused=True)),
        # One decode step of 64 sequences.
        named("append_step", _append(_turn("llama8b"), 64, 1, 2048)),
        # Drafts and short prompt pieces of a few sequences, one of them without new tokens.
        named("append_ragged", _append(_turn("qwen05b", interleaved=True, scaling="ntk", factor=2.0), 7, 37, 700, start=1531)),
        # Prompts of several sequences at once, heads normed on the way.
        named("append_prompt", _append(_turn("llama8b"), 6, 2048, 100, norm=True)),
        # Two conversations behind a short instruction.
        named("prefix_small", _prefix("qwen05b", 2, 1, 117, 9)),
        # One decode step of 64 conversations behind a long instruction.
        named("prefix_step", _prefix("llama8b", 64, 1, 8192, 257)),
        # Eight drafts to verify in each of 16 conversations behind a document that ends inside a page.
        named("prefix_verify", _prefix("granite2b", 16, 8, 4099, 600)),
        # Many questions over a long document.
        named("prefix_long", _prefix("llama8b", 96, 1, 32768, 1500)),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number in lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_turn(rng) -> dict:
    scaling = rng.choice(["none", "linear", "ntk", "parts"])
    turn = _turn(rng.choice(sorted(WIDTHS)), interleaved=rng.random() < 0.5, scaling=scaling,
                 factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 7.5, 32.0]))
    if rng.random() < 0.3:  # other widths of a head, odd ones among them
        turn["head_dim"] = rng.choice([32, 72, 80, 96, 112, 160, 192, 256])
        turn["rotary_dim"] = turn["head_dim"]
    if rng.random() < 0.4:  # part of the head
        turn["rotary_dim"] = 2 * rng.randrange(2, turn["head_dim"] // 2 + 1)
    if scaling == "parts" and rng.random() < 0.5:
        turn["magnitude"] = 0.1 * math.log(turn["factor"]) + 1.0
    return turn


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "norm", "append", "prefix", "prefix"])
    if kind in ("rotary", "norm"):
        return _rows(kind, _draw_turn(rng), _spread(rng, 1, 8192), start=rng.randrange(0, 100000),
                     far=rng.choice([0, 0, 32768, 1000000]), fused=rng.random() < 0.5)
    if kind == "append":
        batch = _spread(rng, 1, 128)
        return _append(_draw_turn(rng), batch, _spread(rng, 1, max(1, 16384 // batch)), _spread(rng, 1, 2048) - 1,
                       start=rng.choice([0, rng.randrange(0, 32768)]), norm=rng.random() < 0.5, fused=rng.random() < 0.5)
    batch, queries = _spread(rng, 1, 96), rng.choice([1, 1, 1, rng.randrange(2, 9), _spread(rng, 9, 64)])
    while batch * queries > 384:
        batch = batch // 2
    prefix = _spread(rng, 1, min(32768, 96 * 32768 // (batch * queries)))
    return _prefix(rng.choice(sorted(WIDTHS)), batch, queries, prefix, queries - 1 + _spread(rng, 1, 1500))


# ---------------------------------------------------------------- inputs


class _Rand:
    """Normal f16 tensors on the GPU from one seed."""

    def __init__(self, seed: int):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)

    def __call__(self, *shape, scale: float = 1.0, mean: float = 0.0) -> torch.Tensor:
        t = torch.randn(shape, generator=self.gen, device=DEVICE, dtype=torch.float32)
        return t.mul_(scale).add_(mean).to(torch.float16)

    def below(self, n: int, *shape) -> torch.Tensor:
        return torch.randint(0, n, shape, generator=self.gen, device=DEVICE, dtype=torch.int32)

    def pages(self, n: int) -> torch.Tensor:
        """The numbers of n pages in the order in which a used pool hands them out."""
        return torch.randperm(n, generator=self.gen, device=DEVICE).to(torch.int32)


def _spaced(n: int, lo: int, hi: int) -> list:
    """n whole numbers evenly from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _counts(c: dict):
    """New and held tokens of each sequence of an ``append`` case."""
    new = _spaced(c["batch"], 0 if c["new"] > 1 else 1, c["new"])
    return new, _spaced(c["batch"], 0, c["held"])[::-1]


def _table(r: _Rand, blocks: list, first: torch.Tensor, spare: int) -> torch.Tensor:
    """A block table with ``blocks[b]`` entries for sequence b taken in order from ``first``."""
    table = torch.full((len(blocks), max(max(blocks), 1) + spare), 0, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = first[at:at + n]
        at += n
    return table


def _qkv(r: _Rand, c: dict, tokens: int, with_v: bool) -> dict:
    hq, hk, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["fused"]:
        rows = r(tokens, hq + 2 * hk, d, scale=1.5)
        got = {"q": rows[:, :hq], "k": rows[:, hq:hq + hk], "v": rows[:, hq + hk:]}
    else:
        got = {"q": r(tokens, hq, d, scale=1.5), "k": r(tokens, hk, d, scale=1.5), "v": r(tokens, hk, d)}
    return got if with_v else {"q": got["q"], "k": got["k"]}


def _inputs(c: dict, seed: int) -> dict:
    r, hq, hk, d = _Rand(seed), c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] in ("rotary", "norm"):
        i = _qkv(r, c, c["tokens"], False)
        i["positions"] = r.below(c["far"], c["tokens"]) if c["far"] else None
    elif c["kind"] == "append":
        new, held = _counts(c)
        i = _qkv(r, c, sum(new), True)
        blocks = [-(-(n + h) // PAGE) for n, h in zip(new, held)]
        pages = sum(blocks) + 3
        i["hot_k"], i["hot_v"] = r(pages, PAGE, hk, d), r(pages, PAGE, hk, d)
        i["refs"] = _table(r, blocks, r.pages(pages), 1)
        i["seq_hot"] = torch.tensor([n + h for n, h in zip(new, held)], dtype=torch.int32, device=DEVICE)
        i["token_offsets"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEVICE)
    else:
        own_lengths = _spaced(c["batch"], c["queries"], c["own_tokens"])
        blocks = [-(-n // PAGE) for n in own_lengths]
        shared = -(-c["prefix"] // PAGE)
        pages = shared + sum(blocks) + 3
        order = r.pages(pages)
        return {"q": r(c["batch"], c["queries"], hq, d), "hot_k": r(pages, PAGE, hk, d), "hot_v": r(pages, PAGE, hk, d),
                "prefix_refs": order[:shared].contiguous(), "refs": _table(r, blocks, order[shared:], 0),
                "seq_own": torch.tensor(own_lengths, dtype=torch.int32, device=DEVICE)}
    if c["kind"] == "norm" or c.get("norm"):
        i["q_norm"], i["k_norm"] = r(d, scale=0.1, mean=1.0), r(d, scale=0.1, mean=1.0)
    return i


def prepare(case: dict, seed: int) -> dict:
    st = {"case": case, **_inputs(case, seed)}
    q = st["q"]
    if case["kind"] == "prefix":
        st["out"] = torch.empty_like(q)
        return st
    st["q_out"] = torch.empty(q.shape, dtype=torch.float16, device=DEVICE)
    if case["kind"] != "append":
        st["k_out"] = torch.empty(st["k"].shape, dtype=torch.float16, device=DEVICE)
    return st


# ---------------------------------------------------------------- one pass, in the plain form


def _frequencies(c: dict) -> torch.Tensor:
    """Radians per position of each pair, in 64 bits."""
    n, factor = c["rotary_dim"], c["factor"]
    theta = THETA * factor ** (n / (n - 2)) if c["scaling"] == "ntk" else THETA
    f = theta ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEVICE) / n)
    if c["scaling"] == "linear":
        return f / factor
    if c["scaling"] == "parts":
        keep = ((c["original"] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return (1.0 - keep) * f / factor + keep * f
    return f


def _normed(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _turned(c: dict, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Rows [tokens][heads][head_dim] in 32 bits, angles in 64."""
    angle = positions.double()[:, None, None] * _frequencies(c)
    cos, sin = (angle.cos() * c["magnitude"]).float(), (angle.sin() * c["magnitude"]).float()
    x, n = x.float(), c["rotary_dim"]
    y = x.clone()
    a = slice(0, n, 2) if c["interleaved"] else slice(0, n // 2)
    b = slice(1, n, 2) if c["interleaved"] else slice(n // 2, n)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _plain_rows(st: dict) -> dict:
    c = st["case"]
    positions = st["positions"]
    if positions is None:
        positions = c["start"] + torch.arange(c["tokens"], device=DEVICE)
    q, k = st["q"], st["k"]
    if c["kind"] == "norm":
        q, k = _normed(q, st["q_norm"]), _normed(k, st["k_norm"])
    st["q_out"].copy_(_turned(c, q, positions))
    st["k_out"].copy_(_turned(c, k, positions))
    return {"q": st["q_out"], "k": st["k_out"]}


def _plain_append(st: dict) -> dict:
    c, offsets = st["case"], st["token_offsets"].long()
    tokens = torch.arange(st["q"].shape[0], device=DEVICE)
    seq = torch.searchsorted(offsets[1:].contiguous(), tokens, right=True)
    place = st["seq_hot"].long()[seq] - (offsets[seq + 1] - tokens)
    row = st["refs"][seq, place // PAGE].long() * PAGE + place % PAGE
    q, k = st["q"], st["k"]
    if c["norm"]:
        q, k = _normed(q, st["q_norm"]), _normed(k, st["k_norm"])
    st["q_out"].copy_(_turned(c, q, place + c["start"]))
    st["hot_k"].flatten(0, 1)[row] = _turned(c, k, place + c["start"]).to(torch.float16)
    st["hot_v"].flatten(0, 1)[row] = st["v"]
    return {"q": st["q_out"], "k": st["hot_k"], "v": st["hot_v"]}


def _plain_prefix(st: dict) -> torch.Tensor:
    c = st["case"]
    b, n, hk, d, p = c["batch"], c["queries"], c["kv_heads"], c["head_dim"], c["prefix"]
    group = c["q_heads"] // hk
    # Rows [kv_heads][batch][queries * group][head_dim].
    q = st["q"].float().view(b, n, hk, group, d).permute(2, 0, 1, 3, 4).reshape(hk, b, n * group, d) / math.sqrt(d)
    refs = st["prefix_refs"].long()
    pk = st["hot_k"][refs].flatten(0, 1)[:p].permute(1, 0, 2).float().contiguous()
    pv = st["hot_v"][refs].flatten(0, 1)[:p].permute(1, 0, 2).float().contiguous()
    refs = st["refs"].long()
    ok = st["hot_k"][refs].flatten(1, 2).permute(2, 0, 1, 3).float().contiguous()
    ov = st["hot_v"][refs].flatten(1, 2).permute(2, 0, 1, 3).float().contiguous()
    sp = torch.matmul(q.flatten(1, 2), pk.transpose(1, 2).contiguous()).view(hk, b, n * group, p)
    so = torch.matmul(q, ok.transpose(2, 3).contiguous())
    sees = st["seq_own"].long()[:, None] - n + 1 + torch.arange(n, device=DEVICE).repeat_interleave(group)
    so = so.masked_fill(torch.arange(so.shape[-1], device=DEVICE) >= sees[..., None], -math.inf)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = (sp - top).exp(), (so - top).exp()
    out = torch.matmul(sp.flatten(1, 2), pv).view(hk, b, n * group, d) + torch.matmul(so, ov)
    out = out / (sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True))
    st["out"].copy_(out.view(hk, b, n, group, d).permute(1, 2, 0, 3, 4).flatten(2, 3))
    return st["out"]


# ---------------------------------------------------------------- one pass, by the framework's operators

_engines: dict = {}


def _ops():
    """The engine of the process, as a program keeps one per GPU."""
    if not _engines:
        from aether_nexus_amd.ops import OpsEngine
        _engines["ops"] = OpsEngine()
    return _engines["ops"]


def _rotary(c: dict):
    from aether_nexus_amd.ops import Rotary
    return Rotary(c["rotary_dim"], THETA, interleaved=c["interleaved"], scaling=c["scaling"], factor=c["factor"],
                  original_length=c["original"], low=1.0, high=32.0, magnitude=c["magnitude"], device=DEVICE)


def _request(st: dict):
    """The descriptor of a state's call, which a program keeps for as long as it calls with these tensors."""
    from aether_nexus_amd import ops
    c = st["case"]
    widths = {n: c[n] for n in ("q_heads", "kv_heads", "head_dim")}
    if c["kind"] == "prefix":
        return ops.make_prefix_desc(**widths, batch=c["batch"], queries=c["queries"], prefix_tokens=c["prefix"],
                                    own_count=st["refs"].shape[1], q=st["q"], hot_k=st["hot_k"], hot_v=st["hot_v"],
                                    prefix_refs=st["prefix_refs"], refs=st["refs"], seq_own=st["seq_own"], out=st["out"],
                                    scale=c["head_dim"] ** -0.5, causal=True)
    norms = {"q_norm": st["q_norm"], "k_norm": st["k_norm"], "eps": EPS} if "q_norm" in st else {}
    rows = {**widths, **norms, "rotary": _rotary(c), "q": st["q"], "k": st["k"], "q_out": st["q_out"]}
    if c["kind"] == "append":
        return ops.make_append_desc(**rows, num_tokens=st["q"].shape[0], batch=c["batch"], v=st["v"], hot_k=st["hot_k"],
                                    hot_v=st["hot_v"], refs=st["refs"], hot_count=st["refs"].shape[1],
                                    seq_hot=st["seq_hot"], token_offsets=st["token_offsets"], start_position=c["start"])
    return ops.make_rotary_desc(**rows, num_tokens=c["tokens"], k_out=st["k_out"], positions=st["positions"],
                                start_position=c["start"])


def run(state: dict):
    st, kind = state, state["case"]["kind"]
    if not own:
        return {"rotary": _plain_rows, "norm": _plain_rows, "append": _plain_append, "prefix": _plain_prefix}[kind](st)
    ops = _ops()
    if "desc" not in st:
        st["desc"] = _request(st)
    if kind == "prefix":
        ops.shared_prefix_attention(st["desc"])
        return st["out"]
    if kind == "append":
        ops.append_paged(st["desc"])
        return {"q": st["q_out"], "k": st["hot_k"], "v": st["hot_v"]}
    if kind == "norm":
        ops.qk_norm_rotary(st["desc"])
    else:
        ops.rotary(st["desc"])
    return {"q": st["q_out"], "k": st["k_out"]}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    c, hq, hk, d = case, case["q_heads"], case["kv_heads"], case["head_dim"]
    if c["kind"] == "prefix":
        lengths = _spaced(c["batch"], c["queries"], c["own_tokens"])
        held = c["prefix"] + sum(lengths)
        pairs = c["batch"] * c["queries"] * c["prefix"] + sum(c["queries"] * n - c["queries"] * (c["queries"] - 1) // 2
                                                              for n in lengths)
        io = 2 * c["batch"] * c["queries"] * hq * d
        return {"bytes": 2 * (2 * held * hk * d + io) + 4 * held // PAGE, "flops": 4 * pairs * hq * d}
    tokens = sum(_counts(c)[0]) if c["kind"] == "append" else c["tokens"]
    heads = hq + 2 * hk if c["kind"] == "append" else hq + hk
    turned = tokens * (hq + hk)
    norm = c["kind"] == "norm" or c.get("norm")
    return {"bytes": 4 * tokens * heads * d + 4 * tokens, "flops": turned * (3 * c["rotary_dim"] + (4 * d if norm else 0))}


# ---------------------------------------------------------------- the same in 64 bits


def _rows64(c: dict, x: torch.Tensor, positions: torch.Tensor, w=None) -> torch.Tensor:
    """Rows normed and turned as complex numbers times e^(i angle)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["head_dim"] + EPS) * w.double()
    n, factor, freq = c["rotary_dim"], c["factor"], []
    for p in range(n // 2):
        base = THETA * factor ** (n / (n - 2.0)) if c["scaling"] == "ntk" else THETA
        f = math.exp(-2.0 * p / n * math.log(base))
        if c["scaling"] == "linear":
            f /= factor
        elif c["scaling"] == "parts":
            turns = c["original"] * f / (2.0 * math.pi)  # over the length that the model was trained on
            g = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            f = f / factor * (1.0 - g) + f * g
        freq.append(f)
    angle = torch.outer(positions.double(), torch.tensor(freq, dtype=torch.float64, device=DEVICE))[:, None]
    turn = torch.polar(torch.full_like(angle, c["magnitude"]), angle)
    head, tail = x[..., :n], x[..., n:]
    if c["interleaved"]:
        z = torch.view_as_complex(head.unflatten(-1, (n // 2, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :n // 2].contiguous(), head[..., n // 2:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, tail], -1)


def _append64(c: dict, i: dict) -> dict:
    new, held = _counts(c)
    k_pool, v_pool = i["hot_k"].double().flatten(0, 1), i["hot_v"].double().flatten(0, 1)
    places = torch.tensor([h + j for n, h in zip(new, held) for j in range(n)], dtype=torch.int64, device=DEVICE)
    k = _rows64(c, i["k"], places + c["start"], i.get("k_norm"))
    at = 0
    for b, (n, h) in enumerate(zip(new, held)):
        p = torch.arange(h, h + n, device=DEVICE)
        rows = i["refs"][b].long()[p // PAGE] * PAGE + p % PAGE
        k_pool[rows], v_pool[rows] = k[at:at + n], i["v"][at:at + n].double()
        at += n
    return {"q": _rows64(c, i["q"], places + c["start"], i.get("q_norm")), "k": k_pool.view(i["hot_k"].shape),
            "v": v_pool.view(i["hot_v"].shape)}


def _prefix64(c: dict, i: dict) -> torch.Tensor:
    out = torch.empty(i["q"].shape, dtype=torch.float64, device=DEVICE)
    n, d, group = c["queries"], c["head_dim"], c["q_heads"] // c["kv_heads"]
    shared = i["prefix_refs"].long()
    for b, length in enumerate(_spaced(c["batch"], n, c["own_tokens"])):
        pages = i["refs"][b, :-(-length // PAGE)].long()
        k, v = (torch.cat([i[t][shared].flatten(0, 1)[:c["prefix"]], i[t][pages].flatten(0, 1)[:length]])
                .double().transpose(0, 1) for t in ("hot_k", "hot_v"))
        q = i["q"][b].double().view(n, c["kv_heads"], group, d).permute(1, 2, 0, 3)
        s = torch.matmul(q, k[:, None].transpose(-1, -2)) / math.sqrt(d)
        last = c["prefix"] + length - n + torch.arange(n, device=DEVICE)
        s = s.masked_fill(torch.arange(k.shape[1], device=DEVICE) > last[:, None], -math.inf)
        out[b] = torch.matmul(torch.softmax(s, -1), v[:, None]).permute(2, 0, 1, 3).flatten(1, 2)
    return out


def exact(case: dict, seed: int):
    c, i = case, _inputs(case, seed)
    if c["kind"] == "append":
        return _append64(c, i)
    if c["kind"] == "prefix":
        return _prefix64(c, i)
    positions = i["positions"]
    if positions is None:
        positions = torch.arange(c["start"], c["start"] + c["tokens"], device=DEVICE)
    return {"q": _rows64(c, i["q"], positions, i.get("q_norm")), "k": _rows64(c, i["k"], positions, i.get("k_norm"))}
