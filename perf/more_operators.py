"""A step of speculative decoding by trees of drafted tokens, as cases to time and compare.

A draft model proposes a tree of tokens for each sequence: node 0 is the newest token,
every other node continues its parent.  One step of the target model checks all of
them.  Kinds of case (the field ``kind``):
  tables  block tables, slots, positions and tree masks of a step, from the lengths
  tree    attention of the nodes over each sequence's pages and their own ancestors
  logits  penalties for repeated tokens, biases and grammar masks, and the best token
  accept  the walk along the target's tokens, the kept rows of every layer into the pages
Each is computed in its plain form, or (``own``) by the framework's operators.
Widths and vocabularies are those of the model presets; pages hold 16 tokens.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 16

#: (q_heads, kv_heads, head_dim, layers, vocabulary) of the model presets.
MODELS = {"llama8b": (32, 8, 128, 32, 128256), "granite2b": (32, 8, 64, 40, 49155), "qwen05b": (14, 2, 64, 24, 151936),
          "deepseek_r1_1_5b": (12, 2, 128, 28, 151936)}


def _tables(batch: int, new: int, held: int, *, tree: bool = False, pad: int = 0) -> dict:
    """Up to ``new`` new tokens for each sequence behind up to ``held``; ``pad`` rows behind the last sequence."""
    return {"kind": "tables", "batch": batch, "new": new, "held": held, "tree": tree, "pad": pad}


def _tree(model: str, batch: int, nodes: int, held: int, *, chain: bool = False, fused: bool = True, pad: int = 0) -> dict:
    """Trees of up to ``nodes`` nodes behind up to ``held`` tokens; ``chain``: no mask, each row sees those before it."""
    q_heads, kv_heads, head_dim, _, _ = MODELS[model]
    return {"kind": "tree", "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "batch": batch, "nodes": nodes,
            "held": held, "chain": chain, "fused": fused, "pad": pad}


def _logits(model: str, batch: int, nodes: int, history: int, *, half: bool = False, bias: int = 0, masks: str = "none",
            best: bool = True) -> dict:
    """Rows of up to ``nodes`` nodes for each sequence (0: one row, no tree).  ``masks``: "none", "open" (most
    tokens allowed) or "tight" (few)."""
    return {"kind": "logits", "vocab": MODELS[model][4], "batch": batch, "nodes": nodes, "history": history, "half": half,
            "bias": bias, "masks": masks, "best": best}


def _accept(model: str, batch: int, nodes: int, *, layers: int = 0, agree: int = 70) -> dict:
    """Trees of up to ``nodes`` nodes, ``agree`` per cent of whose inner nodes have a child that the target keeps."""
    _, kv_heads, head_dim, n, _ = MODELS[model]
    return {"kind": "accept", "kv_heads": kv_heads, "head_dim": head_dim, "layers": layers or n, "batch": batch,
            "nodes": nodes, "agree": agree}


def listed() -> list:
    def named(name: str, case: dict) -> dict:
        return {"name": name, **case}
    return [
        # One decode step of 64 conversations: a launch's latency.
        named("tables_step", _tables(64, 1, 4096)),
        # Trees of a large batch to verify, in a captured step's padded rows.
        named("tables_tree", _tables(256, 48, 9001, tree=True, pad=77)),
        # Prompts of many requests at once.
        named("tables_prompt", _tables(509, 1021, 700, pad=5)),
        # Two conversations with a few drafts each.
        named("tree_small", _tree("qwen05b", 2, 5, 700)),
        # One decode step of a full batch, short drafts: the pages' bytes.
        named("tree_step", _tree("llama8b", 64, 8, 4099, pad=3)),
        # Wide trees over long contexts: many rows to each page.
        named("tree_wide", _tree("llama8b", 16, 64, 8192)),
        # Two documents, questioned with trees.
        named("tree_long", _tree("granite2b", 2, 60, 65521)),
        # One answer's next token.
        named("logits_step", _logits("qwen05b", 1, 0, 1500, bias=20)),
        # A batch of answers under grammars, with biases.
        named("logits_batch", _logits("llama8b", 64, 0, 4096, bias=300, masks="tight")),
        # Every node of wide trees, each in a grammar's state of its own.
        named("logits_tree", _logits("granite2b", 16, 64, 2048, half=True, masks="open")),
        # Two conversations with a few drafts each.
        named("accept_small", _accept("qwen05b", 2, 5)),
        # A full batch of trees.
        named("accept_step", _accept("llama8b", 64, 32, agree=85)),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number in lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["tables", "tree", "tree", "logits", "accept"])
    model = rng.choice(sorted(MODELS))
    if kind == "tables":
        tree = rng.random() < 0.5
        batch = _spread(rng, 1, 512 if not tree else 256)
        new = _spread(rng, 1, 128 if tree else max(1, 500000 // batch))
        return _tables(batch, min(new, 20000), _spread(rng, 1, 40000) - 1, tree=tree, pad=rng.choice([0, 0, rng.randrange(1, 200)]))
    if kind == "tree":
        batch, nodes = _spread(rng, 1, 64), _spread(rng, 1, 128)
        while batch * nodes > 1024:
            batch = batch // 2
        q_heads, kv_heads = MODELS[model][:2]
        # Scores in 32 bits within 1 GiB, pages within 64 sequences of 4099 tokens.
        most = min(65536, (1 << 28) // (batch * nodes * q_heads), 262144 * 8 // (kv_heads * batch))
        return _tree(model, batch, nodes, _spread(rng, 1, max(1, most)) - 1, chain=rng.random() < 0.25, fused=rng.random() < 0.5,
                     pad=rng.choice([0, 0, rng.randrange(1, 9)]))
    if kind == "logits":
        batch, nodes = _spread(rng, 1, 64), rng.choice([0, 0, _spread(rng, 1, 64)])
        while batch * max(1, nodes) * MODELS[model][4] > 50331648:
            batch, nodes = max(1, batch // 2), nodes // 2 if batch < 2 else nodes
        return _logits(model, batch, nodes, _spread(rng, 1, 16384) - 1, half=rng.random() < 0.3,
                       bias=rng.choice([0, _spread(rng, 1, 512)]), masks=rng.choice(["none", "open", "tight"]), best=rng.random() < 0.75)
    batch, nodes = _spread(rng, 1, 64), _spread(rng, 1, 64)
    while batch * nodes > 2048:
        batch = batch // 2
    return _accept(model, batch, nodes, layers=_spread(rng, 1, 32), agree=rng.randrange(20, 101))


# ---------------------------------------------------------------- inputs


class _Rand:
    """Normal tensors on the GPU from one seed, and whole numbers."""

    def __init__(self, seed: int):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)

    def __call__(self, *shape, scale: float = 1.0, dtype=torch.float16) -> torch.Tensor:
        return torch.randn(shape, generator=self.gen, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)

    def unit(self, *shape) -> torch.Tensor:
        return torch.rand(shape, generator=self.gen, device=DEVICE, dtype=torch.float32)

    def pages(self, n: int) -> torch.Tensor:
        """The numbers of n pages in the order in which a used pool hands them out."""
        return torch.randperm(n, generator=self.gen, device=DEVICE).to(torch.int32)


def _ints(values, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _spaced(n: int, lo: int, hi: int) -> list:
    """n whole numbers evenly from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _offsets(counts: list) -> list:
    return [sum(counts[:b]) for b in range(len(counts) + 1)]


def _new(c: dict) -> list:
    """New tokens (nodes) of each sequence: a decode step has one each, others up to as many as the case says."""
    most = c["new"] if c["kind"] == "tables" else c["nodes"]
    if c["kind"] == "logits" and most == 0:
        return [1] * c["batch"]
    return _spaced(c["batch"], 1 if most == 1 or c["kind"] != "tables" else 0, most)


def _held(c: dict) -> list:
    return _spaced(c["batch"], 0 if c["kind"] == "tables" else c["held"] // 2, c["held"])[::-1]


def _grown(seed: int, counts: list) -> list:
    """Parents (within the tree, -1: a root) of trees of ``counts`` nodes, the early nodes with more children."""
    rng, parents = random.Random(seed), []
    for n in counts:
        parents.append([-1] + [int(i * rng.random() ** 1.3) for i in range(1, n)] if n else [])
    return parents


def _depths(parents: list) -> list:
    out = []
    for tree in parents:
        d = []
        for p in tree:
            d.append(d[p] + 1 if p >= 0 else 0)
        out.append(d)
    return out


def _sees(parents: list) -> list:
    """For each node the set, as bits, of itself and its ancestors."""
    out = []
    for tree in parents:
        s = []
        for i, p in enumerate(tree):
            s.append((1 << i) | (s[p] if p >= 0 else 0))
        out.append(s)
    return out


def _mask_words(c: dict) -> int:
    return -(-max(max(_new(c)), 1) // 32)


def _mask(c: dict, parents: list, rows: int) -> torch.Tensor:
    """[rows][words] of tree bits; rows behind the last tree see nothing."""
    words = _mask_words(c)
    flat = [[(s >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for tree in _sees(parents) for s in tree]
    flat += [[0] * words] * (rows - len(flat))
    return _ints(flat, torch.int64).to(torch.int32)


def _inputs_tables(c: dict, seed: int) -> dict:
    r, new, held = _Rand(seed), _new(c), _held(c)
    # Some sequences keep a page that an earlier step of theirs did not fill.
    pages = [-(-h // PAGE) + (b % 3 == 0) for b, h in enumerate(held)]
    need = [max(0, -(-(h + n) // PAGE) - p) for h, n, p in zip(held, new, pages)]
    width = max(max(p + x for p, x in zip(pages, need)), 1) + 1
    order = r.pages(sum(pages) + sum(need) + 9)
    refs = torch.full((c["batch"], width), -1, dtype=torch.int32, device=DEVICE)
    mine = torch.arange(width, device=DEVICE) < _ints(pages)[:, None]
    refs[mine] = order[:sum(pages)]
    i = {"refs": refs, "seq_held": _ints(held), "seq_new": _ints(new), "seq_pages": _ints(pages),
         "free": order[sum(pages):].contiguous(), "first": _ints([4]), "rows": sum(new) + c["pad"]}
    if c["tree"]:
        flat = [p for tree in _grown(seed, new) for p in tree]
        i["parents"] = _ints(flat + [-1] * c["pad"])
    return i


def _inputs_tree(c: dict, seed: int) -> dict:
    r, hq, hk, d = _Rand(seed), c["q_heads"], c["kv_heads"], c["head_dim"]
    new, held = _new(c), _held(c)
    rows, blocks = sum(new) + c["pad"], [-(-h // PAGE) for h in held]
    if c["fused"]:
        qkv = r(rows, hq + 2 * hk, d)
        i = {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:]}
    else:
        i = {"q": r(rows, hq, d), "k": r(rows, hk, d), "v": r(rows, hk, d)}
    pages = sum(blocks) + 3
    i["hot_k"], i["hot_v"] = r(pages, PAGE, hk, d), r(pages, PAGE, hk, d)
    order = r.pages(pages)
    i["refs"] = torch.zeros((c["batch"], max(max(blocks), 1)), dtype=torch.int32, device=DEVICE)
    i["refs"][torch.arange(i["refs"].shape[1], device=DEVICE) < _ints(blocks)[:, None]] = order[:sum(blocks)]
    i["seq_held"], i["token_offsets"] = _ints(held), _ints(_offsets(new))
    if not c["chain"]:
        i["mask"] = _mask(c, _grown(seed, new), rows)
    return i


def _inputs_logits(c: dict, seed: int) -> dict:
    r, v, b, new = _Rand(seed), c["vocab"], c["batch"], _new(c)
    rows = sum(new)

    def tokens(*shape):  # few tokens are common, most are rare
        return (v ** r.unit(*shape)).long().clamp(0, v - 1).to(torch.int32)
    held = _spaced(b, c["history"] // 3, c["history"])
    i = {"logits": r(rows, v, scale=3.0, dtype=torch.float16 if c["half"] else torch.float32),
         "history": tokens(b, max(c["history"], 1) + 7), "history_count": _ints(held), "prompt_count": _ints([h // 2 for h in held]),
         "repetition": 1.0 + 0.3 * r.unit(b), "frequency": 0.5 * r.unit(b), "presence": 0.5 * r.unit(b)}
    if c["nodes"]:
        i["token_offsets"], i["node_tokens"] = _ints(_offsets(new)), tokens(rows)
        i["mask"] = _mask(c, _grown(seed, new), rows)
    if c["bias"]:
        i["bias_ids"], i["bias_values"] = tokens(b, c["bias"]), r(b, c["bias"], scale=2.0, dtype=torch.float32)
        i["bias_count"] = _ints(_spaced(b, c["bias"] // 2, c["bias"]))
    if c["masks"] != "none":
        n, words = max(1, rows - rows // 4), -(-v // 32)
        keep = (0.97, 0.4) if c["masks"] == "open" else (0.003, 0.001)  # a share of tokens in each grammar's state
        bits = torch.zeros((n, words * 32), dtype=torch.bool, device=DEVICE)
        bits[:, :v] = r.unit(n, v) < torch.linspace(keep[0], keep[1], n, device=DEVICE)[:, None]
        i["allowed"] = (bits.view(n, words, 32).long() << torch.arange(32, device=DEVICE)).sum(-1).to(torch.int32)
        i["allowed_index"] = ((r.unit(rows) * (n + 1)).long() - 1).clamp(-1, n - 1).to(torch.int32)  # -1: no grammar
    return i


def _inputs_accept(c: dict, seed: int) -> dict:
    r, rng, hk, d, layers = _Rand(seed), random.Random(seed), c["kv_heads"], c["head_dim"], c["layers"]
    new = _new(c)
    rows, parents = sum(new), _grown(seed, new)
    tokens, targets = [], []
    for tree in parents:
        mine = [rng.randrange(0, 1000) for _ in tree]
        children = [[] for _ in tree]
        for i, p in enumerate(tree):
            if p >= 0:
                children[p].append(i)
        tokens += mine
        targets += [mine[rng.choice(k)] if k and rng.randrange(100) < c["agree"] else rng.randrange(0, 1000) for k in children]
    held = [37 * (b + 1) % 2000 for b in range(c["batch"])]
    pages = [-(-(h % PAGE + n) // PAGE) for h, n in zip(held, new)]
    order, slots, at = r.pages(sum(pages) + 3).tolist(), [], 0
    for h, n, p in zip(held, new, pages):
        slots += [order[at + (h % PAGE + j) // PAGE] * PAGE + (h + j) % PAGE for j in range(n)]
        at += p
    shape = (layers, sum(pages) + 3, PAGE, hk, d)
    return {"parents": _ints([p for tree in parents for p in tree]), "node_tokens": _ints(tokens), "targets": _ints(targets),
            "token_offsets": _ints(_offsets(new)), "seq_held": _ints(held), "slots": _ints(slots, torch.int64),
            "k": r(layers, rows, hk, d), "v": r(layers, rows, hk, d), "hot_k": r(*shape), "hot_v": r(*shape),
            "history": torch.full((c["batch"], 2200), -1, dtype=torch.int32, device=DEVICE), "history_count": _ints(held),
            "depth": max([max(x) for x in _depths(parents) if x] + [0])}


_INPUTS = {"tables": _inputs_tables, "tree": _inputs_tree, "logits": _inputs_logits, "accept": _inputs_accept}


def prepare(case: dict, seed: int) -> dict:
    st = {"case": case, **_INPUTS[case["kind"]](case, seed)}
    b = case["batch"]

    def out(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device=DEVICE)
    if case["kind"] == "tables":
        rows = st["rows"]
        st.update(seq_hot=out(b), pages_out=out(b), token_offsets=out(b + 1), next=out(1), slots=out(rows, dtype=torch.int64),
                  positions=out(rows))
        if case["tree"]:
            st["mask"] = out(rows, _mask_words(case))
    elif case["kind"] == "tree":
        st["out"] = out(*st["q"].shape, dtype=torch.float16)
    elif case["kind"] == "logits":
        st["out"], st["best"] = torch.empty_like(st["logits"]), out(st["logits"].shape[0]) if case["best"] else None
    else:
        st.update(accepted=out(b), next_token=out(b), seq_hot=out(b), path=out(st["k"].shape[1]), count_out=out(b))
    return st


# ---------------------------------------------------------------- one pass, in the plain form


def _bits(mask: torch.Tensor, n: int) -> torch.Tensor:
    """[..][words] -> truth values [..][n]."""
    b = (mask[..., None] >> torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1
    return b.flatten(-2)[..., :n].bool()


def _padded(offsets: torch.Tensor, n: int):
    """Row numbers [batch][n] of each sequence's rows and which of them it has."""
    at = offsets[:-1].long()[:, None] + torch.arange(n, device=DEVICE)
    return at, at < offsets[1:].long()[:, None]


def _plain_tables(st: dict) -> dict:
    c, rows, b = st["case"], st["rows"], st["case"]["batch"]
    held, new, pages = st["seq_held"].long(), st["seq_new"].long(), st["seq_pages"].long()
    first, zero = st["first"].long(), torch.zeros(1, dtype=torch.int64, device=DEVICE)
    ends = new.cumsum(0)
    off = torch.cat([zero, ends])
    after = torch.maximum(pages, (held + new + PAGE - 1) // PAGE)
    taken = torch.cat([zero, (after - pages).cumsum(0)])
    st["seq_hot"].copy_(held + new)
    st["pages_out"].copy_(after)
    st["token_offsets"].copy_(off)
    st["next"].copy_(first + taken[-1:])
    col = torch.arange(st["refs"].shape[1], device=DEVICE)
    at = (first + taken[:-1])[:, None] + (col - pages[:, None])
    fresh = (col >= pages[:, None]) & (col < after[:, None])
    got = st["free"][at.clamp(0, st["free"].numel() - 1)]
    st["refs"].copy_(torch.where(fresh, got, st["refs"]))
    t = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(ends, t, right=True)
    real, seq = seq < b, seq.clamp(max=b - 1)
    i = t - off[seq]
    place = held[seq] + i
    page = st["refs"][seq, (place // PAGE).clamp(max=st["refs"].shape[1] - 1)].long()
    st["slots"].copy_(torch.where(real, page * PAGE + place % PAGE, -1))
    got = {k: st[k] for k in ("refs", "seq_hot", "pages_out", "token_offsets", "next", "slots", "positions")}
    if not c["tree"]:
        st["positions"].copy_(torch.where(real, place, 0))
        return got
    n = c["new"]
    row, has = _padded(off, n)
    parent = torch.where(has, st["parents"].long()[row.clamp(max=rows - 1)], -1)
    node = torch.arange(n, device=DEVICE)
    sees = ((parent[..., None] == node) | (node[:, None] == node)).float()  # itself and its parent
    for _ in range(max(1, (n - 1).bit_length())):
        sees = (torch.matmul(sees, sees) > 0).float()
    words = st["mask"].shape[1]
    bits = torch.zeros((b, n, words * 32), dtype=torch.int64, device=DEVICE)
    bits[..., :n] = sees.long()
    packed = (bits.view(b, n, words, 32) << torch.arange(32, device=DEVICE)).sum(-1).to(torch.int32)
    mine = i.clamp(0, n - 1)
    st["mask"].copy_(torch.where(real[:, None], packed[seq, mine], 0))
    st["positions"].copy_(torch.where(real, held[seq] + sees.sum(-1).long()[seq, mine] - 1, 0))
    return {**got, "mask": st["mask"]}


def _plain_tree(st: dict) -> torch.Tensor:
    c = st["case"]
    b, n, hq, hk, d = c["batch"], c["nodes"], c["q_heads"], c["kv_heads"], c["head_dim"]
    group = hq // hk
    at, has = _padded(st["token_offsets"], n)
    at = at.clamp(max=st["q"].shape[0] - 1)
    # Rows [kv_heads][batch][nodes * group][head_dim].
    q = st["q"][at].float().view(b, n, hk, group, d).permute(2, 0, 1, 3, 4).reshape(hk, b, n * group, d) / math.sqrt(d)
    refs = st["refs"].long()
    pk = st["hot_k"][refs].flatten(1, 2).permute(2, 0, 1, 3).float().contiguous()
    pv = st["hot_v"][refs].flatten(1, 2).permute(2, 0, 1, 3).float().contiguous()
    nk, nv = (st[x][at].permute(2, 0, 1, 3).float().contiguous() for x in ("k", "v"))
    sp = torch.matmul(q, pk.transpose(2, 3).contiguous())
    sn = torch.matmul(q, nk.transpose(2, 3).contiguous())
    sp.masked_fill_(torch.arange(sp.shape[-1], device=DEVICE) >= st["seq_held"].long()[:, None, None], -math.inf)
    if c["chain"]:
        node = torch.arange(n, device=DEVICE)
        sees = (node <= node[:, None]).expand(b, n, n)
    else:
        sees = _bits(st["mask"], n)[at]
    sees = sees & has[:, None, :]
    sn.masked_fill_(~sees.repeat_interleave(group, 1), -math.inf)
    top = torch.maximum(sp.amax(-1, keepdim=True), sn.amax(-1, keepdim=True))
    sp, sn = (sp - top).exp(), (sn - top).exp()
    out = (torch.matmul(sp, pv) + torch.matmul(sn, nv)) / (sp.sum(-1, keepdim=True) + sn.sum(-1, keepdim=True))
    out = out.view(hk, b, n, group, d).permute(1, 2, 0, 3, 4).reshape(b, n, hq, d).to(torch.float16)
    st["out"][at[has]] = out[has]
    return st["out"]


def _plain_logits(st: dict) -> dict:
    c, v, b = st["case"], st["case"]["vocab"], st["case"]["batch"]
    x = st["logits"].float()
    rows = x.shape[0]
    place, ids = torch.arange(st["history"].shape[1], device=DEVICE), st["history"].long()
    held, prompt = st["history_count"].long()[:, None], st["prompt_count"].long()[:, None]

    def count(which):
        return torch.zeros((b, v), dtype=torch.float32, device=DEVICE).scatter_add_(1, ids, which.float())
    old, made = count(place < torch.minimum(prompt, held)), count((place >= prompt) & (place < held))
    seq = torch.arange(rows, device=DEVICE)
    if c["nodes"]:
        off = st["token_offsets"].long()
        seq = torch.searchsorted(off[1:].contiguous(), seq, right=True)
        n = c["nodes"]
        at = off[seq][:, None] + torch.arange(n, device=DEVICE)
        sees = _bits(st["mask"], n) & (at < off[seq + 1][:, None])
        made = made[seq].scatter_add_(1, st["node_tokens"].long()[at.clamp(max=rows - 1)], sees.float())
    else:
        made = made[seq]
    r, f, p = (st[k][seq][:, None] for k in ("repetition", "frequency", "presence"))
    x = torch.where((old[seq] > 0) | (made > 0), torch.where(x > 0, x / r, x * r), x)
    x = x - f * made
    x = torch.where(made > 0, x - p, x)
    if c["bias"]:
        n = c["bias"]
        entry = torch.arange(1, n + 1, device=DEVICE).expand(b, n)
        entry = torch.where(entry <= st["bias_count"].long()[:, None], entry, 0)
        last = torch.zeros((b, v), dtype=torch.int64, device=DEVICE).scatter_reduce_(1, st["bias_ids"].long(), entry, "amax")
        add = torch.cat([torch.zeros((b, 1), device=DEVICE), st["bias_values"]], 1).gather(1, last)
        x = torch.where(last[seq] > 0, x + add[seq], x)
    if c["masks"] != "none":
        which = st["allowed_index"].long()
        ok = _bits(st["allowed"], v)[which.clamp(min=0)] | (which < 0)[:, None]
        x = x.masked_fill(~ok, -math.inf)
    st["out"].copy_(x)
    if not c["best"]:
        return {"logits": st["out"]}
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device=DEVICE), v).amin(-1)
    st["best"].copy_(torch.where(top[:, 0] > -math.inf, first, -1))
    return {"logits": st["out"], "best": st["best"]}


def _plain_accept(st: dict) -> dict:
    c, n, rows = st["case"], st["case"]["nodes"], st["k"].shape[1]
    b = c["batch"]
    at, has = _padded(st["token_offsets"], n)
    at = at.clamp(max=rows - 1)
    parent = torch.where(has, st["parents"].long()[at], -2)
    token, target = st["node_tokens"].long()[at], st["targets"].long()[at]
    node, lane = torch.arange(n, device=DEVICE), torch.arange(b, device=DEVICE)
    cur = torch.where(has[:, 0], 0, -1)
    kept, steps = cur, [cur]
    for _ in range(st["depth"]):
        want = target[lane, cur.clamp(min=0)]
        child = (parent == cur[:, None]) & (token == want[:, None]) & (cur >= 0)[:, None]
        nxt = torch.where(child, node, n).amin(-1)
        cur = torch.where(nxt < n, nxt, -1)
        kept = torch.where(cur >= 0, cur, kept)
        steps.append(cur)
    steps = torch.stack(steps, 1)
    accepted = (steps >= 0).sum(1)
    st["accepted"].copy_(accepted)
    st["next_token"].copy_(torch.where(kept >= 0, target[lane, kept.clamp(min=0)], -1))
    st["seq_hot"].copy_(st["seq_held"].long() + accepted)
    m = min(steps.shape[1], n)
    full = torch.full((b, n), -1, dtype=torch.int64, device=DEVICE)
    full[:, :m] = steps[:, :m]
    st["path"].fill_(-1)
    st["path"][at[has]] = full[has].to(torch.int32)
    keep = full >= 0
    src = (st["token_offsets"].long()[:-1, None] + full)[keep]
    dst = st["slots"][at[keep]]
    for x in ("k", "v"):
        st["hot_" + x].flatten(1, 2)[:, dst] = st[x][:, src]
    start = st["history_count"].long()[:, None] + node
    st["history"][lane[:, None].expand(b, n)[keep], start[keep]] = token[lane[:, None].expand(b, n)[keep], full[keep]].to(torch.int32)
    st["count_out"].copy_(st["history_count"].long() + accepted)
    return {k: st[k] for k in ("accepted", "next_token", "seq_hot", "path", "history", "count_out", "hot_k", "hot_v")}


# ---------------------------------------------------------------- one pass, by the framework's operators

_engines: dict = {}


def _ops():
    """The engine of the process, as a program keeps one per GPU."""
    if not _engines:
        from aether_nexus_amd.ops import OpsEngine
        _engines["ops"] = OpsEngine()
    return _engines["ops"]


def _request(st: dict):
    """The descriptor of a state's call, which a program keeps for as long as it calls with these tensors."""
    from aether_nexus_amd import ops
    c = st["case"]
    if c["kind"] == "tables":
        return ops.make_tables_desc(batch=c["batch"], num_tokens=st["rows"], seq_held=st["seq_held"], seq_new=st["seq_new"],
                                    seq_pages=st["seq_pages"], free_pages=st["free"], free_first=st["first"], refs=st["refs"],
                                    seq_hot=st["seq_hot"], pages_out=st["pages_out"], token_offsets=st["token_offsets"],
                                    free_next=st["next"], slots=st["slots"], positions=st["positions"], parents=st.get("parents"),
                                    tree_mask=st.get("mask"))
    if c["kind"] == "tree":
        return ops.make_tree_desc(batch=c["batch"], num_tokens=st["q"].shape[0], q_heads=c["q_heads"], kv_heads=c["kv_heads"],
                                  head_dim=c["head_dim"], q=st["q"], k=st["k"], v=st["v"], out=st["out"], hot_k=st["hot_k"],
                                  hot_v=st["hot_v"], refs=st["refs"], seq_held=st["seq_held"], token_offsets=st["token_offsets"],
                                  tree_mask=st.get("mask"), scale=c["head_dim"] ** -0.5)
    if c["kind"] == "logits":
        names = ("history", "history_count", "prompt_count", "repetition", "frequency", "presence", "token_offsets", "node_tokens",
                 "bias_ids", "bias_values", "bias_count", "allowed", "allowed_index", "best")
        return ops.make_logits_desc(batch=c["batch"], num_tokens=st["logits"].shape[0], vocab_size=c["vocab"], logits=st["logits"],
                                    out=st["out"], tree_mask=st.get("mask"), **{k: st[k] for k in names if st.get(k) is not None})
    return ops.make_accept_desc(batch=c["batch"], num_tokens=st["k"].shape[1], layers=c["layers"], kv_heads=c["kv_heads"],
                                head_dim=c["head_dim"], parents=st["parents"], node_tokens=st["node_tokens"], targets=st["targets"],
                                token_offsets=st["token_offsets"], seq_held=st["seq_held"], slots=st["slots"], k=st["k"], v=st["v"],
                                hot_k=st["hot_k"], hot_v=st["hot_v"], accepted=st["accepted"], next_token=st["next_token"],
                                seq_hot=st["seq_hot"], path=st["path"], history=st["history"], history_count=st["history_count"],
                                history_count_out=st["count_out"])


def run(state: dict):
    st, kind = state, state["case"]["kind"]
    if not own:
        return {"tables": _plain_tables, "tree": _plain_tree, "logits": _plain_logits, "accept": _plain_accept}[kind](st)
    ops = _ops()
    if "desc" not in st:
        st["desc"] = _request(st)
    if kind == "tables":
        ops.page_tables(st["desc"])
        names = ("refs", "seq_hot", "pages_out", "token_offsets", "next", "slots", "positions", "mask")
        return {k: st[k] for k in names if k in st}
    if kind == "tree":
        ops.tree_attention(st["desc"])
        return st["out"]
    if kind == "logits":
        ops.adjust_logits(st["desc"])
        return {"logits": st["out"], "best": st["best"]} if st["case"]["best"] else {"logits": st["out"]}
    ops.accept_tree(st["desc"])
    return {k: st[k] for k in ("accepted", "next_token", "seq_hot", "path", "history", "count_out", "hot_k", "hot_v")}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    c, b = case, case["batch"]
    new = _new(c)
    rows = sum(new) + c.get("pad", 0)
    if c["kind"] == "tables":
        pages = sum(-(-n // PAGE) for n in new)
        per_token = 12 + ((4 + 4 * _mask_words(c)) if c["tree"] else 0)
        return {"bytes": 24 * b + 8 * pages + per_token * rows, "flops": rows}
    if c["kind"] == "tree":
        hq, hk, d, held = c["q_heads"], c["kv_heads"], c["head_dim"], _held(c)
        return {"bytes": 2 * (2 * (sum(held) + sum(new)) * hk * d + 2 * sum(new) * hq * d) + sum(held) // 4,
                "flops": 4 * hq * d * sum(n * (h + 1) for n, h in zip(new, held))}
    if c["kind"] == "logits":
        size = 2 if c["half"] else 4
        masks = rows * c["vocab"] // 8 if c["masks"] != "none" else 0
        return {"bytes": 2 * size * rows * c["vocab"] + masks + 4 * sum(_spaced(b, c["history"] // 3, c["history"])) + 8 * b * c["bias"],
                "flops": rows * c["vocab"]}
    row = 2 * c["layers"] * c["kv_heads"] * c["head_dim"] * 2
    # The root of each tree and, by the way trees grow here, a step or more for each doubling of its nodes.
    kept = sum(1 + c["agree"] / 100 * math.log2(n) for n in new)
    return {"bytes": int(2 * row * kept) + 16 * rows + 24 * b, "flops": rows}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_tree(c: dict, seed: int) -> torch.Tensor:
    i = _inputs_tree(c, seed)
    hq, hk, d, group = c["q_heads"], c["kv_heads"], c["head_dim"], c["q_heads"] // c["kv_heads"]
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device=DEVICE)
    sets = None if c["chain"] else _sees(_grown(seed, _new(c)))
    at = 0
    for b, (n, h) in enumerate(zip(_new(c), _held(c))):
        pages = i["refs"][b, :-(-h // PAGE)].long()
        k, v = (torch.cat([i["hot_" + x][pages].flatten(0, 1)[:h], i[x][at:at + n]]).double().transpose(0, 1) for x in ("k", "v"))
        hidden = torch.tensor([[(j > x) if sets is None else not (sets[b][x] >> j) & 1 for j in range(n)] for x in range(n)],
                              dtype=torch.bool, device=DEVICE)
        hidden = torch.cat([torch.zeros((n, h), dtype=torch.bool, device=DEVICE), hidden], 1)
        q = i["q"][at:at + n].double().view(n, hk, group, d)
        for g in range(hk):
            s = torch.matmul(q[:, g].reshape(n * group, d), k[g].t().contiguous()) / math.sqrt(d)
            s = s.view(n, group, h + n).masked_fill(hidden[:, None], -math.inf)
            o = torch.matmul(torch.softmax(s, -1).view(n * group, h + n), v[g].contiguous())
            out[at:at + n, g * group:(g + 1) * group] = o.view(n, group, d)
        at += n
    return out


def _exact_logits(c: dict, seed: int) -> dict:
    i, v, row = _inputs_logits(c, seed), c["vocab"], 0
    out = torch.empty(i["logits"].shape, dtype=torch.float64, device=DEVICE)
    new = _new(c)
    sets = _sees(_grown(seed, new)) if c["nodes"] else None
    for b, n in enumerate(new):
        held = int(i["history_count"][b])
        prompt, answer = i["history"][b, :held // 2].long(), i["history"][b, held // 2:held].long()
        first = row
        for node in range(n):
            ids = answer
            if sets:
                mine = [first + j for j in range(n) if (sets[b][node] >> j) & 1]
                ids = torch.cat([answer, i["node_tokens"][mine].long()])
            made = torch.bincount(ids, minlength=v).double()
            x = i["logits"][row].double()
            seen = made > 0
            seen[prompt] = True
            r = i["repetition"][b].double()
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
            x = x - i["frequency"][b].double() * made - i["presence"][b].double() * (made > 0)
            if c["bias"]:
                last = {}
                for e, t in enumerate(i["bias_ids"][b, :int(i["bias_count"][b])].tolist()):
                    last[t] = e
                x[list(last)] += i["bias_values"][b][list(last.values())].double()
            if c["masks"] != "none" and int(i["allowed_index"][row]) >= 0:
                words = i["allowed"][int(i["allowed_index"][row])].long() & 0xFFFFFFFF
                t = torch.arange(v, device=DEVICE)
                x[(words[t // 32] >> (t % 32)) % 2 == 0] = -math.inf
            out[row] = x
            row += 1
    return {"logits": out, "best": None} if c["best"] else {"logits": out}


def _exact_accept(c: dict, seed: int) -> dict:
    i, at = _inputs_accept(c, seed), 0
    k_pool, v_pool = i["hot_k"].double().flatten(1, 2), i["hot_v"].double().flatten(1, 2)
    parents, tokens, targets = (i[x].tolist() for x in ("parents", "node_tokens", "targets"))
    for n in _new(c):
        path = [0]
        while True:
            nxt = [j for j in range(n) if parents[at + j] == path[-1] and tokens[at + j] == targets[at + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        for j, node in enumerate(path):
            slot = int(i["slots"][at + j])
            k_pool[:, slot], v_pool[:, slot] = i["k"][:, at + node].double(), i["v"][:, at + node].double()
        at += n
    names = ("accepted", "next_token", "seq_hot", "path", "history", "count_out")
    return {**{x: None for x in names}, "hot_k": k_pool.view(i["hot_k"].shape), "hot_v": v_pool.view(i["hot_v"].shape)}


def exact(case: dict, seed: int):
    if case["kind"] == "tables":
        return None
    return {"tree": _exact_tree, "logits": _exact_logits, "accept": _exact_accept}[case["kind"]](case, seed)
