"""A step over trees of drafted tokens as it runs: page tables, every layer's attention, adjusted logits and the
accepted tree, each of what the calls before it left on cuda:0, for several steps; each call against
oracle/step_oracle.py on the same inputs, and the same steps from one captured graph."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import prefix_errors
from oracle import step_oracle as S

pytestmark = pytest.mark.gpu

LAYERS, HQ, HK, VOCAB, PAGES, HISTORY = 2, 8, 2, 500, 24, 200
BATCH = 4
NODES = [10, 4, 1, 10]  # of the sequences' trees
PARENTS = [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3]
PAD = 2
ROWS = sum(NODES) + PAD


class Run:
    """Sequences that generate: a draft model that is a table of the three tokens after each token, a grammar that
    allows those and one more, a model whose rows are tables of tokens and positions."""

    def __init__(self, hd):
        import torch
        self.hd = hd
        rng = np.random.default_rng(hd)
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.drafts = cuda(np.stack([rng.permutation(VOCAB)[:3] for _ in range(VOCAB)]))
        allowed = np.zeros((VOCAB, 16 * 32), dtype=np.uint8)
        for t in range(VOCAB):
            allowed[t, self.drafts[t].cpu().numpy()] = 1
            allowed[t, rng.integers(0, VOCAB)] = 1
        self.allowed_host = np.packbits(allowed, axis=1, bitorder="little").view("<u4")
        self.allowed = cuda(self.allowed_host.astype(np.int64)).to(torch.int32)
        heads = HQ + 2 * HK
        self.embed = cuda((rng.standard_normal((LAYERS, VOCAB, heads, hd))).astype(np.float32))
        self.turn = cuda((1 + 0.2 * rng.standard_normal((PAGES * 16, 1, 1))).astype(np.float32))
        self.head = cuda((rng.standard_normal((HQ * hd, VOCAB)) * 0.1).astype(np.float32))
        order = rng.permutation(BATCH * PAGES + 5)
        held = [0, 17, 16, 30]
        self.prompts = [rng.integers(0, VOCAB, h) for h in held]
        i32 = lambda a: cuda(np.asarray(a, dtype=np.int64)).to(torch.int32)
        self.held, self.pages = i32(held), i32([-(-h // 16) for h in held])
        refs = np.full((BATCH, PAGES), 0x7FFFFFFF, dtype=np.int64)
        at = 0
        for b, h in enumerate(held):
            refs[b, :-(-h // 16)] = order[at:at + -(-h // 16)]
            at += -(-h // 16)
        self.refs, self.free, self.first = i32(refs), i32(order[at:]), i32([0])
        self.blocks = BATCH * PAGES + 5
        f16 = dict(dtype=torch.float16, device="cuda:0")
        self.hot_k, self.hot_v = (torch.full((LAYERS, self.blocks, 16, HK, hd), float("nan"), **f16) for _ in range(2))
        for b, h in enumerate(held):
            for p in range(h):
                rows = (self.embed[:, int(self.prompts[b][p])] * self.turn[p]).half()
                self.hot_k[:, int(refs[b, p // 16]), p % 16] = rows[:, HQ:HQ + HK]
                self.hot_v[:, int(refs[b, p // 16]), p % 16] = rows[:, HQ + HK:]
        self.new, self.parents = i32(NODES), i32([p for n in NODES for p in PARENTS[:n]] + [-1] * PAD)
        self.token = i32(rng.integers(0, VOCAB, BATCH))
        # The history holds the tokens in pages; a tree's first node joins it when it is kept.
        history = np.zeros((BATCH, HISTORY), dtype=np.int64)
        for b, p in enumerate(self.prompts):
            history[b, :len(p)] = p
        self.history, self.count, self.prompt = i32(history), i32(held), i32(held)
        self.penalty = [cuda(np.asarray(x, dtype=np.float32)) for x in ([1.1, 1.0, 1.3, 1.2], [0.1, 0.2, 0.0, 0.4], [0.0, 0.3, 0.1, 0.2])]
        new = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device="cuda:0")
        self.seq_hot, self.pages_out, self.offsets, self.next_first = new(BATCH), new(BATCH), new(BATCH + 1), new(1)
        self.slots, self.positions, self.mask = new(ROWS, dtype=torch.int64), new(ROWS), new(ROWS, 1)
        self.nodes = new(ROWS)
        self.rows = new(LAYERS, ROWS, heads, hd, dtype=torch.float16)
        self.out = new(LAYERS, ROWS, HQ, hd, dtype=torch.float16)
        self.logits = new(ROWS, VOCAB, dtype=torch.float32)
        self.best, self.accepted, self.following, self.path, self.after = new(ROWS), new(BATCH), new(BATCH), new(ROWS), new(BATCH)
        self.level = torch.zeros(ROWS, dtype=torch.int64, device="cuda:0")
        child, owner = [], []
        for b, n in enumerate(NODES):
            seen = {}
            for i in range(n):
                seen[PARENTS[i]] = seen.get(PARENTS[i], -1) + 1
                child.append((sum(NODES[:b]) + PARENTS[i] if i else 0, seen[PARENTS[i]], i))
                owner.append(b)
        self.owner = cuda(np.array(owner))
        # Rows at depth 1 and 2: their parents' rows, which of the three drafts they are.
        depth = [0 if i == 0 else 1 if PARENTS[i] == 0 else 2 for _, _, i in child]
        self.depths = [[cuda(np.array([t for t in range(len(child)) if depth[t] == x])), cuda(np.array([child[t][0] for t in range(len(child)) if depth[t] == x])),
                        cuda(np.array([child[t][1] for t in range(len(child)) if depth[t] == x]))] for x in range(3)]
        from aether_nexus_amd import ops as O
        self.d_tables = O.make_tables_desc(batch=BATCH, num_tokens=ROWS, seq_held=self.held, seq_new=self.new, seq_pages=self.pages, refs=self.refs,
                                           free_pages=self.free, free_first=self.first, seq_hot=self.seq_hot, pages_out=self.pages_out,
                                           token_offsets=self.offsets, free_next=self.next_first, slots=self.slots, positions=self.positions,
                                           parents=self.parents, tree_mask=self.mask)
        k, v = self.rows[:, :, HQ:HQ + HK], self.rows[:, :, HQ + HK:]
        self.d_tree = [O.make_tree_desc(batch=BATCH, num_tokens=ROWS, q_heads=HQ, kv_heads=HK, head_dim=hd, q=self.rows[l, :, :HQ], k=k[l], v=v[l],
                                        out=self.out[l], hot_k=self.hot_k[l], hot_v=self.hot_v[l], refs=self.refs, hot_count=PAGES, seq_held=self.held,
                                        token_offsets=self.offsets, tree_mask=self.mask) for l in range(LAYERS)]
        self.d_logits = O.make_logits_desc(num_tokens=ROWS, vocab_size=VOCAB, batch=BATCH, logits=self.logits, out=self.logits, best=self.best,
                                           token_offsets=self.offsets, history=self.history, history_count=self.count, prompt_count=self.prompt,
                                           repetition=self.penalty[0], frequency=self.penalty[1], presence=self.penalty[2], node_tokens=self.nodes,
                                           tree_mask=self.mask, allowed=self.allowed, allowed_index=self.nodes)
        self.d_accept = O.make_accept_desc(batch=BATCH, num_tokens=ROWS, layers=LAYERS, kv_heads=HK, head_dim=hd, parents=self.parents,
                                           node_tokens=self.nodes, targets=self.best, token_offsets=self.offsets, seq_held=self.held, slots=self.slots,
                                           k=k, v=v, hot_k=self.hot_k, hot_v=self.hot_v, accepted=self.accepted, next_token=self.following,
                                           seq_hot=self.after, path=self.path, history=self.history, history_count=self.count,
                                           history_count_out=self.count)

    def step(self, ops, look=None):
        look = look or (lambda what: None)
        look("begin")
        ops.page_tables(self.d_tables)
        look("tables")
        at, _, _ = self.depths[0]
        self.nodes[at] = self.token
        for at, above, which in self.depths[1:]:
            self.nodes[at] = self.drafts[self.nodes[above].long(), which].int()
        self.rows.copy_(self.embed[:, self.nodes.long()] * self.turn[self.positions.long()])
        for l, d in enumerate(self.d_tree):
            ops.tree_attention(d)
        look("attention")
        self.logits.copy_(self.out[-1].reshape(ROWS, HQ * self.hd).float() @ self.head)
        look("scores")
        ops.adjust_logits(self.d_logits)
        look("logits")
        ops.accept_tree(self.d_accept)
        look("accepted")
        self.held.copy_(self.after)  # pages that the step took and did not fill stay the sequence's
        self.pages.copy_(self.pages_out)
        self.first.copy_(self.next_first)
        self.token.copy_(self.following)

    def state(self):
        import torch
        torch.cuda.synchronize()
        return [x.cpu().numpy().copy() for x in (self.held, self.pages, self.first, self.token, self.refs, self.history, self.count, self.path, self.best)] + \
            [x.view(torch.int16).cpu().numpy().copy() for x in (self.hot_k, self.hot_v, self.out[:, :sum(NODES)])]


class Watch:
    """Compares each call of a step with the oracle."""

    def __init__(self, run):
        self.run, self.kept = run, 0

    def __call__(self, what):
        import torch
        torch.cuda.synchronize()
        r = self.run
        cpu = lambda t: t.cpu().numpy()
        if what == "begin":
            self.refs, self.held, self.pages, self.first = cpu(r.refs).astype(np.int64), cpu(r.held), cpu(r.pages), int(r.first[0])
            self.hot_k, self.hot_v = cpu(r.hot_k), cpu(r.hot_v)
            self.history, self.count = cpu(r.history), cpu(r.count)
        elif what == "tables":
            want = S.page_tables(self.refs, self.held, NODES, self.pages, cpu(r.free), self.first, ROWS, PAGES, parents=cpu(r.parents), words=1)
            assert not want["errors"]
            for name, t in (("refs", r.refs), ("seq_hot", r.seq_hot), ("pages_out", r.pages_out), ("token_offsets", r.offsets), ("free_next", r.next_first),
                            ("slots", r.slots), ("positions", r.positions), ("tree_mask", r.mask)):
                w = np.asarray(want[name]).astype(np.int64)
                assert np.array_equal(cpu(t).astype(np.int64).reshape(w.shape), w), name
        elif what == "attention":
            n, rows = sum(NODES), cpu(r.rows)
            for l in range(LAYERS):
                want, absolute, total = S.tree_attention(rows[l, :, :HQ], rows[l, :, HQ:HQ + HK], rows[l, :, HQ + HK:], self.hot_k[l], self.hot_v[l],
                                                         cpu(r.refs).astype(np.int64), self.held, cpu(r.offsets), cpu(r.mask).view(np.uint32), r.hd ** -0.5)
                worst, _ = prefix_errors(cpu(r.out[l])[:n], want[:n], absolute[:n], total[:n], int(self.held.max()) + 10, 16.0)
                assert worst <= 1.0, l
        elif what == "scores":
            self.scores = cpu(r.logits)
        elif what == "logits":
            n = sum(NODES)
            x, best = S.adjust_logits(self.scores, offsets=cpu(r.offsets), history=self.history, history_count=self.count, prompt_count=cpu(r.prompt),
                                      repetition=cpu(r.penalty[0]), frequency=cpu(r.penalty[1]), presence=cpu(r.penalty[2]), node_tokens=cpu(r.nodes),
                                      mask=cpu(r.mask).view(np.uint32), allowed=r.allowed_host, allowed_index=cpu(r.nodes))
            assert np.array_equal(cpu(r.logits)[:n], x[:n].astype(np.float32)) and cpu(r.best)[:n].tolist() == best[:n].tolist()
        elif what == "accepted":
            paths = S.accept_tree(cpu(r.parents), cpu(r.nodes), cpu(r.best), cpu(r.offsets))
            assert cpu(r.accepted).tolist() == [len(p) for p in paths] and cpu(r.after).tolist() == [int(h) + len(p) for h, p in zip(self.held, paths)]
            rows, slots, offsets = cpu(r.rows), cpu(r.slots), cpu(r.offsets)
            for b, p in enumerate(paths):
                for j, node in enumerate(p):
                    s = slots[offsets[b] + j]
                    self.hot_k[:, s // 16, s % 16] = rows[:, offsets[b] + node, HQ:HQ + HK]
                    self.hot_v[:, s // 16, s % 16] = rows[:, offsets[b] + node, HQ + HK:]
                    self.history[b, self.count[b] + j] = cpu(r.nodes)[offsets[b] + node]
                self.kept += len(p)
            assert np.array_equal(cpu(r.hot_k).view(np.int16), self.hot_k.view(np.int16))
            assert np.array_equal(cpu(r.hot_v).view(np.int16), self.hot_v.view(np.int16))
            assert np.array_equal(cpu(r.history), self.history)
            assert cpu(r.following).tolist() == [int(cpu(r.best)[offsets[b] + p[-1]]) for b, p in enumerate(paths)]


@pytest.fixture(scope="module")
def ops(engine):
    from aether_nexus_amd.ops import OpsEngine
    return OpsEngine(engine)


@pytest.mark.parametrize("hd", [64, 128])
def test_steps_of_generation(ops, engine, hd):
    run = Run(hd)
    watch = Watch(run)
    for i in range(8):
        run.step(ops, watch)
        print(f"step {i}: {watch.kept} tokens kept", flush=True)
    engine.check_device_errors()
    assert watch.kept > 8 * BATCH  # some drafts were kept


@pytest.mark.parametrize("hd", [64, 128])
def test_steps_from_one_graph(ops, engine, hd):
    """The calls read all lengths on the device: one graph runs every step."""
    import torch
    eager, captured = Run(hd), Run(hd)
    eager.step(ops)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        captured.step(ops)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step(ops)
    for i in range(8):
        eager.step(ops)
        graph.replay()
        for x, y in zip(eager.state(), captured.state()):
            assert np.array_equal(x, y), i
    engine.check_device_errors()
