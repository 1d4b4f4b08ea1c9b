"""Batched speculative decoding with drafted token trees over a paged K/V cache: a small decoder that
runs the tree-verification operators together as a server would.

    python -m g4dense_b200.tree_decode [--sequences 4] [--tokens 32] [--temperature 0]

The model is a toy of the library's own parts (two layers of INT4 G64 projections, grouped-query
attention, random weights); what it shows is the round:

    draft a tree per sequence -> every layer: g4b_tree_attention over the pages and the tree
    -> g4b_sample_rows for every node -> g4b_tree_accept -> g4b_pages_reserve -> g4b_pages_commit

Prompts go through the same attention as chains of nodes; `fork` shares a prompt's pages between
continuations, `finish` releases them. The operators of a round wait for nothing on the host. This decoder
does: its drafter lives there, so that every round uploads the trees and reads the accepted tokens back.
"""
from __future__ import annotations

import argparse

import numpy as np

from . import api


class Model:
    """Random weights: dim 256, 4 query heads on 2 K/V heads of 64, FFN 512, a 4096-token vocabulary."""

    dim, heads, kv_heads, head_dim, ffn, vocab, layers = 256, 4, 2, 64, 512, 4096, 2

    def __init__(self, seed=0):
        import torch
        g = torch.Generator().manual_seed(seed)

        def matrix(n, k):
            words = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
            scale = torch.full((n, k // 64), 0.25 * k ** -0.5).to(torch.bfloat16)
            bias = (-7.5 * scale.float()).to(torch.bfloat16)  # nibbles 0..15, centred
            return api.QMat(words.cuda(), scale.view(torch.int16).cuda(), bias.view(torch.int16).cuda(),
                            torch.cuda.current_stream())

        q, kv = self.heads * self.head_dim, self.kv_heads * self.head_dim
        self.embed = torch.randn(self.vocab, self.dim, generator=g).cuda()
        self.blocks = [dict(qkv=matrix(q + 2 * kv, self.dim), o=matrix(self.dim, q), up=matrix(2 * self.ffn, self.dim),
                            down=matrix(self.dim, self.ffn)) for _ in range(self.layers)]
        self.head = matrix(self.vocab, self.dim)
        half = self.head_dim // 2
        self.freq = (10000.0 ** (-torch.arange(half) / half)).cuda()


def _product(m, x):
    """x [rows][K] fp32 through a prepared matrix, 128 rows a call."""
    import torch
    out, stream = x.new_empty(x.shape[0], m.N), torch.cuda.current_stream()
    for i in range(0, x.shape[0], 128):
        m.gemm(x[i:i + 128].contiguous(), out[i:i + 128], stream)
    return out


def _norm(x):
    return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()


class Decoder:
    """Up to `seqs` sequences over one pool of pages: planes [2 * layers] of K and V rows."""

    def __init__(self, model, seqs, pages=256, page_size=16, width=16, max_nodes=32):
        import torch
        self.m, self.seqs, self.page, self.max_nodes = model, seqs, page_size, max_nodes
        i32 = dict(dtype=torch.int32, device="cuda")
        self.pool = torch.zeros(2 * model.layers, pages, page_size, model.kv_heads, model.head_dim, dtype=torch.bfloat16,
                                device="cuda")
        self.refs, self.table = torch.zeros(pages, **i32), torch.full((seqs, width), -1, **i32)
        self.lens, self.status = torch.zeros(seqs, **i32), torch.zeros(1, **i32)
        self.path, self.count, self.next = torch.zeros(seqs, max_nodes, **i32), torch.zeros(seqs, **i32), torch.zeros(seqs, **i32)
        self.held = [0] * seqs  # lens as the host knows them
        self.workspace = torch.empty(api.tree_attention_workspace(max_nodes, model.heads, model.kv_heads, model.head_dim),
                                     dtype=torch.uint8, device="cuda")

    def _forward(self, tokens, cu, mask, depth, position):
        """Logits of every node, and the rows of K and V that a commit would write."""
        import torch
        m, n = self.m, tokens.numel()
        rows = torch.empty(2 * m.layers, n, m.kv_heads, m.head_dim, dtype=torch.bfloat16, device="cuda")
        angle = position[:, None, None].float() * m.freq
        cos, sin = angle.cos(), angle.sin()

        def turn(x):
            a, b = x.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        h, out = m.embed[tokens.long()], torch.empty(n, m.heads, m.head_dim, dtype=torch.bfloat16, device="cuda")
        for i, b in enumerate(m.blocks):
            qkv = _product(b["qkv"], _norm(h)).view(n, -1, m.head_dim)
            q = turn(_norm(qkv[:, :m.heads])).to(torch.bfloat16)
            rows[2 * i] = turn(_norm(qkv[:, m.heads:m.heads + m.kv_heads]))
            rows[2 * i + 1] = qkv[:, m.heads + m.kv_heads:]
            api.tree_attention(q, self.pool[2 * i], self.pool[2 * i + 1], self.table, self.lens, rows[2 * i],
                               rows[2 * i + 1], cu, mask, out, self.workspace, max_nodes=self.max_nodes,
                               scale=m.head_dim ** -0.5, depth=depth)
            h = h + _product(b["o"], out.float().view(n, -1))
            gate, up = _product(b["up"], _norm(h)).chunk(2, -1)
            h = h + _product(b["down"], torch.nn.functional.gelu(gate, approximate="tanh") * up)
        return 4.0 * _product(m.head, _norm(h)), rows

    def _fits(self, trees, positions):
        """Refuses trees whose tokens, nodes or positions lie outside the arrays that they index on the device."""
        for s, t in enumerate(trees):
            if t is None:
                continue
            if len(t[0]) != len(t[1]) or len(t[0]) > self.max_nodes:
                raise ValueError(f"sequence {s}: {len(t[0])} tokens, {len(t[1])} parents, at most {self.max_nodes} nodes")
            if any(not 0 <= x < self.m.vocab for x in t[0]):
                raise ValueError(f"sequence {s}: a token outside the vocabulary of {self.m.vocab}")
            deepest = self.held[s] + int(api.tree_mask(t[1])[1].max(initial=0))
            if positions is not None and deepest >= positions:
                raise ValueError(f"sequence {s}: no uniform number for position {deepest}")

    def _nodes(self, trees):
        """Device arrays of the sequences' trees, each a (tokens, parents) pair (None: no nodes)."""
        import torch
        trees = [t if t is not None else ([], []) for t in trees]
        words = (self.max_nodes + 31) // 32
        masks, depths = zip(*(api.tree_mask(p, words) for _, p in trees))
        i32 = lambda x: torch.tensor(np.concatenate(x) if isinstance(x, list) else x, dtype=torch.int32, device="cuda")  # noqa: E731
        cu = np.concatenate([[0], np.cumsum([len(t) for t, _ in trees])])
        owner = torch.tensor(np.repeat(np.arange(self.seqs), np.diff(cu)), device="cuda")
        tokens = i32([np.array(t, np.int64) for t, _ in trees])
        return (tokens, i32([np.array(p, np.int64) for _, p in trees]), i32(cu),
                torch.from_numpy(np.concatenate(masks)).cuda(), i32(list(depths)), owner)

    def _grow(self):
        api.pages_reserve(self.refs, self.table, self.lens, self.count, self.page, self.refs, self.table, self.status)

    def _commit(self, rows, cu, path):
        api.pages_commit(self.pool, self.table, self.lens, rows, cu, path, self.count, self.lens, status=self.status)

    def prompt(self, prompts):
        """Caches prompts (lists of tokens, None for the sequences left alone) as chains, max_nodes at a time."""
        import torch
        for at in range(0, max(len(p) for p in prompts if p), self.max_nodes):
            parts = [p[at:at + self.max_nodes] if p else [] for p in prompts]
            trees = [(p, list(range(-1, len(p) - 1))) for p in parts]
            self._fits(trees, None)
            tokens, _, cu, mask, depth, owner = self._nodes(trees)
            _, rows = self._forward(tokens, cu, mask, depth, self.lens[owner] + depth)
            self.count.copy_(torch.tensor([len(p) for p in parts], dtype=torch.int32))
            self._grow()
            self._commit(rows, cu, None)
            self.check()  # before the next chunk, whose status replaces this one's
            self.held = [n + len(p) for n, p in zip(self.held, parts)]

    def round(self, trees, uniform, temperature=0.0, top_k=0, top_p=1.0):
        """One verification round. trees[s]: (tokens, parents) with the pending token first, or None;
        uniform [seqs][positions]: the number that decides the token after each position.
        Returns per sequence the accepted drafts and the token drawn after them."""
        import torch
        self._fits(trees, uniform.shape[1])
        tokens, parents, cu, mask, depth, owner = self._nodes(trees)
        position = self.lens[owner] + depth
        logits, rows = self._forward(tokens, cu, mask, depth, position)
        n = tokens.numel()
        drawn = torch.empty(n, dtype=torch.int32, device="cuda")
        full = lambda v, t: torch.full((n,), v, dtype=t, device="cuda")  # noqa: E731
        # The same number at the same position, whichever node stands there: the stream that comes out
        # does not depend on the drafts.
        api.sample_rows(logits, uniform[owner, position.long()].contiguous(), drawn, temperature=full(temperature, torch.float32),
                        top_k=full(top_k, torch.int32), top_p=full(top_p, torch.float32))
        api.tree_accept(tokens, parents, drawn, cu, self.path, self.count, self.next)
        self._grow()
        self._commit(rows, cu, self.path)
        # The host drafter's read; no operator above needed one.
        count, path, nxt = self.count.tolist(), self.path.tolist(), self.next.tolist()
        self.check()
        self.held = [n + c for n, c in zip(self.held, count)]
        return [None if trees[s] is None else [trees[s][0][i] for i in path[s][1:count[s]]] + [nxt[s]]
                for s in range(self.seqs)]

    def fork(self, src, dst):
        import torch
        ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (src, dst)]
        api.pages_fork(self.pool, self.refs, self.table, self.lens, *ids, self.refs, self.table, self.lens, self.status)
        self.check()
        for a, b in zip(src, dst):
            self.held[b] = self.held[a]

    def finish(self, seqs):
        import torch
        api.pages_free(self.refs, self.table, self.lens, torch.tensor(seqs, dtype=torch.int32, device="cuda"), self.page,
                       self.refs, self.table, self.lens)
        for s in seqs:
            if 0 <= s < self.seqs:
                self.held[s] = 0

    def compact(self):
        import torch
        moves = torch.empty(1 + 2 * self.refs.numel(), dtype=torch.int32, device="cuda")
        api.pages_compact(self.pool, self.refs, self.table, self.refs, self.table, moves)
        return int(moves[0])

    def check(self):
        if int(self.status):
            raise RuntimeError(f"no pages: status {int(self.status)}")


def draft_tree(pending, guesses, rng, vocab, width=3):
    """A tree whose trunk follows `guesses`, with `width` - 1 random siblings at every level."""
    tokens, parents, trunk = [pending], [-1], 0
    for g in guesses:
        level = [g] + [rng.randrange(vocab) for _ in range(width - 1)]
        at = rng.randrange(width)
        level[0], level[at] = level[at], level[0]
        tokens += level
        parents += [trunk] * width
        trunk = len(tokens) - width + at
    return tokens, parents


def main(argv=None):
    import random

    import torch
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=0.0)
    args = ap.parse_args(argv)
    rng, model, n = random.Random(1), Model(), args.sequences
    uniform = torch.rand(n, 512, generator=torch.Generator().manual_seed(2)).cuda()
    prompt = [rng.randrange(model.vocab) for _ in range(21)]
    streams = []
    for drafts in (False, True):
        d = Decoder(model, n)
        d.prompt([prompt] + [None] * (n - 1))       # one prompt, ...
        d.fork([0] * (n - 1), list(range(1, n)))    # ... continued n times
        out, pending, rounds = [[] for _ in range(n)], [7 + s for s in range(n)], 0
        while min(map(len, out)) < args.tokens:
            # The guesses replay the first run's stream, one in four wrong: a drafter of that quality.
            guess = [[t if rng.random() < 0.75 else rng.randrange(model.vocab) for t in streams[0][s][len(out[s]):][:4]]
                     if drafts else [] for s in range(n)]
            got = d.round([draft_tree(pending[s], guess[s], rng, model.vocab) for s in range(n)], uniform, args.temperature)
            for s in range(n):
                out[s] += got[s]
                pending[s] = got[s][-1]
            rounds += 1
        d.finish(list(range(n)))
        print(f"{'trees of drafts' if drafts else 'one token a round'}: {sum(map(len, out))} tokens in {rounds} rounds, "
              f"pages left in use: {int((d.refs != 0).sum())}")
        streams.append(out)
    same = sum(a[:args.tokens] == b[:args.tokens] for a, b in zip(*streams))
    print(f"{same} of {n} streams are the same with and without drafts")


if __name__ == "__main__":
    main()
