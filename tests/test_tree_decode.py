"""The batched tree decoder (g4dense_b200/tree_decode.py) that runs the tree operators together.

With the same uniform number at the same position, the stream must not depend on the drafts. Logits do
depend on the batch a little: attention outputs are rounded to bf16 (2^-8) after sums whose grouping
differs, and the verify GEMM's modes differ in the last bits. So streams are compared up to the first
token whose greedy margin is below that noise: 2^-8 of the logits' range, times four layers' roundings.
"""
from __future__ import annotations

import random

import pytest

pytestmark = pytest.mark.gpu


def margins(decoder, prompt, stream, pending):
    """Greedy margins and logit ranges along a stream, one token a round on a fresh decoder."""
    import torch
    decoder.prompt([prompt] + [None] * (decoder.seqs - 1))
    out = []
    for t in [pending] + stream[:-1]:
        tokens, _, cu, mask, depth, owner = decoder._nodes([([t], [-1])] + [None] * (decoder.seqs - 1))
        logits, rows = decoder._forward(tokens, cu, mask, depth, decoder.lens[owner] + depth)
        top = torch.topk(logits[0], 2).values
        out.append(float(top[0] - top[1]) / float(logits[0].abs().max()))
        decoder.count.copy_(torch.tensor([1] + [0] * (decoder.seqs - 1), dtype=torch.int32))
        decoder._grow()
        decoder._commit(rows, cu, None)
    return out


def test_streams_do_not_depend_on_drafts(built_lib):
    import torch
    from g4dense_b200 import tree_decode as T
    rng, model, n, length = random.Random(3), T.Model(), 3, 40
    uniform = torch.rand(n, 256, generator=torch.Generator().manual_seed(4)).cuda()
    prompt = [rng.randrange(model.vocab) for _ in range(37)]  # more than max_nodes: two chunks
    streams = []
    for drafts in (0, 1, 2):
        d = T.Decoder(model, n, pages=40)
        d.prompt([prompt, None, None])
        used = int((d.refs != 0).sum())
        d.fork([0, 0], [1, 2])
        assert int((d.refs != 0).sum()) == used + 2 and int(d.refs.max()) == 3  # full pages shared, the last copied
        out, pending, rounds = [[] for _ in range(n)], [11, 12, 13], 0
        while min(map(len, out)) < length:
            guess = [streams[0][s][len(out[s]):][:4] if drafts else [] for s in range(n)]
            if drafts == 2:
                guess = [[t if rng.random() < 0.6 else rng.randrange(model.vocab) for t in x] for x in guess]
            got = d.round([T.draft_tree(pending[s], guess[s], rng, model.vocab) for s in range(n)], uniform)
            for s in range(n):
                out[s] += got[s]
                pending[s] = got[s][-1]
            rounds += 1
            if rounds == 5:  # moving pages does not change what comes out
                d.finish([2])
                d.compact()
                d.fork([1], [2])
                out[2], pending[2] = list(out[1]), pending[1]
                live = (d.refs != 0).nonzero()
                assert int(live.max()) < 40
                uniform[2] = uniform[1]
        if drafts == 1:
            assert rounds < length / 2
        d.finish([0, 1, 2])
        assert int(d.refs.abs().sum()) == 0 and int(d.lens.sum()) == 0 and int(d.table.max()) == -1
        streams.append(out)
    margin = margins(T.Decoder(model, n, pages=40), prompt, streams[0][0][:length], 11)
    sure = next((i for i, m in enumerate(margin) if m < 4 * 2.0 ** -8), length)
    assert sure > 5
    for other in streams[1:]:
        assert other[0][:sure] == streams[0][0][:sure]


def test_sampled_rounds_and_exhausted_pool(built_lib):
    import torch
    from g4dense_b200 import tree_decode as T
    model = T.Model()
    d = T.Decoder(model, 2, pages=3)
    d.prompt([[5] * 30, None])
    uniform = torch.rand(2, 256, generator=torch.Generator().manual_seed(5)).cuda()
    got = d.round([([1, 2, 3], [-1, 0, 0]), None], uniform, temperature=0.9, top_k=50, top_p=0.95)
    assert got[1] is None and 1 <= len(got[0]) <= 2 and int(d.lens[0]) == 30 + len(got[0])
    before = [t.clone() for t in (d.refs, d.table, d.lens, d.pool)]
    with pytest.raises(RuntimeError, match="status 1"):
        d.prompt([[9] * 30, None])
    assert all(torch.equal(a, b) for a, b in zip(before, (d.refs, d.table, d.lens, d.pool)))


def test_command(built_lib, capsys):
    from g4dense_b200 import tree_decode as T
    T.main(["--sequences", "2", "--tokens", "12", "--temperature", "0.8"])
    out = capsys.readouterr().out
    assert "pages left in use: 0" in out and "trees of drafts" in out
