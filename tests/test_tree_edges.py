"""Edges of the tree operators: how their blocks and streams wait for one another, settings at the ends of
their ranges, indices that belong to nobody, many sequences, large pools.

What cannot be shown without a race on the device is checked on the host: on the kernels' source, or
through bindings whose library and tensors are stand-ins.
"""
from __future__ import annotations

import re
from pathlib import Path

import pytest

from test_tree_round import check_row, sample

CSRC = Path(__file__).resolve().parent.parent / "turbo-winfare-dense_b200" / "csrc"


def code_of(name):
    """A kernel file without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


# ------------------------------------------------------------------------------------- sampling

def test_sampling_blocks_have_started_before_remote_access():
    """A cluster's blocks write into each other's shared memory: every block has to have started by then.
    The kernel says so at its entry, and waits for it ahead of the first exchange."""
    code = code_of("sample_rows.cu")
    assert re.search(r"void started\(\) const \{\s*if \(blocks > 1\) asm volatile\(\"barrier\.cluster\.arrive", code)
    assert re.search(r"void meet\(\) const \{\s*if \(blocks > 1\) asm volatile\(\"barrier\.cluster\.wait\.acquire", code)
    kernel = code[code.index("sample_rows_kernel(SampleRowsArgs a)"):]
    assert 0 < kernel.index("row.started();") < kernel.index("sample_row(a, sm, row")
    body = code[code.index("void sample_row(const SampleRowsArgs& a"):code.index("sample_rows_kernel(SampleRowsArgs a)")]
    first = min(body.index(x) for x in (".exchange(", ".merge(", ".gather(", "map_shared_rank"))
    assert body.index("row.meet();") < first and "return" not in body[:body.index("row.meet();")]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 4097), (1, 262144), (9, 262144), (70, 20001)])
def test_sampling_beside_other_work(built_lib, rows, vocab):
    """Clusters whose blocks are placed while another stream keeps the multiprocessors busy."""
    import torch
    from g4dense_b200 import api
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    u = torch.rand(rows, generator=g, device="cuda")
    cold, k = torch.zeros(rows, device="cuda"), torch.full((rows,), 20, dtype=torch.int32, device="cuda")
    token = torch.empty(2, rows, dtype=torch.int32, device="cuda")
    api.sample_rows(x, u, token[0], top_k=k)
    want, best = token[0].clone(), x.argmax(1).int()
    busy, a = torch.cuda.Stream(), torch.randn(1024, 1024, device="cuda")
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(busy):
            b = a * 1.5 + a
            b = b.relu().sum(0)
        api.sample_rows(x, u, token[0], top_k=k)
        api.sample_rows(x, u, token[1], temperature=cold)
        assert torch.equal(token[0], want) and torch.equal(token[1], best)


CUTS = [(0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.3), (700, 0.6, 0.0), (2000, 1.0, 0.0), (3, 0.9, 0.2)]


def logits_with_masks(rows, vocab, seed):
    """Rows of whole numbers (ties all over) whose entries are masked here and there, ends included."""
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, (rows, vocab), generator=g).float()
    x[torch.rand(rows, vocab, generator=g) < 0.2] = -float("inf")
    x[:, 0], x[:, -1], x[:, vocab // 2] = -float("inf"), -float("inf"), 3.0
    return x, torch.rand(rows, generator=g).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 1003, 40000, 262144])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_infinite_temperature(built_lib, vocab, dtype):
    """Every entry that is not masked weighs the same; a masked one, or the padding behind the row, nothing."""
    import torch
    x, u = logits_with_masks(len(CUTS), vocab, vocab)
    k, p, low = zip(*CUTS)
    token, prob, kept = sample(x.to(getattr(torch, dtype)).cuda(), u, temperature=[float("inf")] * len(u), top_k=k, top_p=p,
                               min_p=low)
    for r in range(len(CUTS)):  # 1e30 leaves weights of 1 - 1e-29
        check_row(x[r].double().numpy(), u[r], 1e30, k[r], p[r], low[r], token[r], prob[r], kept[r])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 1003, 40000])
@pytest.mark.parametrize("temperature", [1e-36, 1e-38, 1e-40, 1.5e-45])
def test_tiny_temperatures(built_lib, vocab, temperature):
    """All that is below the maximum weighs nothing, and the maxima that tie share the mass, whatever cuts."""
    x, u = logits_with_masks(len(CUTS), vocab, vocab + 1)
    k, p, low = zip(*CUTS)
    token, prob, kept = sample(x.cuda(), u, temperature=[temperature] * len(u), top_k=k, top_p=p, min_p=low)
    for r in range(len(CUTS)):  # 1e-3 leaves exp(-1000) of the next logit
        check_row(x[r].double().numpy(), u[r], 1e-3, k[r], p[r], low[r], token[r], prob[r], kept[r])


@pytest.mark.gpu
def test_settings_that_are_not_numbers(built_lib):
    """A NaN top_p or min_p is off, whichever way the row takes; a NaN temperature picks the maximum."""
    import torch
    nan = float("nan")
    g = torch.Generator().manual_seed(9)
    x = torch.randn(5, 5000, generator=g)
    k = [20, 300, 2000, 0, 20]
    t = [1.0, 1.0, 1.0, 1.0, nan]
    token, prob, kept = sample(x.cuda(), [0.4] * 5, temperature=t, top_k=k, top_p=[nan] * 5, min_p=[nan] * 5)
    for r in range(4):
        check_row(x[r].double().numpy(), 0.4, 1.0, k[r], 1.0, 0.0, token[r], prob[r], kept[r])
    assert (token[4], prob[4], kept[4]) == (int(x[4].argmax()), 1.0, 1)
