"""Edges of the tree operators: how their blocks and streams wait for one another, settings at the ends of
their ranges, indices that belong to nobody, many sequences, large pools.

What cannot be shown without a race on the device is checked on the host: on the kernels' source, or
through bindings whose library and tensors are stand-ins.
"""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest

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
