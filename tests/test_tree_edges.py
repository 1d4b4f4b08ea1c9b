"""Edges of the tree operators: how their blocks and streams wait for one another, settings at the ends of
their ranges, indices that belong to nobody, many sequences, large pools.

What cannot be shown without a race on the device is checked on the host: on the kernels' source, or
through bindings whose library and tensors are stand-ins.
"""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import numpy as np
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


# -------------------------------------------------------------------------------------- streams

class Stand:
    """What the bindings look at in a tensor, without a device."""

    def __init__(self, shape, dtype=None, device=0):
        import torch
        self.shape, self.dtype, self.device = tuple(shape), dtype or torch.int32, device
        self.is_cuda = True

    def numel(self):
        n = 1
        for k in self.shape:
            n *= k
        return n

    def stride(self):
        out, n = [], 1
        for k in reversed(self.shape):
            out.insert(0, n)
            n *= k
        return tuple(out)

    dim = lambda self: len(self.shape)  # noqa: E731
    is_contiguous = lambda self: True  # noqa: E731
    data_ptr = lambda self: 4096  # noqa: E731
    element_size = lambda self: self.dtype.itemsize  # noqa: E731
    get_device = lambda self: self.device  # noqa: E731


def operator_calls(api, device=None, **kw):
    """One call of every operator on stand-ins; `device` names the tensors that are elsewhere."""
    import torch
    bf, f32 = torch.bfloat16, torch.float32
    t = lambda *shape, dtype=None: Stand(shape, dtype)  # noqa: E731
    q, pool, new = t(6, 4, 64, dtype=bf), t(9, 16, 2, 64, dtype=bf), t(6, 2, 64, dtype=bf)
    planes, state = t(2, 9, 16, 2, 64, dtype=bf), (t(9), t(3, 4), t(3))
    n = Stand((3,), device=1) if device else t(3)
    return {
        "tree_attention": lambda: api.tree_attention(q, pool, pool, t(3, 4), n, new, new, t(4), t(6, 1), q, t(1 << 20, dtype=torch.uint8),
                                                     max_nodes=6, scale=1.0, **kw),
        "sample_rows": lambda: api.sample_rows(t(3, 50, dtype=f32), t(3, dtype=f32), n, **kw),
        "tree_accept": lambda: api.tree_accept(t(6), t(6), t(6), t(4), t(3, 6), n, t(3), **kw),
        "pages_reserve": lambda: api.pages_reserve(*state, n, 16, *state[:2], t(1), **kw),
        "pages_fork": lambda: api.pages_fork(planes, *state, n, t(3), *state, t(1), **kw),
        "pages_free": lambda: api.pages_free(*state, n, 16, *state, **kw),
        "pages_compact": lambda: api.pages_compact(planes, *state[:2], *state[:2], t(19) if not device else Stand((19,), device=1), **kw),
        "pages_copy": lambda: api.pages_copy(planes, planes, n, t(3), **kw),
        "pages_commit": lambda: api.pages_commit(planes, t(3, 4), t(3), t(2, 6, 2, 64, dtype=bf), t(4), t(3, 6), n, t(3), **kw),
    }


OPERATORS = ["tree_attention", "sample_rows", "tree_accept", "pages_reserve", "pages_fork", "pages_free", "pages_compact",
             "pages_copy", "pages_commit"]


class Calls:
    """A library that takes down the stream, the last argument, of every call."""

    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        def call(*args):
            self.streams.append(args[-1])
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    """The bindings over a stand-in library, current device 0 and current stream 1234."""
    import torch
    from g4dense_b200 import api
    calls = Calls()
    api._types()
    monkeypatch.setattr(api, "lib", lambda: calls)
    monkeypatch.setattr(api, "_here", lambda: 0)
    monkeypatch.setattr(api, "_stream_of", lambda dev: 1234)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": 1234}))
    return calls


@pytest.mark.parametrize("name", OPERATORS)
def test_calls_go_to_the_current_stream(calls, name):
    from g4dense_b200 import api
    operator_calls(api)[name]()
    assert calls.streams == [1234]
    operator_calls(api, stream=type("S", (), {"cuda_stream": 77}))[name]()
    assert calls.streams == [1234, 77]


@pytest.mark.parametrize("name", OPERATORS)
def test_tensors_of_another_device_are_refused(calls, name):
    """A kernel runs on the current device: an array of another one would be a bad address there."""
    from g4dense_b200 import api
    with pytest.raises(ValueError, match="current device"):
        operator_calls(api, device=1)[name]()
    assert calls.streams == []


def test_expanded_workspace_is_refused(calls):
    """A view with more elements than memory behind it."""
    import torch
    from g4dense_b200 import api

    class Wide(Stand):
        is_contiguous = lambda self: False  # noqa: E731
    q, pool, new = (Stand(n, torch.bfloat16) for n in ((6, 4, 64), (9, 16, 2, 64), (6, 2, 64)))
    with pytest.raises(ValueError, match="workspace"):
        api.tree_attention(q, pool, pool, Stand((3, 4)), Stand((3,)), new, new, Stand((4,)), Stand((6, 1)), q,
                           Wide((1 << 20,), torch.uint8), max_nodes=6, scale=1.0)
    assert calls.streams == []


def test_decoder_products_go_to_the_current_stream(calls):
    import torch
    from g4dense_b200 import tree_decode as T
    got = []

    class Matrix:
        N = 5

        def gemm(self, x, out, stream=None):
            got.append((x.shape[0], stream.cuda_stream))
    T._product(Matrix(), torch.zeros(130, 8))
    assert got == [(128, 1234), (2, 1234)]


@pytest.mark.gpu
def test_calls_wait_for_the_current_stream(built_lib):
    """Inputs that a side stream is still to make, outputs that it reads next, no stream given."""
    import torch
    from g4dense_b200 import api
    from test_tree_attention import make, run
    c = make([300, 40], [5, 3], 4, 2, 64, 16, "bf16", seed=1)
    want = run(c)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, u = torch.randn(40, 3000, generator=g, device="cuda"), torch.rand(40, generator=g, device="cuda")
    token = torch.empty(40, dtype=torch.int32, device="cuda")
    api.sample_rows(x, u, token)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.randn(3, 6, 8, 16, generator=g, device="cuda")
    there, src, dst = torch.zeros_like(pool), dev([0, 5, 2]), dev([4, 1, 3])
    late, side = [torch.zeros_like(t) for t in (c["q"], x, pool)], torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        for a, b in zip(late, (c["q"], x, pool)):
            a.copy_(b)
        out = run(dict(c, q=late[0])).clone()
        drawn = torch.empty_like(token)
        api.sample_rows(late[1], u, drawn)
        drawn = drawn.clone()
        api.pages_copy(late[2], there, src, dst)
        moved = there.clone()
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(drawn, token)
    assert all(torch.equal(moved[:, d], pool[:, s]) for s, d in ((0, 4), (5, 1), (2, 3)))


@pytest.mark.gpu
def test_decoder_on_a_side_stream(built_lib):
    import torch
    from g4dense_b200 import tree_decode as T

    def go():
        d = T.Decoder(T.Model(3), 2)
        d.prompt([[5] * 40, [9, 8, 7]])
        uniform = torch.rand(2, 300, generator=torch.Generator().manual_seed(5)).cuda()
        got = [d.round([([1, 2, 3], [-1, 0, 0]), ([4], [-1])], uniform) for _ in range(3)]
        return got, d.pool.clone()
    want, pool = go()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got, other = go()
        side.synchronize()
    assert got == want and torch.equal(pool, other)


# -------------------------------------------------------------------------------------- devices

def test_once_per_device(tmp_path):
    """csrc/per_device.h on the host, with a stand-in for the runtime's current device."""
    out = tmp_path / "test_per_device"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", str(CSRC), "-I", "/usr/local/cuda/include",
                        str(Path(__file__).resolve().parent / "cpp" / "test_per_device.cpp"), "-o", str(out)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("name", ["tree_attn.cu", "sample_rows.cu"])
def test_attributes_are_set_on_every_device(name):
    """cudaFuncSetAttribute holds for the current device: no flag of the whole process may stand for it."""
    code = code_of(name)
    assert "static bool" not in code and "static int n" not in code
    assert code.count("cudaFuncSetAttribute") and "static OncePerDevice" in code


@pytest.mark.gpu
def test_two_devices_in_one_process(built_lib):
    import torch
    from test_tree_attention import check, make
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    for d in (0, 1):
        with torch.cuda.device(d):
            check(make([900, 40], [5, 3], 8, 2, 128, 16, "bf16", seed=1))
            x = torch.randn(2, 262144, device="cuda")
            token, _, _ = sample(x, [0.5, 0.5], temperature=[0.0, 0.0])
            assert token == x.argmax(1).tolist()


# ----------------------------------------------------------------------------------- attention

@pytest.mark.gpu
def test_check_error_waits_for_every_stream(built_lib):
    """The launch that is reported on may run on a stream that the default one does not wait for."""
    import torch
    from g4dense_b200 import api
    from test_tree_attention import make, run
    c = make([300, 40], [5, 3], 4, 2, 64, 16, "bf16", seed=1)
    run(c)
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        run(c)
        done.record()
    api.tree_attention_check_error()
    assert done.query()


# ------------------------------------------------------------------------------------- decoder

@pytest.mark.gpu
def test_prompt_chunks_that_do_not_fit(built_lib):
    """A first chunk without pages must not be forgotten when a later, smaller one finds some."""
    import torch
    from g4dense_b200 import tree_decode as T
    d = T.Decoder(T.Model(), 2, pages=1)
    before = [t.clone() for t in (d.refs, d.table, d.lens, d.pool)]
    with pytest.raises(RuntimeError, match="status 1"):
        d.prompt([[5] * (d.max_nodes + 5), None])
    assert all(torch.equal(a, b) for a, b in zip(before, (d.refs, d.table, d.lens, d.pool)))


@pytest.mark.parametrize("tree,match", [(([1, 2], [-1, 0]), "position 30"), (([-1], [-1]), "vocabulary"),
                                        (([4096], [-1]), "vocabulary"), (([1] * 33, [-1] + [0] * 32), "at most 32"),
                                        (([1, 2], [-1]), "1 parents")])
def test_decoder_refuses_what_it_cannot_index(tree, match):
    """A position without a uniform number, a token outside the vocabulary and a tree too large would be
    indexes out of range on the device; they are refused before anything is queued."""
    import torch
    from g4dense_b200 import tree_decode as T
    d = object.__new__(T.Decoder)
    d.m, d.seqs, d.max_nodes, d.held = T.Model, 2, 32, [0, 29]
    with pytest.raises(ValueError, match=match):
        d.round([None, tree], torch.zeros(2, 30))


@pytest.mark.gpu
def test_decoder_knows_its_lengths(built_lib):
    import torch
    from g4dense_b200 import tree_decode as T
    d = T.Decoder(T.Model(), 3)
    uniform = torch.rand(3, 60, generator=torch.Generator().manual_seed(5)).cuda()
    d.prompt([[5] * 40, None, [1, 2]])
    d.round([([1, 2, 3], [-1, 0, 0]), None, ([7], [-1])], uniform)
    d.fork([0], [1])
    assert d.held == d.lens.tolist() and d.held[0] > 40 and d.held[2] == 3
    d.finish([0])
    assert d.held == d.lens.tolist() and d.held[0] == 0


# ----------------------------------------------------------------------------------------- pages

@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_commit_stops_at_the_first_row_without_a_place(built_lib, in_place):
    """A path entry that is not one of the sequence's nodes, a count above them, a position past the table
    or without a page: the rows ahead of it are committed, and the length grows by those alone."""
    import torch
    from g4dense_b200 import api
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    planes, page, sizes = 3, 4, [3, 2, 0, 40, 5, 1, 4]
    lens = [2, 7, 0, 1, 5, 3, -4]
    table = [[0, 1, 2] + [-1] * 9, [3, 4, -1] + [-1] * 9, [5] + [-1] * 11, list(range(6, 18)), [18, 19, 99] + [-1] * 9,
             [20, -1, -1] + [-1] * 9, [21] * 12]
    cu = np.concatenate([[0], np.cumsum(sizes)])
    width = 41
    for kind in ("path", "first"):
        path = [[0, 3, 1], [0, 1, 2, -1], [0], list(range(40)) + [40], [0, 2, 4, 1, 3], [0, 0, 0], [0, 1]]
        count = [3, 2, 1, 41, 5, 3, 2]
        if kind == "first":
            path, count = [list(range(60)) for _ in sizes], [3, 5, 1, 2 ** 31 - 1, 3, -2, 4]
        g = torch.Generator(device="cuda").manual_seed(1)
        pool = torch.randn(planes, 22, page, 8, generator=g, device="cuda")
        rows = torch.randn(planes, int(cu[-1]), 8, generator=g, device="cuda")
        want, grown = pool.clone(), list(lens)
        for s, n in enumerate(lens):
            for i in range(min(max(count[s], 0), len(path[s]))):
                col = (n + i) // page
                if n < 0 or not 0 <= path[s][i] < sizes[s] or col >= 12 or not 0 <= table[s][col] < 22:
                    break
                want[:, table[s][col], (n + i) % page] = rows[:, cu[s] + path[s][i]]
                grown[s] += 1
        old = dev(lens)
        new = old if in_place else torch.full_like(old, 9)
        api.pages_commit(pool, dev(table), old, rows, dev(cu.tolist()),
                         dev([(p + [-1] * width)[:width] for p in path]) if kind == "path" else None, dev(count), new)
        assert new.tolist() == grown and torch.equal(pool, want), kind


def test_fork_checks_do_not_depend_on_timing():
    """Whether a warp looks at its sources' pages may not depend on what other warps have found by then: the
    word they raise is read between two barriers of the block, once, for all of them."""
    code = code_of("pages.cu")
    body = code[code.index("fork_kernel(PageTables t"):code.index("compact_kernel(PageTables t")]
    reads = [m.start() for m in re.finditer(r"code == kPagesOk", body)]
    marks = [m.start() for m in re.finditer(r"__syncthreads\(\)", body)]
    raises = [m.start() for m in re.finditer(r"atomicMax\(&code", body)]
    between = lambda a, b: any(a < m < b for m in marks)  # noqa: E731
    assert len(reads) >= 2
    for r in reads:
        assert all(between(w, r) if w < r else between(r, w) for w in raises)


@pytest.mark.gpu
def test_fork_with_several_faults(built_lib):
    """The largest code of all faults, whichever warp meets which first."""
    import torch
    from g4dense_b200 import api
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    seqs, width, n = 400, 64, 200
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    table[:n] = torch.arange(n * width).reshape(n, width)
    lens = dev([4 * width] * n + [0] * (seqs - n))
    refs, status = torch.ones(n * width + 8, dtype=torch.int32, device="cuda"), dev([9])
    pool = torch.zeros(1, n * width + 8, 4, 4, device="cuda")
    for bad_page, bad_seq in ((0, 150), (150, 0), (37, 38), (199, 1)):
        t = table.clone()
        t[bad_page, width - 1] = 10 ** 6  # found in the last round of its warp
        t[n + bad_seq, 0] = 3             # a destination that holds a page
        t = t.cuda()
        for _ in range(20):
            outs = [torch.full_like(x, 5) for x in (refs, t, lens)]
            api.pages_fork(pool, refs, t, lens, dev(list(range(n))), dev(list(range(n, 2 * n))), *outs, status)
            assert status.item() == 4
            assert all(torch.equal(a, b) for a, b in zip(outs, (refs, t, lens)))


def test_tables_beyond_whole_number_counts_are_refused(built_lib):
    """Page counts of a call are summed in 32 bits: a table of 2^31 cells or more could wrap them, and a
    reserve would report success without a page. Refused on the host."""
    from g4dense_b200 import api
    pack = lambda seqs, width: api._PAGE_TABLES.pack(*[4096] * 6, 1 << 20, seqs, width, 1)  # noqa: E731
    L = api.lib()
    for seqs, width in ((4096, 1 << 19), (2, 1 << 30)):
        assert L.g4b_pages_reserve(pack(seqs, width), 4096, 4096, None) == 1
        assert b"2^31 cells" in L.g4b_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ahead", [5.4, 18.0, 21.0])
@pytest.mark.parametrize("place", [0, 200])
def test_many_small_probabilities(built_lib, dtype, ahead, place):
    """One key, with no value, `ahead` nats above 299 others: the others' small probabilities make up the
    output. A probability is held to u of itself or, where fp16 is subnormal (below 2^-21 of the row's
    reference, its numbers being held 2^7 times), to 2^-32; the output to u, or to 2^-25 where it is
    subnormal. Scores are at most 21: fp32 adds 2 units in the last place of 32 and a few of the sums."""
    import torch
    from test_tree_attention import UNIT, make, run
    c = make([300], [2], 1, 1, 64, 16, dtype, seed=1)
    c["q"][:] = 1.0
    c["k_pool"][:], c["v_pool"][:], c["k_new"][:], c["v_new"][:] = 0, 1000.0, 0, 0
    p = c["table"][0, place // 16].long()
    c["k_pool"][p, place % 16], c["v_pool"][p, place % 16] = ahead / 8, 0
    score = float(c["k_pool"][p, place % 16, 0, 0]) * 8
    seen = 300 + (c["depth"].double() + 1)  # keys a node sees, itself and its parent among them
    small = np.exp(-score)
    want = (299 * 1000.0 * small) / (1 + (seen - 1) * small)
    u, err = UNIT[dtype], (run(c).double() - want[:, None, None]).abs()
    tol = want * (2.1 * u + 2.0 ** -18) + (299 * 1000 * 2.0 ** -32 + 2.0 ** -25 if dtype == "fp16" else 0)
    assert (err <= tol[:, None, None]).all(), (err.max().item(), tol.min().item(), want.tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [33, 64, 65, 100, 333])
@pytest.mark.parametrize("longest", [40, 900])
@pytest.mark.parametrize("window", [0, 30])
def test_many_sequences(built_lib, seqs, longest, window):
    """More sequences than a warp has lanes, and than the scheduling warp adds up by itself; whole runs of
    them without nodes, at both ends too; items that stay whole (tables of up to 4 tiles) and that are cut."""
    import random
    from test_tree_attention import check, make
    rng = random.Random(seqs + longest)
    lens = [rng.choice([0, 1, rng.randrange(longest), longest]) for _ in range(seqs)]
    nodes = [rng.choice([0, 1, 2, 4]) for _ in range(seqs)]
    for a, b in ((0, 3), (seqs // 2, seqs // 2 + 18), (seqs - 2, seqs)):
        nodes[a:min(b, seqs)] = [0] * (min(b, seqs) - a)
    lens[4] = longest
    check(make(lens, nodes, 4, 2, 64, 16, "bf16", seed=seqs), window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_hidden_values_in_items_that_are_cut(built_lib, dtype, dim, poison):
    """Infinities and NaN in values that some nodes see and others do not, in the first and last tiles of an
    item that several blocks work on."""
    import torch
    from test_tree_attention import formula, make, run
    chain = [-1, 0, 1, 2, 3, 4, 5, 6]
    c = make([3000, 2100], [8, 5], 4, 2, dim, 16, dtype, seed=dim, parents=[chain, chain])
    want = run(c, 1000)
    key = 3000 + 3 - 1000  # seen by depths 0..2 of the first sequence
    c["v_pool"][c["table"][0, key // 16].long(), key % 16, :, 5] = poison
    c["v_new"][6, 0, 9] = poison  # by nodes 6 and 7, in the heads of K/V head 0
    got, (o, _, _) = run(c, 1000), formula(c, 1000)
    strange = torch.zeros_like(got, dtype=torch.bool)
    strange[:3, :, 5] = True
    strange[6:8, :2, 9] = True
    assert torch.equal(~torch.isfinite(got), strange) and torch.equal(~torch.isfinite(o), strange)
    assert torch.equal(got[~strange], want[~strange])
    assert torch.equal(torch.nan_to_num(got[strange].double(), nan=3.0), torch.nan_to_num(o[strange].to(got.dtype).double(), nan=3.0))


@pytest.mark.gpu
def test_bad_pages_and_lengths_give_the_formula_without_them(built_lib):
    """A page id out of range reads as zeros, a length past the table is the table's."""
    import torch
    from test_tree_attention import UNIT, formula, make, run
    c = make([50, 10, 30], [3, 2, 1], 4, 2, 64, 16, "bf16", seed=2)
    c["table"][0, 1], c["table"][1, 0], c["lens"][0], c["lens"][2] = 10 ** 6, -5, 10 ** 9, -7
    got = run(c)
    zero = c["k_pool"].shape[0]
    d = dict(c, k_pool=torch.cat([c["k_pool"], torch.zeros_like(c["k_pool"][:1])]),
             v_pool=torch.cat([c["v_pool"], torch.zeros_like(c["v_pool"][:1])]), table=c["table"].clone(), lens=c["lens"].clone())
    d["table"][0, 1], d["table"][1, 0], d["lens"][0], d["lens"][2] = zero, zero, 16 * c["table"].shape[1], 0
    o, a, _ = formula(d)
    assert ((got.double() - o).abs() <= UNIT["bf16"] * (o.abs() + a) * 1.05 + 4e-5 * a).all()


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_large_pools(built_lib, in_place):
    """Reserve, fork, free and compaction in a pool of 70000 pages, nearly full, its free pages far in."""
    import torch
    from g4dense_b200 import api
    from test_tree_round import Plain
    rng = np.random.default_rng(3)
    pages, seqs, width = 70001, 90, 1500
    plain = Plain(rng.integers(0, 2 ** 15, (1, pages, 2, 8)).astype(np.int16), seqs, width)
    dev = lambda x: torch.from_numpy(np.array(x, dtype=np.int32)).cuda()  # noqa: E731
    pool = torch.from_numpy(plain.pool.copy()).cuda()
    state, status = [dev(plain.refs), dev(plain.table), dev(plain.lens)], dev([9])

    def step(what, call, expect):
        new = state if in_place else [torch.full_like(t, 77) for t in state]
        call(new)
        code = expect()
        assert code is None or status.item() == code, what
        state[:] = new
        for name, a, b in zip(("refs", "table", "lens"), state, (plain.refs, plain.table, plain.lens)):
            assert np.array_equal(a.cpu().numpy(), b), (what, name)
        assert np.array_equal(pool.cpu().numpy(), plain.pool), what

    def reserve(grow):
        def call(new):
            api.pages_reserve(*state, dev(grow), 2, new[0], new[1], status)
            if not in_place:
                new[2] = state[2]
            ok = 1 - status.clamp(max=1)
            new[2] = new[2] + dev(grow) * ok

        def expect():
            code = plain.reserve(grow.tolist())
            if code == 0:
                plain.lens += grow.astype(np.int32)
            return code
        step("reserve", call, expect)

    reserve(np.array([1801] * 76 + [0] * 14))           # 68476 pages
    reserve(np.array([1000] + [0] * 89))                 # the rest is far in
    reserve(np.array([0] * 76 + [400] * 14))             # too many
    src, dst = list(range(0, 20)), list(range(76, 90))
    step("fork", lambda new: api.pages_fork(pool, *state, dev(src[:14]), dev(dst), *new, status),
         lambda: plain.fork(src[:14], dst))
    gone = [0, 3, 4, 5, 40, 41, 76, 80]
    step("free", lambda new: api.pages_free(*state, dev(gone), 2, *new), lambda: plain.free(gone))
    moves = dev([0] * (1 + 2 * pages))

    def compact(new):
        api.pages_compact(pool, state[0], state[1], new[0], new[1], moves)
        new[2] = state[2]
    step("compact", compact, lambda: (plain.compact(), None)[1])
    assert moves[0].item() > 1000
    reserve(np.array([0] * 76 + [3] + [0] * 13))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(built_lib):
    """Pages and logits rows that lie gigabytes apart: element and byte offsets above 2^32."""
    import torch
    from g4dense_b200 import api
    from test_tree_attention import make, run
    c = make([300, 40], [5, 3], 4, 2, 64, 16, "bf16", seed=1)
    c["v_new"][3, 1, 7] = float("inf")  # values looked up one by one too
    want = run(c)
    pages, apart = c["k_pool"].shape[0], 1 << 28
    far = torch.empty(pages * apart, dtype=torch.bfloat16, device="cuda").view(pages, apart)
    assert (pages - 1) * apart > 1 << 32
    wide = [far[:, i * 4096:i * 4096 + 2048].view(pages, 16, 2, 64) for i in range(3)]
    wide[0].copy_(c["k_pool"])
    wide[1].copy_(c["v_pool"])
    got = run(dict(c, k_pool=wide[0], v_pool=wide[1]))
    assert torch.equal(torch.nan_to_num(got.double(), nan=1e9), torch.nan_to_num(want.double(), nan=1e9))
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    api.pages_copy(wide[0][None], wide[2][None], dev([0, pages - 1]), dev([pages - 1, 0]))
    assert torch.equal(wide[2][pages - 1], c["k_pool"][0]) and torch.equal(wide[2][0], c["k_pool"][pages - 1])
    rows, lens = torch.randn(1, 3, 2, 64, device="cuda").bfloat16(), dev([20])
    api.pages_commit(wide[2][None], dev([[0, pages - 2]]), lens, rows, dev([0, 3]), None, dev([3]), lens)
    assert torch.equal(wide[2][pages - 2, 4:7], rows[0]) and lens.item() == 23
    x = far[:, 8192:8192 + 5000]
    x.copy_(torch.randn(pages, 5000, generator=torch.Generator().manual_seed(3)))
    token, _, _ = sample(x, [0.5] * pages, temperature=[0.0] * pages)
    best = x.float().max(1, keepdim=True).values
    assert token == [int((r == b).nonzero()[0]) for r, b in zip(x.float(), best)]


def test_refusal_of_too_many_tiles_says_why(built_lib):
    """Tiles are counted in 32 bits over all sequences and heads; a call beyond that names the sizes."""
    from g4dense_b200 import api
    L = api.lib()
    args = api._TREE_ATTENTION.pack(*[4096] * 12, 1 << 40, 1024, 1024, 1024, 1 << 18, 1 << 20, 1 << 20, 1, 1000, 16,
                                    1 << 26, 1, 16, 16, 64, 0, 0, 1.0)
    assert L.g4b_tree_attention(args, None) != 0
    assert b"32 bits" in L.g4b_last_error() and b"n_seqs" in L.g4b_last_error()


def test_head_counts_beyond_32_bits_are_refused(built_lib):
    """A row's offset of heads * head_dim elements, and a group of max_nodes * heads rows, are 32-bit numbers."""
    from g4dense_b200 import api
    L = api.lib()
    assert L.g4b_tree_attention_workspace(256, 1 << 14, 1 << 14, 512) > 0
    assert L.g4b_tree_attention_workspace(1, 1 << 22, 1, 512) == 0
    assert L.g4b_tree_attention_workspace(256, 1 << 23, 1, 64) == 0
