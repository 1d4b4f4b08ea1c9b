"""Tree attention over a paged K/V cache (g4b_tree_attention) against the formula in 64 bits.

Tolerance: with u the unit roundoff of the type (bf16 2^-8, fp16 2^-11), a probability is rounded
once (u) and the output once (u), so |error| <= u (|o| + A) with A = sum_j p_j |v_j|, up to second
order (5 %). fp32 scores and exponentials add at most 4e-5 of A (|scale q.k| <= 100 here, times
2^-22, and a few units in the last place of the exponential and of the sums). fp16 also has an
absolute error: probabilities below 2^-14 of the row's reference are subnormal (2^-25 each, the
reference at most e^8 below the maximum is on the safe side), and outputs likewise.
"""
from __future__ import annotations

import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def make(seqs, nodes, heads, kv_heads, dim, page, dtype, seed=0, width=None, spare=2, parents=None, std=1.0):
    """seqs: cached lengths; nodes: tree sizes."""
    import torch
    from g4dense_b200 import api
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    need = [-(-n // page) for n in seqs]
    width = width or max(1, max(need))
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    table = np.full((len(seqs), width), -1, np.int32)
    for s, n in enumerate(need):
        table[s, :n] = [ids.pop() for _ in range(n)]
    words = max(1, -(-max(nodes) // 32))
    masks, depths, ups = [], [], []
    for s, n in enumerate(nodes):
        up = parents[s] if parents else [-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)]
        m, d = api.tree_mask(up[:n], words)
        masks.append(m)
        depths.append(d)
        ups.append(up)
    total = sum(nodes)

    def normal(*shape, k=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * k).to(kind)

    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return dict(q=normal(total, heads, dim, k=std), k_pool=normal(sum(need) + spare, page, kv_heads, dim),
                v_pool=normal(sum(need) + spare, page, kv_heads, dim), k_new=normal(total, kv_heads, dim),
                v_new=normal(total, kv_heads, dim), table=t(table), lens=t(np.array(seqs, np.int32)),
                cu=t(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)),
                mask=t(np.concatenate(masks) if total else np.zeros((0, words), np.int32)),
                depth=t(np.concatenate(depths) if total else np.zeros(0, np.int32)), max_nodes=max(max(nodes), 1),
                scale=dim ** -0.5, dtype=dtype)


def run(c, window=0, out=None, stream=None):
    import torch
    from g4dense_b200 import api
    heads, dim = c["q"].shape[1:]
    out = torch.full_like(c["q"], 7.0) if out is None else out
    ws = torch.empty(api.tree_attention_workspace(c["max_nodes"], heads, c["k_new"].shape[1], dim), dtype=torch.uint8,
                     device="cuda")
    api.tree_attention(c["q"], c["k_pool"], c["v_pool"], c["table"], c["lens"], c["k_new"], c["v_new"], c["cu"],
                       c["mask"], out, ws, max_nodes=c["max_nodes"], scale=c["scale"], depth=c["depth"], window=window,
                       stream=stream)
    return out


def formula(c, window=0):
    """(o, A, sum of |v| a row sees) in float64, node by node over exactly the keys it sees."""
    import torch
    cu, lens, table = c["cu"].tolist(), c["lens"].tolist(), c["table"].cpu().numpy()
    mask, depth = c["mask"].cpu().numpy().view(np.uint32), c["depth"].tolist()
    page, kv = c["k_pool"].shape[1], c["k_pool"].shape[2]
    heads, dim = c["q"].shape[1:]
    o = torch.zeros(c["q"].shape, dtype=torch.float64, device="cuda")
    a, b = torch.zeros_like(o), torch.zeros_like(o)
    for s, n in enumerate(lens):
        ids = torch.from_numpy(table[s, :-(-n // page)].astype(np.int64)).cuda()
        k = c["k_pool"][ids].reshape(-1, kv, dim)[:n].double()
        v = c["v_pool"][ids].reshape(-1, kv, dim)[:n].double()
        for t in range(cu[s], cu[s + 1]):
            first = max(0, n + depth[t] - window + 1) if window else 0
            seen = [j for j in range(cu[s + 1] - cu[s]) if (mask[t, j // 32] >> (j % 32)) & 1]
            seen = [cu[s] + j for j in seen if not window or depth[t] - depth[cu[s] + j] < window]
            kk = torch.cat([k[first:], c["k_new"][seen].double()])
            vv = torch.cat([v[first:], c["v_new"][seen].double()])
            if kk.shape[0] == 0:
                continue
            q = c["q"][t].double().reshape(kv, heads // kv, dim)
            p = torch.softmax(torch.einsum("hgd,lhd->hgl", q, kk) * c["scale"], -1)
            o[t] = torch.einsum("hgl,lhd->hgd", p, vv).reshape(heads, dim)
            a[t] = torch.einsum("hgl,lhd->hgd", p, vv.abs()).reshape(heads, dim)
            b[t] = vv.abs().sum(0)[:, None].expand(kv, heads // kv, dim).reshape(heads, dim)
    return o, a, b


def check(c, window=0, **kw):
    import torch
    got = run(c, window, **kw)
    torch.cuda.synchronize()
    o, a, b = formula(c, window)
    u = UNIT[c["dtype"]]
    tol = u * (o.abs() + a) * 1.05 + 4e-5 * a
    if c["dtype"] == "fp16":
        tol = tol + 2.0 ** -24 * b + 2.0 ** -24
    bad = ~((got.double() - o).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got.double() - o).abs() / tol).max():.2f} of the tolerance"
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (6, 1)])
def test_matches_formula(built_lib, dtype, dim, heads, kv_heads):
    check(make([0, 1, 15, 16, 17, 130, 400, 127, 128, 129], [1, 5, 3, 1, 9, 4, 12, 2, 1, 7], heads, kv_heads, dim, 16,
               dtype, seed=dim + heads))


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 136, 256])
def test_page_sizes(built_lib, page):
    """Pages that do and do not divide a 128-key tile, and sequences that end anywhere in one."""
    check(make([page - 1, page, page + 1, 3 * page + 5, 1000, 0], [3, 1, 2, 6, 2, 4], 4, 2, 128, page, "bf16", seed=page))


@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 256])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 4, 2), (64, 9, 1)])
def test_tree_sizes(built_lib, nodes, dim, heads, kv_heads):
    check(make([70, 0, 300], [nodes, max(1, nodes // 3), nodes], heads, kv_heads, dim, 16, "bf16", seed=nodes))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 16, 256), (32, 4, 512), (16, 1, 128), (64, 1, 64), (12, 4, 128),
                                                (5, 5, 512), (40, 1, 512), (256, 1, 64)])
def test_head_layouts(built_lib, heads, kv_heads, dim):
    check(make([333, 5, 90], [17, 3, 8], heads, kv_heads, dim, 32, "bf16", seed=heads * dim))


@pytest.mark.parametrize("window", [1, 2, 7, 48, 128, 129, 300, 5000])
@pytest.mark.parametrize("dim", [64, 256, 512])
def test_windows(built_lib, window, dim):
    check(make([0, 1, 47, 48, 49, 200, 450, 129], [6, 1, 12, 3, 1, 20, 33, 2], 4, 2, dim, 24, "bf16", seed=window), window)


def test_window_never_reads_released_pages(built_lib):
    """Table entries of pages that lie wholly before every node's window may be empty."""
    import torch
    c = make([500, 321, 64], [9, 2, 5], 4, 2, 128, 16, "bf16", seed=3)
    want = run(c, 100)
    t = c["table"].clone()
    for s, n in enumerate([500, 321, 64]):
        t[s, :max(0, n - 100 + 1) // 16] = -1
    gone = torch.ones(c["k_pool"].shape[0], dtype=torch.bool, device="cuda")
    gone[t[t >= 0].long()] = False
    c["k_pool"][gone] = float("nan")
    c["v_pool"][gone] = float("nan")
    c["table"] = t
    assert torch.equal(run(c, 100), want)


@pytest.mark.parametrize("dim,heads,kv_heads,nodes", [(128, 8, 8, 1), (256, 32, 16, 5), (512, 32, 4, 9), (64, 4, 4, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_long_contexts(built_lib, dim, heads, kv_heads, nodes, dtype):
    """Tens of tiles per sequence, ragged: splits over the long axis and their sum."""
    check(make([9000, 37, 5001, 0], [nodes, nodes, 1, nodes], heads, kv_heads, dim, 64, dtype, seed=dim, std=2.0))


def test_peaked_and_rising_scores(built_lib):
    """Row maxima that rise steadily along the keys, by hundreds in all: every rescale path; and one
    key that outweighs all others."""
    import torch
    c = make([1500, 800], [7, 3], 4, 2, 128, 16, "bf16", seed=11)
    c["q"][:] = 1.0
    for s, n in enumerate([1500, 800]):
        ids = c["table"][s, :-(-n // 16)].long()
        ramp = torch.linspace(-2.5, 2.5, ids.numel() * 16, device="cuda").reshape(-1, 16, 1, 1)
        c["k_pool"][ids] = (ramp if s == 0 else -ramp).to(torch.bfloat16).expand(-1, -1, 2, 128)
    check(c)
    c = make([600], [4], 4, 4, 64, 16, "fp16", seed=12)
    c["q"][:] = 2.0
    c["k_pool"][c["table"][0, 20].long(), 5] = 6.0
    check(c)


def test_rows_that_see_nothing(built_lib):
    import torch
    c = make([0, 0, 40], [4, 1, 3], 4, 2, 128, 16, "bf16", seed=5)
    c["mask"][1] = 0
    c["mask"][4] = 0
    got = check(c)
    assert (got[1] == 0).all() and (got[4] == 0).all() and (got[0] != 0).any()
    c["window"] = 0
    assert not torch.isnan(got).any()


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128, 512])
def test_hidden_values_are_never_used(built_lib, poison, dim):
    """Rows past a sequence's end, pages of nobody, other sequences' nodes and hidden siblings hold
    NaN or infinities; nodes that do not see them come out as if those were absent."""
    import torch
    c = make([37, 130, 0, 64], [9, 12, 5, 1], 4, 2, dim, 16, "bf16", seed=dim)
    want = run(c)
    for s, n in enumerate([37, 130, 0, 64]):
        if n % 16:
            last = c["table"][s, n // 16].long()
            c["k_pool"][last, n % 16:] = poison
            c["v_pool"][last, n % 16:] = poison
    used = torch.zeros(c["k_pool"].shape[0], dtype=torch.bool, device="cuda")
    used[c["table"][c["table"] >= 0].long()] = True
    c["k_pool"][~used] = poison
    c["v_pool"][~used] = poison
    assert torch.equal(run(c), want)
    # One node of sequence 1 (and of 0, which then is sequence 1's neighbour) becomes unusable: only
    # the nodes that see it change.
    mask = c["mask"].cpu().numpy().view(np.uint32)
    for base, n, j in ((9, 12, 7), (0, 9, 8)):
        c["v_new"][base + j, :, 3] = poison
        c["k_new"][base + j] = 0
        got = run(c)
        o, _, _ = formula(c)
        for i in range(n):
            sees = (mask[base + i, 0] >> j) & 1
            if not sees:
                assert torch.equal(got[base + i], want[base + i]), (base, i)
            else:
                assert (got[base + i, :, 3].double() == o[base + i, :, 3]).all() or torch.isnan(got[base + i, :, 3]).all()
        c["v_new"][base + j, :, 3] = 0
        want = run(c)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_window_hides_values_from_some_nodes(built_lib, poison):
    """A key that a deep node's window has passed but a shallow node's has not."""
    import torch
    c = make([300], [8], 4, 2, 128, 16, "bf16", seed=8, parents=[[-1, 0, 1, 2, 3, 4, 5, 6]])
    want = run(c, 100)
    key = 300 + 3 - 100  # seen by depths 0..2 only
    c["v_pool"][c["table"][0, key // 16].long(), key % 16, :, 5] = poison
    got = run(c, 100)
    assert torch.equal(got[3:], want[3:])
    assert not torch.isfinite(got[:3, :, 5]).any()
    assert torch.equal(got[:3, :, :5], want[:3, :, :5]) and torch.equal(got[:3, :, 6:], want[:3, :, 6:])


def test_strides_stream_and_interleaved_pool(built_lib):
    """q, k, v as slices of one projection, an output inside a wider buffer, K and V pages in one
    pool, and a stream of its own."""
    import torch
    c = make([200, 61], [6, 9], 8, 2, 128, 16, "bf16", seed=21)
    want = check(c)
    tokens = c["q"].shape[0]
    qkv = torch.zeros(tokens, 12, 128, dtype=torch.bfloat16, device="cuda")
    qkv[:, :8], qkv[:, 8:10], qkv[:, 10:] = c["q"], c["k_new"], c["v_new"]
    pages = c["k_pool"].shape[0]
    both = torch.zeros(pages, 2, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    both[:, 0], both[:, 1] = c["k_pool"], c["v_pool"]
    wide = torch.full((tokens, 10, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d = dict(c, q=qkv[:, :8], k_new=qkv[:, 8:10], v_new=qkv[:, 10:], k_pool=both[:, 0], v_pool=both[:, 1])
    with torch.cuda.stream(side):
        run(d, out=wide[:, 1:9], stream=side)
    side.synchronize()
    assert torch.equal(wide[:, 1:9], want) and (wide[:, 0] == 3).all() and (wide[:, 9] == 3).all()


def test_repeats_bit_for_bit_and_in_a_graph(built_lib):
    import torch
    from g4dense_b200 import api
    c = make([3000, 77, 1200], [9, 3, 5], 8, 2, 128, 16, "bf16", seed=30)
    want = check(c)
    for _ in range(3):
        assert torch.equal(run(c), want)
    out = torch.empty_like(c["q"])
    ws = torch.empty(api.tree_attention_workspace(9, 8, 2, 128), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()

    def go():
        api.tree_attention(c["q"], c["k_pool"], c["v_pool"], c["table"], c["lens"], c["k_new"], c["v_new"], c["cu"],
                           c["mask"], out, ws, max_nodes=9, scale=c["scale"], depth=c["depth"], stream=side)
    with torch.cuda.stream(side):
        go()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            go()
        c["lens"][0] = 2000  # lengths are read on the device
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, run(c)) and not torch.equal(out, want)


def test_empty_sequences_and_batches(built_lib):
    import torch
    c = make([50, 10, 90], [3, 0, 2], 4, 2, 64, 16, "bf16", seed=2)
    check(c)
    c = make([50], [0], 4, 2, 64, 16, "bf16", seed=2)
    run(c)  # no token at all
    # Bad device-side indices are skipped, not followed.
    c = make([50, 10], [3, 2], 4, 2, 64, 16, "bf16", seed=2)
    c["table"][0, 1] = 10 ** 6
    c["table"][1, 0] = -5
    c["lens"][0] = 10 ** 9
    run(c)
    torch.cuda.synchronize()


def test_refusals(built_lib):
    import torch
    from g4dense_b200 import api
    c = make([50], [3], 4, 2, 64, 16, "bf16", seed=2)
    ws = torch.empty(api.tree_attention_workspace(3, 4, 2, 64), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(c["q"])

    def call(**kw):
        a = dict(q=c["q"], k_pool=c["k_pool"], v_pool=c["v_pool"], table=c["table"], lens=c["lens"], k_new=c["k_new"],
                 v_new=c["v_new"], cu=c["cu"], mask=c["mask"], out=out, ws=ws, max_nodes=3, window=0, depth=None) | kw
        api.tree_attention(a["q"], a["k_pool"], a["v_pool"], a["table"], a["lens"], a["k_new"], a["v_new"], a["cu"],
                           a["mask"], a["out"], a["ws"], max_nodes=a["max_nodes"], scale=1.0, depth=a["depth"],
                           window=a["window"])
    call()
    with pytest.raises(ValueError, match="dtype"):
        call(q=c["q"].float())
    with pytest.raises(ValueError, match="k_new"):
        call(k_new=c["k_new"].half())
    with pytest.raises(ValueError, match="lens"):
        call(lens=c["lens"].long())
    with pytest.raises(ValueError, match="window"):
        call(window=5)
    with pytest.raises(RuntimeError, match="workspace too small"):
        call(ws=ws[:64])
    with pytest.raises(RuntimeError, match="1..256"):
        call(max_nodes=257)
    with pytest.raises(RuntimeError, match="mask_words"):
        call(max_nodes=40)
    with pytest.raises(RuntimeError, match="page_size"):
        call(k_pool=c["k_pool"][:, :12].contiguous(), v_pool=c["v_pool"][:, :12].contiguous())
    with pytest.raises(ValueError, match="64, 128, 256 or 512"):
        api.tree_attention_workspace(3, 4, 2, 96)
    with pytest.raises(ValueError, match="multiple"):
        api.tree_attention_workspace(3, 5, 2, 64)


@pytest.mark.parametrize("dim,nodes", [(256, 64), (512, 9), (64, 256)])
def test_windows_shorter_than_the_tree(built_lib, dim, nodes):
    """Chains of nodes longer than the window, whose first node falls anywhere in a group of 32 keys, with
    values that are not numbers in every row of the pages that no sequence holds; and nothing timed out."""
    import torch
    from g4dense_b200 import api
    lens = [0, 5, 31, 63, 104, 127]
    chain = [-1] + list(range(nodes - 1))
    c = make(lens, [nodes] * len(lens), 2, 1, dim, 8, "bf16", seed=dim, parents=[chain] * len(lens))
    held = torch.zeros(c["k_pool"].shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for j in range(n):
            held[c["table"][s, j // 8], j % 8] = True
    c["k_pool"][~held] = float("inf")
    c["v_pool"][~held] = float("nan")
    for window in (1, nodes // 2, nodes - 1, nodes, nodes + 40):
        check(c, window)
    api.tree_attention_check_error()
