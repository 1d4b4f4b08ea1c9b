"""The tree-verification operators over a paged K/V cache, in plain torch and through the library.

A round of speculative decoding over a batch of sequences with a drafted token tree each: the
attention of every node over its sequence's cached pages and its own ancestors ("attend"), one
token drawn per node from its logits row ("sample"), the accepted path walked and its K/V rows
written into the sequence's pages ("commit"), and the page keeping around it ("pages": a fork that
shares a prefix and the release of its copies, moving live pages together, copying pages to another
pool). `own` selects the library's kernels; otherwise the same results come from elementary torch
operations in 32 bits. `exact` restates the operators whose outputs are computed numbers in 64 bits.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# The sampling settings of the rows of a batch, in turn: temperature, top-k, top-p, min-p.
SETTINGS = [(0.8, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.7, 0, 1.0, 0.05), (1.3, 256, 1.0, 0.0),
            (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.9, 64, 0.8, 0.02)]


def listed():
    return [
        # One pending token of one short sequence with the small test models' heads: pure latency.
        dict(name="attend_one_token", op="attend", type="bf16", seqs=1, context=96, nodes=1, heads=4, kv_heads=4,
             dim=64, page=16, window=0),
        # Ragged batch, odd page size, fp16: sequences of 1..2500 cached tokens with trees of up to 13 nodes.
        dict(name="attend_ragged_f16", op="attend", type="f16", seqs=21, context=2500, nodes=13, heads=8, kv_heads=2,
             dim=128, page=24, window=0),
        # The 31B's sliding layers (32 query heads on 16 K/V heads of 256, a 1024-key window): 64-node trees.
        dict(name="attend_sliding_tree64", op="attend", type="bf16", seqs=32, context=4096, nodes=64, heads=32,
             kv_heads=16, dim=256, page=16, window=1024),
        # The 31B's full-attention layers (32 query heads on 4 K/V heads of 512) at 30 000 cached tokens, trees of
        # 9 nodes (the long-context verify width).
        dict(name="attend_full_30k", op="attend", type="bf16", seqs=8, context=30000, nodes=9, heads=32, kv_heads=4,
             dim=512, page=64, window=0),
        # One row over the small test vocabulary: latency.
        dict(name="sample_one_row", op="sample", type="f32", rows=1, vocab=4096),
        # A batch's tree nodes over the full vocabulary, every sampling setting among the rows.
        dict(name="sample_tree_batch", op="sample", type="bf16", rows=128, vocab=262144),
        # The end of a round for one sequence of a small model: accept, reserve, commit.
        dict(name="commit_small", op="commit", planes=8, row=256, page=16, seqs=1, nodes=5, context=70),
        # The end of a round for 64 sequences over the 31B's 50 sliding layers (K and V planes of 16 x 256).
        dict(name="commit_batch_31b", op="commit", planes=100, row=4096, page=16, seqs=64, nodes=16, context=41),
        # A prompt of one small model shared by two continuations.
        dict(name="fork_small", op="pages", what="fork", planes=8, row=256, page=16, seqs=4, context=70),
        # Best-of-n sampling: 24 prompts forked into 24 further continuations, partial pages copied, then released.
        dict(name="fork_batch_31b", op="pages", what="fork", planes=100, row=4096, page=32, seqs=48, context=75),
        # Live pages moved to the front of a pool before it is shrunk.
        dict(name="compact_pool", op="pages", what="compact", planes=20, row=2048, page=64, seqs=40, context=640),
        # Pages handed to another pool (a larger one, or the one sequences wait in).
        dict(name="copy_pages", op="pages", what="copy", planes=20, row=2048, page=64, seqs=24, context=640),
    ]


def spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "sample", "sample", "commit", "pages"])
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(4, 4, 64), (8, 8, 64), (8, 2, 128), (8, 1, 256), (32, 16, 256),
                                           (32, 8, 128), (32, 4, 512), (16, 1, 128), (12, 4, 128), (4, 1, 512)])
        nodes = spread(rng, 1, 64)
        context = spread(rng, 1, 30000)
        seqs = spread(rng, 1, 48)
        while seqs > 1 and (seqs * context * kv_heads * dim > 3.2e8 or seqs * nodes * heads * context * dim > 3.2e10):
            seqs //= 2
        return dict(op=op, type=rng.choice(["bf16", "bf16", "f16"]), seqs=seqs, context=context, nodes=nodes,
                    heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 16, 24, 32, 64, 128, 256]),
                    window=rng.choice([0, 0, 0, spread(rng, 16, 4096)]))
    if op == "sample":
        vocab = spread(rng, 50, 262144)
        rows = spread(rng, 1, 300)
        while rows > 1 and rows * vocab > 3.3e7:
            rows //= 2
        return dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), rows=rows, vocab=vocab)
    row = rng.choice([64, 256, 512, 1000, 2048, 4096])
    page = rng.choice([8, 16, 24, 32, 64])
    planes = spread(rng, 2, 100)
    seqs = spread(rng, 2 if op == "pages" else 1, 64)
    if op == "commit":
        context, nodes = spread(rng, 1, 300), spread(rng, 1, 48)
        while seqs > 1 and planes * row * seqs * (context + 2 * page + nodes) > 6e8:
            seqs //= 2
        return dict(op=op, planes=planes, row=row, page=page, seqs=seqs, nodes=nodes, context=context)
    context = spread(rng, 1, 700)
    while seqs > 2 and planes * row * seqs * (context + 2 * page) > 4e8:
        seqs //= 2
    while planes > 2 and planes * row * seqs * (context + 2 * page) > 4e8:
        planes //= 2
    return dict(op=op, what=rng.choice(["fork", "compact", "copy"]), planes=planes, row=row, page=page, seqs=seqs,
                context=context)


# ------------------------------------------------------------------------------------------ sizes

def ceil_div(a, b):
    return -(-a // b)


def lengths(case):
    """Cached tokens of each sequence: the longest first, then ragged, some very short."""
    rng = random.Random(case["seqs"] * 1000003 + case["context"])
    c = case["context"]
    return [c if i == 0 else rng.randint(0, min(c, 3)) if i % 11 == 7 else rng.randint((c + 1) // 2, c)
            for i in range(case["seqs"])]


def tree_sizes(case):
    """Nodes of each sequence's tree: the largest first, then ragged, some of the root alone."""
    rng = random.Random(case["seqs"] * 7919 + case["nodes"])
    n = case["nodes"]
    return [n if i % 3 == 0 else 1 if i % 7 == 5 else rng.randint((n + 1) // 2, n) for i in range(case["seqs"])]


def trees(sizes, rng):
    """Parents, depths and ancestor bit masks (32-bit words) of a random tree per sequence, node 0 its root."""
    words = ceil_div(max(sizes), 32)
    parents, depths, masks = [], [], []
    for n in sizes:
        up, deep, seen = [-1], [0], [1]
        for i in range(1, n):
            p = rng.randint(max(0, i - 6), i - 1)
            up.append(p)
            deep.append(deep[p] + 1)
            seen.append(seen[p] | 1 << i)
        parents += up
        depths += deep
        masks += [[((s >> 32 * w & 0xFFFFFFFF) ^ 0x80000000) - 0x80000000 for w in range(words)] for s in seen]
    return parents, depths, masks


def offsets(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def whole(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def paged(case, lens, spare, rng, width=None):
    """A block table over a shuffled pool: (table rows, page count, reference counts)."""
    page = case["page"]
    need = [ceil_div(n, page) for n in lens]
    width = width or max(1, max(need))
    total = sum(need) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    table, at, refs = [], 0, [0] * total
    for n in need:
        row = ids[at:at + n]
        at += n
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (width - n))
    return table, total, refs


# ----------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

    if case["op"] == "attend":
        kind, dim = TYPES[case["type"]], case["dim"]
        lens, sizes = lengths(case), tree_sizes(case)
        table, pages, _ = paged(case, lens, 3, rng)
        _, depths, masks = trees(sizes, rng)
        total = sum(sizes)
        pool = (pages, case["page"], case["kv_heads"], dim)
        return dict(case=case, q=normal(total, case["heads"], dim, dtype=kind, std=2.0),
                    k_pool=normal(*pool, dtype=kind), v_pool=normal(*pool, dtype=kind),
                    k_new=normal(total, case["kv_heads"], dim, dtype=kind),
                    v_new=normal(total, case["kv_heads"], dim, dtype=kind), table=whole(table), lens=whole(lens),
                    cu=whole(offsets(sizes)), mask=whole(masks), depth=whole(depths),
                    out=torch.empty((total, case["heads"], dim), dtype=kind, device="cuda"))
    if case["op"] == "sample":
        rows = case["rows"]
        picked = [SETTINGS[r % len(SETTINGS)] for r in range(rows)]
        f32 = dict(dtype=torch.float32, device="cuda")
        return dict(case=case, logits=normal(rows, case["vocab"], dtype=TYPES[case["type"]], std=2.5),
                    uniform=torch.rand(rows, generator=g, **f32), temperature=torch.tensor([s[0] for s in picked], **f32),
                    top_k=whole([s[1] for s in picked]), top_p=torch.tensor([s[2] for s in picked], **f32),
                    min_p=torch.tensor([s[3] for s in picked], **f32), token=torch.empty(rows, dtype=torch.int32, device="cuda"),
                    prob=torch.empty(rows, **f32), kept=torch.empty(rows, dtype=torch.int32, device="cuda"))

    lens, page = lengths(case), case["page"]
    if case["op"] == "commit":
        sizes = tree_sizes(case)
        width = ceil_div(case["context"] + case["nodes"], page)
        table, pages, refs = paged(case, lens, sum(ceil_div(n, page) + 1 for n in sizes), rng, width)
        parents, depths, masks = trees(sizes, rng)
        tokens = [rng.randrange(262144) for _ in parents]
        sampled, at = [rng.randrange(262144) for _ in parents], 0
        for n in sizes:  # most nodes draw the token of one of their children
            for i in range(1, n):
                if rng.random() < 0.75:
                    sampled[at + parents[at + i]] = tokens[at + i]
            at += n
        deepest = case["nodes"]
        return dict(case=case, pool=normal(case["planes"], pages, page, case["row"]),
                    rows=normal(case["planes"], sum(sizes), case["row"]), table=whole(table), lens=whole(lens),
                    refs=whole(refs), cu=whole(offsets(sizes)), parents=whole(parents), depth=whole(depths),
                    mask=whole(masks), tokens=whole(tokens), sampled=whole(sampled),
                    path=torch.empty((case["seqs"], deepest), dtype=torch.int32, device="cuda"),
                    count=whole([0] * case["seqs"]), next=whole([0] * case["seqs"]), table_out=whole(table),
                    refs_out=whole(refs), lens_out=whole(lens), status=whole([0]))
    if case["what"] == "fork":
        half = case["seqs"] // 2
        lens = [n if i < half else 0 for i, n in enumerate(lens)]
        table, pages, refs = paged(case, lens, half + 2, rng)
        out = dict(src=whole([rng.randrange(half) for _ in range(half)]), dst=whole(list(range(half, 2 * half))),
                   lens_out=whole(lens), lens_freed=whole(lens), table_freed=whole(table), refs_freed=whole(refs))
    else:
        table, pages, refs = paged(case, lens, sum(ceil_div(n, page) for n in lens) // 2 + 1, rng)
        if case["what"] == "compact":
            out = dict(moves=torch.full((1 + 2 * pages,), -1, dtype=torch.int32, device="cuda"))
        else:
            used = [p for row in table for p in row if p >= 0]
            there = list(range(len(used) + 5))
            rng.shuffle(there)
            out = dict(src=whole(used), dst=whole(there[:len(used)]),
                       other=normal(case["planes"], len(there), page, case["row"]))
    return dict(case=case, pool=normal(case["planes"], pages, page, case["row"]), table=whole(table), lens=whole(lens),
                refs=whole(refs), table_out=whole(table), refs_out=whole(refs), status=whole([0]), **out)


# ------------------------------------------------------------------------------------ plain forms

def plain_attend(s):
    q, cu, lens = s["q"].float(), s["cu"].long(), s["lens"].long()
    case = s["case"]
    page, nodes, window = case["page"], case["nodes"], case["window"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    seqs, total = lens.numel(), q.shape[0]
    at = torch.arange(case["context"], device=q.device)
    held = at[None] < lens[:, None]
    pages = s["table"].long()[:, at // page].clamp(min=0)
    node = torch.arange(nodes, device=q.device)
    real = node[None] < (cu[1:] - cu[:-1])[:, None]
    idx = (cu[:-1, None] + node[None]).clamp(max=total - 1)
    zero = torch.zeros((), device=q.device)

    def keys(pool, new):
        old = torch.where(held[:, :, None, None], pool[pages, (at % page)[None]].float(), zero)
        fresh = torch.where(real[:, :, None, None], new[idx].float(), zero)
        return torch.cat([old, fresh], 1)

    k, v = keys(s["k_pool"], s["k_new"]), keys(s["v_pool"], s["v_new"])
    depth = s["depth"].long()[idx]
    bits = (s["mask"].long()[idx][:, :, node // 32] >> (node % 32)) & 1
    seen_new = (bits == 1) & real[:, None]
    seen_old = held[:, None].expand(seqs, nodes, -1)
    if window:
        pos = lens[:, None] + depth
        seen_old = seen_old & (pos[:, :, None] - at < window)
        seen_new = seen_new & (depth[:, :, None] - depth[:, None] < window)
    seen = torch.cat([seen_old, seen_new], 2)[:, None, None]
    qs = q[idx].reshape(seqs, nodes, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(qs.reshape(seqs, kv, -1, dim), k.permute(0, 2, 3, 1)) * dim ** -0.5
    score = score.reshape(seqs, kv, heads // kv, nodes, -1).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), zero, top))
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    out = torch.matmul(e.reshape(seqs, kv, -1, e.shape[-1]), v.permute(0, 2, 1, 3))
    out = out.reshape(seqs, heads, nodes, dim).permute(0, 2, 1, 3)
    return out[real].to(s["q"].dtype)


def plain_sample(s):
    x = s["logits"].float()
    t, k, p, low = s["temperature"][:, None], s["top_k"][:, None], s["top_p"][:, None], s["min_p"][:, None]
    vocab = x.shape[1]
    x = torch.where(torch.isnan(x), -math.inf, x)
    line, order = torch.sort(x, dim=1, descending=True, stable=True)
    live = line > -math.inf
    heat = torch.where(t > 0, t, torch.ones_like(t))
    e = torch.exp((line - line[:, :1]) / heat)
    # Weights as whole numbers of 2^-40: their sums are exact in any order.
    w = torch.where(live, (e * 2.0 ** 40), 0.0).long()
    rank = torch.arange(vocab, device=x.device)[None]
    k = torch.where(t > 0, torch.where(k > 0, k, vocab), 1)
    keep = live & (rank < k)
    w = torch.where(keep, w, 0)
    mass = w.sum(1, keepdim=True)
    before = w.cumsum(1) - w
    keep = keep & ((p >= 1.0) | (before.double() < p.double() * mass.double())) & (e >= low)
    w = torch.where(keep, w, 0)
    total = w.sum(1)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    r = torch.floor(s["uniform"].double() * total.double()).long()
    token = (by_index.cumsum(1) <= r[:, None]).sum(1).clamp(max=vocab - 1)
    prob = by_index.gather(1, token[:, None])[:, 0].float() / total.float()
    return dict(token=token.int(), prob=prob, kept=keep.sum(1).int())


def plain_reserve(refs, table, lens, grow, page):
    have, want = (lens + page - 1) // page, (lens + grow + page - 1) // page
    col = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    rank = fresh.reshape(-1).long().cumsum(0) - 1
    free = torch.sort((refs != 0).long(), stable=True)[1]
    ids = free[rank.clamp(min=0)].reshape(fresh.shape).int()
    taken = torch.zeros_like(refs).index_put_((ids[fresh].long(),), torch.ones((), dtype=torch.int32, device=refs.device))
    return refs + taken, torch.where(fresh, ids, table)


def plain_commit(s):
    cu, lens, page, case = s["cu"].long(), s["lens"], s["case"]["page"], s["case"]
    nodes = case["nodes"]
    node = torch.arange(nodes, device=lens.device)
    total = s["tokens"].numel()
    real = node[None] < (cu[1:] - cu[:-1])[:, None]
    idx = (cu[:-1, None] + node[None]).clamp(max=total - 1)
    tok, up = s["tokens"][idx], s["parents"].long()[idx]
    drawn = s["sampled"][idx]
    good = real & (up >= 0) & (tok == drawn.gather(1, up.clamp(min=0)))
    same = good[:, None] & (up[:, :, None] == up[:, None]) & (node[None, :, None] > node[None, None])
    good = (good & ~same.any(2)) | (real & (node == 0)[None])
    bits = ((s["mask"].long()[idx][:, :, node // 32] >> (node % 32)) & 1) == 1
    taken = real & ~(bits & ~good[:, None]).any(2)
    count = taken.sum(1).int()
    place = torch.where(taken, s["depth"].long()[idx], nodes)
    path = torch.full((lens.numel(), nodes + 1), -1, dtype=torch.int32, device=lens.device)
    path = path.scatter(1, place, node[None].int().expand_as(idx).contiguous())[:, :nodes].contiguous()
    last = path.long().gather(1, (count.long() - 1)[:, None])
    following = drawn.gather(1, last)[:, 0]
    refs, table = plain_reserve(s["refs"], s["table"], lens, count, page)
    pos = lens[:, None] + node[None]
    put = node[None] < count[:, None]
    page_of = table.long().gather(1, (pos // page).long().clamp(max=table.shape[1] - 1))
    rows = cu[:-1, None] + path.long()
    s["pool"][:, page_of[put], (pos % page).long()[put]] = s["rows"][:, rows[put]]
    return dict(path=path, count=count, next=following, table=table, refs=refs, lens=lens + count,
                status=torch.zeros_like(s["status"]), pool=s["pool"])


def plain_fork(s):
    page, table, refs, lens = s["case"]["page"], s["table"], s["refs"], s["lens"]
    src, dst = s["src"].long(), s["dst"].long()
    full, rest = (lens[src] // page).long(), lens[src] % page
    part = rest > 0
    free = torch.sort((refs != 0).long(), stable=True)[1]
    fresh = free[(part.long().cumsum(0) - 1).clamp(min=0)].int()
    rows = table[src].clone()
    col = torch.arange(rows.shape[1], device=rows.device)[None]
    tail = (col == full[:, None]) & part[:, None]
    old = rows[tail].long()
    new = fresh[part].long()
    rows[tail] = fresh[part]
    shared = rows[col < full[:, None]].long()
    one = torch.ones((), dtype=torch.int32, device=refs.device)
    refs_out = refs.index_put((torch.cat([shared, new]),), one, accumulate=True)
    table_out, lens_out = table.index_put((dst,), rows), lens.index_put((dst,), lens[src])
    slot = torch.arange(page, device=rows.device)
    keep = (slot[None] < rest[part][:, None])[None, :, :, None]
    s["pool"][:, new] = torch.where(keep, s["pool"][:, old], s["pool"][:, new])
    # The forked continuations end: their references go, and pages nobody holds are free again.
    gone = table_out[dst]
    refs_freed = refs_out.index_put((gone[gone >= 0].long(),), -one, accumulate=True)
    return dict(table=table_out, refs=refs_out, lens=lens_out, status=torch.zeros_like(s["status"]), pool=s["pool"],
                table_freed=table_out.index_put((dst,), -one), refs_freed=refs_freed,
                lens_freed=lens_out.index_put((dst,), 0 * one))


def plain_compact(s):
    refs, table = s["refs"], s["table"]
    ids = torch.arange(refs.numel(), device=refs.device)
    live = refs != 0
    front = ids < live.sum()
    old, new = ids[live & ~front], ids[~live & front]
    goes = ids.index_put((old,), new)
    table_out = torch.where(table >= 0, goes[table.long().clamp(min=0)].int(), table)
    refs_out = torch.where(front, refs, 0).index_put((new,), refs[old])
    moves = torch.full_like(s["moves"], -1)
    moves[0] = old.numel()
    moves[1:1 + 2 * old.numel()] = torch.stack([old, new], 1).reshape(-1).int()
    s["pool"][:, new] = s["pool"][:, old]
    return dict(table=table_out, refs=refs_out, moves=moves, pool=s["pool"])


def plain_copy(s):
    s["other"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    return s["other"]


# ------------------------------------------------------------------------------- through the library

def library():
    where = str(Path(__file__).resolve().parent.parent / "turbo-winfare-dense_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    from g4dense_b200 import api
    return api


def own_run(s):
    api, case = library(), s["case"]
    if case["op"] == "attend":
        if "workspace" not in s:
            need = api.tree_attention_workspace(case["nodes"], case["heads"], case["kv_heads"], case["dim"])
            s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        api.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], s["k_new"], s["v_new"], s["cu"],
                           s["mask"], s["out"], s["workspace"], max_nodes=case["nodes"], scale=case["dim"] ** -0.5,
                           depth=s["depth"], window=case["window"])
        return s["out"]
    if case["op"] == "sample":
        api.sample_rows(s["logits"], s["uniform"], s["token"], prob=s["prob"], kept=s["kept"],
                        temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return dict(token=s["token"], prob=s["prob"], kept=s["kept"])
    if case["op"] == "commit":
        api.tree_accept(s["tokens"], s["parents"], s["sampled"], s["cu"], s["path"], s["count"], s["next"])
        api.pages_reserve(s["refs"], s["table"], s["lens"], s["count"], case["page"], s["refs_out"], s["table_out"],
                          s["status"])
        api.pages_commit(s["pool"], s["table_out"], s["lens"], s["rows"], s["cu"], s["path"], s["count"], s["lens_out"])
        return dict(path=s["path"], count=s["count"], next=s["next"], table=s["table_out"], refs=s["refs_out"],
                    lens=s["lens_out"], status=s["status"], pool=s["pool"])
    if case["what"] == "fork":
        api.pages_fork(s["pool"], s["refs"], s["table"], s["lens"], s["src"], s["dst"], s["refs_out"], s["table_out"],
                       s["lens_out"], s["status"])
        api.pages_free(s["refs_out"], s["table_out"], s["lens_out"], s["dst"], case["page"], s["refs_freed"],
                       s["table_freed"], s["lens_freed"])
        return dict(table=s["table_out"], refs=s["refs_out"], lens=s["lens_out"], status=s["status"], pool=s["pool"],
                    table_freed=s["table_freed"], refs_freed=s["refs_freed"], lens_freed=s["lens_freed"])
    if case["what"] == "compact":
        api.pages_compact(s["pool"], s["refs"], s["table"], s["refs_out"], s["table_out"], s["moves"])
        return dict(table=s["table_out"], refs=s["refs_out"], moves=s["moves"], pool=s["pool"])
    api.pages_copy(s["pool"], s["other"], s["src"], s["dst"])
    return s["other"]


def run(state):
    if own:
        return own_run(state)
    case = state["case"]
    if case["op"] == "pages":
        return {"fork": plain_fork, "compact": plain_compact, "copy": plain_copy}[case["what"]](state)
    return {"attend": plain_attend, "sample": plain_sample, "commit": plain_commit}[case["op"]](state)


# ------------------------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "attend":
        lens, sizes, window = lengths(case), tree_sizes(case), case["window"]
        size = 4 if case["type"] == "f32" else 2
        seen = [min(n, window) if window else n for n in lens]
        rows = sum(sizes) * case["heads"] * case["dim"]
        keys = (sum(seen) + sum(sizes)) * case["kv_heads"] * case["dim"]
        pairs = sum(m * (n + ceil_div(m, 2)) for n, m in zip(seen, sizes))
        return dict(bytes=2 * size * (rows + keys) + 4 * sum(sizes) * ceil_div(case["nodes"], 32),
                    flops=4 * pairs * case["heads"] * case["dim"])
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (4 if case["type"] == "f32" else 2) + case["rows"] * 32, flops=8 * n)
    lens, page = lengths(case), case["page"]
    token = 2 * 2 * case["planes"] * case["row"]  # one token's rows read and written
    entries = sum(ceil_div(n, page) for n in lens)
    if case["op"] == "commit":
        sizes = tree_sizes(case)
        # Accepted depths vary with the draws; every tree commits its root, and most a few nodes more.
        return dict(bytes=token * sum(min(n, 3) for n in sizes) + 8 * entries + 12 * sum(sizes), flops=sum(sizes))
    if case["what"] == "fork":
        half = case["seqs"] // 2
        return dict(bytes=token * sum(n % page for n in lens[:half]) + 16 * entries, flops=entries)
    if case["what"] == "compact":
        total = entries + entries // 2 + 1
        moved = entries * (total - entries) // total
        return dict(bytes=token * page * moved + 8 * (entries + total), flops=total)
    return dict(bytes=token * page * entries + 8 * entries, flops=entries)


# ---------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    if case["op"] == "attend":
        s = prepare(case, seed)
        dim, window, group = case["dim"], case["window"], case["heads"] // case["kv_heads"]
        cu, lens, outs = s["cu"].tolist(), s["lens"].tolist(), []
        for b, n in enumerate(lens):
            a, z = cu[b], cu[b + 1]
            m = z - a
            ids = s["table"][b, :ceil_div(n, case["page"])].long()
            first = max(0, n - window + 1) if window else 0

            def side(pool, new):
                old = pool[ids].reshape(-1, case["kv_heads"], dim)[first:n]
                return torch.cat([old, new[a:z]]).double().permute(1, 0, 2)

            k, v = side(s["k_pool"], s["k_new"]), side(s["v_pool"], s["v_new"])
            words = s["mask"][a:z].cpu().tolist()
            tree = torch.tensor([[(row[j // 32] >> (j % 32)) & 1 for j in range(m)] for row in words]) == 1
            hide = torch.cat([torch.zeros(m, n - first, dtype=torch.bool), ~tree], 1).cuda()
            if window:
                depth = s["depth"][a:z].long()
                pos = torch.cat([torch.arange(first, n, device="cuda"), n + depth])
                hide |= (n + depth)[:, None] - pos[None] >= window
            q = s["q"][a:z].double().reshape(m, case["kv_heads"], group, dim)
            score = torch.einsum("mhgd,hld->hgml", q, k) / math.sqrt(dim)
            p = torch.softmax(score.masked_fill(hide, -math.inf), -1)
            outs.append(torch.einsum("hgml,hld->mhgd", p, v).reshape(m, case["heads"], dim))
        return torch.cat(outs)
    if case["op"] == "sample":
        s = prepare(case, seed)
        x, probs = s["logits"].double(), []
        for r in range(case["rows"]):
            t, k, p, low = SETTINGS[r % len(SETTINGS)]
            if t <= 0:
                probs.append(torch.ones((), dtype=torch.float64, device="cuda"))
                continue
            w = torch.exp((x[r] - x[r].max()) / float(s["temperature"][r]))
            order = torch.argsort(w, descending=True, stable=True)
            order = order[:k] if k else order
            line = w[order]
            keep = line >= float(s["min_p"][r])
            if p < 1:
                keep &= line.cumsum(0) - line < float(s["top_p"][r]) * line.sum()
            left = torch.zeros_like(w)
            left[order[keep]] = line[keep]
            line = left.cumsum(0)
            i = int(torch.searchsorted(line, float(s["uniform"][r]) * line[-1:], right=True))
            probs.append(left[min(i, left.numel() - 1)] / line[-1])
        return dict(token=None, prob=torch.stack(probs), kept=None)
    return None
