"""Row sampling, tree acceptance and page keeping against plain implementations.

Pages, tables, counts and accepted paths are whole numbers or copies: equality. Sampled tokens are
checked against the distribution in 64 bits: the kernel's weights are within E = 2^-20 of exact ones
(the quotient's rounding, |x| <= 28 times 2^-24, two units in the last place of expf, and 2^-40 of
truncation), so the token's interval of the running mass holds u within 2 E, the kept set is a prefix
of the descending order whose end lies within 2 E of the cut, and prob is right to 4 E. Rows whose
weights are exact (equal logits) are checked for equality.
"""
from __future__ import annotations

import random

import numpy as np
import pytest

E = 2.0 ** -20


# ------------------------------------------------------------------------------------- sampling

def sample(logits, u, **kw):
    import torch
    from g4dense_b200 import api
    rows = logits.shape[0]
    f = lambda x, d: None if x is None else torch.tensor(x, dtype=d, device="cuda")  # noqa: E731
    token = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -7.0, device="cuda")
    kept = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    api.sample_rows(logits, f(u, torch.float32), token, prob=prob, kept=kept,
                    temperature=f(kw.get("temperature"), torch.float32), top_k=f(kw.get("top_k"), torch.int32),
                    top_p=f(kw.get("top_p"), torch.float32), min_p=f(kw.get("min_p"), torch.float32))
    return token.tolist(), prob.tolist(), kept.tolist()


def check_row(x, u, t, k, p, low, token, prob, kept):
    """x: float64 logits of one row."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    live = int((x > -np.inf).sum())
    t, p, low, u = (float(np.float32(v)) for v in (t, p, low, u))
    if live == 0:
        assert (token, prob, kept) == (-1, 0.0, 0)
        return
    if t <= 0:
        assert (token, prob, kept) == (order[0], 1.0, 1)
        return
    w = np.exp((x - x[order[0]]) / t)
    line = w[order]
    n = min(live, k) if k > 0 else live
    mass = line[:n].sum()
    before = np.concatenate([[0], np.cumsum(line)[:-1]])
    fits = lambda slack: int(((before[:n] < (p + slack) * mass) | (p >= 1)).sum())  # noqa: E731
    lo, hi = max(1, fits(-2 * E)), fits(2 * E)
    heavy = lambda f: int((line >= low * f).sum())  # noqa: E731
    lo, hi = min(lo, heavy(1 + 2 * E)), min(hi, heavy(1 - 2 * E))
    assert max(1, lo) <= kept <= max(1, hi), (lo, kept, hi)
    held = np.zeros(len(x))
    held[order[:kept]] = line[:kept]
    assert held[token] > 0
    total = held.sum()
    upto = held[:token + 1].sum()
    assert upto - held[token] <= (u + 2 * E) * total and upto >= (u - 2 * E) * total
    assert abs(prob - held[token] / total) <= 4 * E * held[token] / total


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.7, 0, 1.0, 0.05), (1.5, 7, 1.0, 0.0),
            (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (2.0, 300, 0.3, 0.1), (0.05, 0, 0.999, 0.0), (1.0, 0, 1e-6, 0.0),
            (30.0, 0, 0.5, 0.0), (1.0, 10 ** 6, 1.0, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 1000, 4096, 4097, 16384, 16385, 50001, 131072, 262143, 262144])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sample_rows(built_lib, vocab, dtype):
    import torch
    kind = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    g = torch.Generator().manual_seed(vocab)
    rows = len(SETTINGS)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(kind)
    u = torch.rand(rows, generator=g).tolist()
    u[0], u[1], u[2] = 0.0, 1.0 - 2.0 ** -24, 0.5
    t, k, p, low = zip(*SETTINGS)
    token, prob, kept = sample(x.cuda(), u, temperature=t, top_k=k, top_p=p, min_p=low)
    for r in range(rows):
        check_row(x[r].double().numpy(), u[r], t[r], k[r], p[r], low[r], token[r], prob[r], kept[r])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 700, 40000, 262144])
def test_sample_rows_exact_weights(built_lib, vocab):
    """Equal logits: every weight is 1, so counts and tokens follow from u alone; ties go to the lowest
    index."""
    import torch
    x = torch.full((6, vocab), -2.5, device="cuda")
    half = vocab // 2
    x[3, :half] = 1.0
    x[4, half:] = 40.0
    u = [0.0, 0.75, 0.3, 0.999, 0.25, 0.5]
    k, p = [0, 4, 0, 0, 3, vocab], [1.0, 1.0, 0.5, 0.25, 1.0, 1.0]
    token, prob, kept = sample(x, u, top_k=k, top_p=p)
    n = [vocab, 4, -(-vocab // 2), None, 3, vocab]
    for r, base in ((0, 0), (1, 0), (2, 0), (4, half), (5, 0)):
        assert kept[r] == n[r] and token[r] == base + int(np.float64(np.float32(u[r])) * n[r]), r
        assert prob[r] == np.float32(1) / np.float32(n[r])
    assert token[3] < half


@pytest.mark.gpu
def test_sample_rows_special_values(built_lib):
    """Masked entries, whole rows masked, infinities and NaN, the type's lowest values, unaligned and
    strided rows, numbers outside [0, 1)."""
    import torch
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    x = torch.zeros(12, 3000)
    x[0] = -inf
    x[1] = nan
    x[2], x[2, 77] = -inf, -80.0
    x[3, 5:] = nan
    x[4, 100], x[4, 200] = inf, inf
    x[5] = low
    x[6], x[6, 9] = low, low / 2
    x[7], x[7, 2999] = -inf, nan
    x[8, 0] = -0.0
    x[9], x[9, 1500] = -inf, inf
    x[10, :2999] = -1e4
    x[11] = torch.arange(3000) % 2 * -inf
    x[11][torch.isnan(x[11])] = 0.0
    u = [0.5, 0.5, 0.5, 0.99, 0.6, 0.5, 0.5, 0.1, -3.0, 0.2, 1.5, nan]
    token, prob, kept = sample(x.cuda(), u, top_p=[1, 1, 0.5, 1, 1, 1, 1, 1, 1, 1, 0.9, 1])
    assert (token[0], prob[0], kept[0]) == (-1, 0.0, 0) and token[1] == -1 and token[7] == -1
    assert (token[2], prob[2], kept[2]) == (77, 1.0, 1)
    assert kept[3] == 5 and token[3] == 4
    # +inf outweighs every finite entry; the others are kept with weight 0.
    assert token[4] == 200 and prob[4] == 0.5
    assert kept[5] == 3000 and token[5] == 1500
    assert token[6] == 9 and prob[6] == 1.0
    assert token[8] == 0 and kept[8] == 3000 and token[9] == 1500 and token[10] == 2999 and token[11] == 0
    wide = torch.zeros(5, 1003, device="cuda")
    g = torch.Generator().manual_seed(1)
    wide[:, 1:1001] = (torch.randn(5, 1000, generator=g) * 2).cuda()
    view = wide[:, 1:1001]
    u = [0.1, 0.3, 0.5, 0.7, 0.9]
    assert sample(view, u, top_p=[0.9] * 5) == sample(view.contiguous(), u, top_p=[0.9] * 5)
    h = wide.to(torch.bfloat16)
    assert sample(h[:, 1:1001], u, top_k=[50] * 5) == sample(h[:, 1:1001].contiguous(), u, top_k=[50] * 5)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 40000, 262144])
def test_sample_rows_wide_cuts(built_lib, vocab):
    """Cuts that leave thousands of entries, by number and by mass, in rows with and without ties, and
    cuts that fall far below the maximum (where most entries share the last histogram bin)."""
    import torch
    g = torch.Generator().manual_seed(vocab + 1)
    settings = [(1.0, vocab // 2, 1.0, 0.0), (1.0, vocab // 3, 0.5, 0.0), (0.02, vocab // 2, 1.0, 0.0), (1.0, 0, 0.5, 0.0),
                (4.0, 0, 0.9, 0.0), (0.01, 500, 1.0, 0.0), (50.0, 700, 0.7, 0.0), (1.0, vocab - 1, 0.999, 0.001)]
    for kind in (torch.float32, torch.bfloat16):
        x = (torch.randn(len(settings), vocab, generator=g) * 2).to(kind)
        x[6] = torch.round(x[6].float() / 3).to(kind)  # ties by the thousand
        u = torch.rand(len(settings), generator=g).tolist()
        t, k, p, low = zip(*settings)
        token, prob, kept = sample(x.cuda(), u, temperature=t, top_k=k, top_p=p, min_p=low)
        for r in range(len(settings)):
            check_row(x[r].double().numpy(), u[r], t[r], k[r], p[r], low[r], token[r], prob[r], kept[r])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1500, 262144])
@pytest.mark.parametrize("p", [1.0, 0.9, 1e-6])
def test_sample_rows_list_lengths(built_lib, vocab, p):
    """Short cuts by number around the lengths at which a list is ranked, searched or left to all blocks,
    without ties and with hundreds of entries in a tie across the cut."""
    import torch
    g = torch.Generator().manual_seed(vocab + 2)
    ks = [254, 255, 256, 257, 511, 512, 513, 600, 1022, 1023, 1024, 1025]
    x = torch.randn(2 * len(ks), vocab, generator=g) * 2
    x[len(ks):, :300] = x[len(ks):].median(1, keepdim=True).values + 9
    u = torch.rand(2 * len(ks), generator=g).tolist()
    token, prob, kept = sample(x.cuda(), u, top_k=ks * 2, top_p=[p] * len(u))
    for r, k in enumerate(ks * 2):
        check_row(x[r].double().numpy(), u[r], 1.0, k, p, 0.0, token[r], prob[r], kept[r])


@pytest.mark.gpu
def test_sample_rows_split_does_not_matter(built_lib):
    """A row alone is spread over more blocks than among many: the same token, share and count."""
    import torch
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(1, 100000, generator=g) * 2).cuda()
    for kw in (dict(top_p=0.97), dict(top_k=50), dict(top_k=3000, top_p=0.8), dict(min_p=0.01), dict()):
        one = sample(x, [0.37], **{k: [v] for k, v in kw.items()})
        many = sample(x.repeat(300, 1), [0.37] * 300, **{k: [v] * 300 for k, v in kw.items()})
        assert all(set(m) == set(o) for m, o in zip(many, one)), kw


@pytest.mark.gpu
def test_sample_rows_frequencies(built_lib):
    """Evenly spaced uniform numbers hit each kept entry as often as its probability says."""
    import torch
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625])
    n = 1024
    x = torch.log(p)[None].repeat(n, 1).cuda()
    u = [(i + 0.5) / n for i in range(n)]
    token, _, _ = sample(x, u)
    counts = np.bincount(token, minlength=5)
    assert np.abs(counts - p.numpy() * n).max() <= 1, counts
    token, _, kept = sample(x, u, top_k=[2] * n)
    assert set(kept) == {2} and np.abs(np.bincount(token, minlength=5)[:2] - np.array([2, 1]) * n / 3).max() <= 1


@pytest.mark.gpu
def test_sample_rows_refusals(built_lib):
    import torch
    from g4dense_b200 import api
    x = torch.zeros(2, 10, device="cuda")
    u, tok = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    api.sample_rows(x, u, tok)
    with pytest.raises(ValueError, match="dtype"):
        api.sample_rows(x.double(), u, tok)
    with pytest.raises(ValueError, match="uniform"):
        api.sample_rows(x, u[:1], tok)
    with pytest.raises(ValueError, match="token"):
        api.sample_rows(x, u, tok.long())
    with pytest.raises(RuntimeError, match="262144"):
        api.sample_rows(torch.zeros(2, 262145, device="cuda"), u, tok)


# ----------------------------------------------------------------------------------- acceptance

def accept_plain(tokens, parents, sampled, width):
    path, cur = [], 0
    while cur is not None and len(tokens) and len(path) < width:
        path.append(cur)
        nxt = sampled[cur]
        cur = next((i for i in range(cur + 1, len(tokens)) if parents[i] == path[-1] and tokens[i] == nxt), None)
    return path, (sampled[path[-1]] if path else -1)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 3, 256])
def test_tree_accept(built_lib, width):
    import torch
    from g4dense_b200 import api
    rng = random.Random(width)
    sizes = [1, 0, 2, 5, 31, 32, 33, 64, 100, 255, 256, 1, 256]
    tokens, parents, sampled, want = [], [], [], []
    for s, n in enumerate(sizes):
        up = [-1] + [i - 1 if s == 12 else rng.randrange(max(0, i - 4), i) for i in range(1, n)]
        up = up[:n]
        tk = [rng.randrange(3) if s != 12 else 7 for _ in range(n)]  # few values: siblings with equal tokens
        sm = [rng.randrange(3) if s != 12 else 7 for _ in range(n)]
        want.append(accept_plain(tk, up, sm, width))
        tokens, parents, sampled = tokens + tk, parents + up, sampled + sm
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cu = t([0] + np.cumsum(sizes).tolist())
    path, count, nxt = t([[5] * width] * len(sizes)), t([9] * len(sizes)), t([9] * len(sizes))
    api.tree_accept(t(tokens), t(parents), t(sampled), cu, path, count, nxt)
    for s, (p, after) in enumerate(want):
        assert count[s].item() == len(p) and nxt[s].item() == after
        assert path[s].tolist() == p + [-1] * (width - len(p))
    if width == 256:
        assert count[12].item() == 256
    with pytest.raises(ValueError, match="sampled"):
        api.tree_accept(t(tokens), t(parents), t(sampled[:-1]), cu, path, count, nxt)


# ---------------------------------------------------------------------------------------- pages

class Plain:
    """The same page keeping on NumPy arrays; a call that fails changes nothing."""

    def __init__(self, pool, seqs, width):
        self.pool, self.page = pool, pool.shape[2]
        self.refs = np.zeros(pool.shape[1], np.int32)
        self.table = np.full((seqs, width), -1, np.int32)
        self.lens = np.zeros(seqs, np.int32)

    def free_ids(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def reserve(self, grow):
        want = [-(-int(n + g) // self.page) for n, g in zip(self.lens, grow)]
        if any(g < 0 for g in grow) or any(w > self.table.shape[1] for w in want):
            return 2
        cells = [(s, c) for s, w in enumerate(want) for c in range(-(-int(self.lens[s]) // self.page), w)
                 if self.table[s, c] < 0]
        ids = self.free_ids()
        if len(ids) < len(cells):
            return 1
        for (s, c), p in zip(cells, ids):
            self.table[s, c] = p
            self.refs[p] = 1
        return 0

    def fork(self, src, dst):
        n = len(self.lens)
        if any(not 0 <= a < n or not 0 <= b < n for a, b in zip(src, dst)) or len(set(dst)) < len(dst) or \
           set(src) & set(dst) or any(self.lens[b] or (self.table[b] >= 0).any() for b in dst):
            return 3
        part = [i for i, a in enumerate(src) if self.lens[a] % self.page]
        ids = self.free_ids()
        if len(ids) < len(part):
            return 1
        fresh = dict(zip(part, ids))
        for i, (a, b) in enumerate(zip(src, dst)):
            full, rest = divmod(int(self.lens[a]), self.page)
            self.table[b, :full] = self.table[a, :full]
            self.refs[self.table[a, :full]] += 1
            if rest:
                self.table[b, full] = fresh[i]
                self.refs[fresh[i]] = 1
                self.pool[:, fresh[i], :rest] = self.pool[:, self.table[a, full], :rest]
            self.lens[b] = self.lens[a]
        return 0

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = -1
            self.lens[s] = 0

    def compact(self):
        live = int((self.refs > 0).sum())
        old = [p for p in range(live, len(self.refs)) if self.refs[p]]
        new = [p for p in range(live) if not self.refs[p]]
        goes = {a: b for a, b in zip(old, new)}
        self.table = np.vectorize(lambda p: goes.get(p, p))(self.table).astype(np.int32)
        for a, b in goes.items():
            self.pool[:, b] = self.pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        moves = np.full(1 + 2 * len(self.refs), -1, np.int32)
        moves[0] = len(old)
        for i, (a, b) in enumerate(zip(old, new)):
            moves[1 + 2 * i], moves[2 + 2 * i] = a, b
        return moves

    def commit(self, rows, cu, path, count):
        for s, n in enumerate(count):
            for i in range(n):
                pos = int(self.lens[s]) + i
                self.pool[:, self.table[s, pos // self.page], pos % self.page] = rows[:, cu[s] + path[s][i]]
            self.lens[s] += n


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page,planes,row,pages", [(8, 3, 8, 90), (16, 2, 512, 60), (24, 5, 40, 1500), (1, 1, 8, 700)])
def test_page_keeping(built_lib, in_place, page, planes, row, pages):
    """A random history of reserve, commit, fork, free and compact, the state compared after each call;
    in place, or into other arrays (then the inputs must not change). Failing calls change nothing."""
    import torch
    from g4dense_b200 import api
    rng = random.Random(page * 7 + in_place)
    seqs, width = 13, 3 + 120 // page
    plain = Plain(np.random.default_rng(1).integers(0, 2 ** 15, (planes, pages, page, row)).astype(np.int16), seqs, width)
    dev = lambda x: torch.from_numpy(np.array(x, dtype=np.int32)).cuda()  # noqa: E731
    pool = torch.from_numpy(plain.pool.copy()).cuda()
    state = [dev(plain.refs), dev(plain.table), dev(plain.lens)]
    status = dev([-1])
    codes = set()

    def outs():
        return state if in_place else [torch.full_like(t, 77) for t in state]

    def same(what):
        for name, a, b in zip(("refs", "table", "lens"), state, (plain.refs, plain.table, plain.lens)):
            assert np.array_equal(a.cpu().numpy(), b), (what, name)
        assert np.array_equal(pool.cpu().numpy(), plain.pool), what

    for step in range(120):
        what = rng.choice(["grow", "grow", "fork", "free", "compact", "reserve"])
        before = [t.clone() for t in state]
        new = outs()
        if what == "compact":
            moves = dev([0] * (1 + 2 * pages))
            api.pages_compact(pool, state[0], state[1], new[0], new[1], moves)
            new[2] = state[2]
            assert np.array_equal(plain.compact(), moves.cpu().numpy())
        elif what == "free":
            gone = rng.sample(range(seqs), rng.randint(1, 4))
            api.pages_free(*state, dev(gone + gone[:1]), page, *new)
            plain.free(gone)
        elif what == "fork":
            empty = [s for s in range(seqs) if plain.lens[s] == 0]
            src = [rng.randrange(seqs) for _ in range(rng.randint(0, 3))]
            dst = rng.sample(empty, min(len(empty), len(src)))
            src = src[:len(dst)]
            api.pages_fork(pool, *state, dev(src), dev(dst), *new, status)
            code = plain.fork(src, dst)
            codes.add(code)
            assert status.item() == code, (step, src, dst)
        else:
            sizes = [rng.randint(0, 7) for _ in range(seqs)]
            count = [rng.randint(0, n) for n in sizes]
            if what == "reserve":
                count = [c * 9 for c in count] if rng.random() < 0.4 else count
            api.pages_reserve(*state, dev(count), page, new[0], new[1], status)
            code = plain.reserve(count)
            codes.add(code)
            assert status.item() == code, step
            if what == "grow":
                rows = np.random.default_rng(step).integers(0, 2 ** 15, (planes, sum(sizes) + 1, row)).astype(np.int16)
                cu = np.concatenate([[0], np.cumsum(sizes)])
                path = [sorted(rng.sample(range(n), c)) + [-1] * (7 - c) for n, c in zip(sizes, count)]
                api.pages_commit(pool, new[1], state[2], torch.from_numpy(rows).cuda(), dev(cu), dev(path), dev(count),
                                 new[2], status=status)
                if code == 0:
                    plain.commit(rows, cu, path, count)
            else:
                new[2] = state[2]
        if not in_place:
            assert all(torch.equal(a, b) for a, b in zip(before, state))
        state = new
        same((step, what))
    assert 0 in codes


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_reserve_takes_all_or_nothing(built_lib, in_place):
    """Too few free pages, too narrow a table and negative growth leave everything as it was; the last
    free page is found, and entries reserved before are kept."""
    import torch
    from g4dense_b200 import api
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    status = dev([9])

    def reserve(refs, table, lens, grow):
        old = [dev(refs), dev(table)]
        new = old if in_place else [torch.full_like(t, 55) for t in old]
        api.pages_reserve(old[0], old[1], dev(lens), dev(grow), 4, new[0], new[1], status)
        return status.item(), new[0].tolist(), new[1].tolist()
    refs, table, lens = [1, 0, 1, 0, 0], [[2, -1, -1], [0, -1, -1]], [3, 4]
    assert reserve(refs, table, lens, [1, 4]) == (0, [1, 1, 1, 0, 0], [[2, -1, -1], [0, 1, -1]])
    assert reserve(refs, table, lens, [9, 4]) == (0, [1, 1, 1, 1, 1], [[2, 1, 3], [0, 4, -1]])
    assert reserve(refs, table, lens, [9, 8]) == (1, refs, table)
    assert reserve(refs, table, lens, [10, 0]) == (2, refs, table)
    assert reserve(refs, table, lens, [-1, 0]) == (2, refs, table)
    assert reserve(refs, table, [3, -4], [1, 0]) == (2, refs, table)
    early = [[2, -1, 4], [0, -1, -1]]
    assert reserve([1, 0, 1, 0, 1], early, lens, [9, 1]) == (0, [1, 1, 1, 1, 1], [[2, 1, 4], [0, 3, -1]])
    assert reserve(refs, table, lens, [0, 0]) == (0, refs, table)


@pytest.mark.gpu
def test_reserve_many_sequences(built_lib):
    """More sequences and pages than one block has threads."""
    import torch
    from g4dense_b200 import api
    rng = np.random.default_rng(4)
    plain = Plain(np.zeros((1, 20000, 2, 8), np.int16), 4096, 6)
    taken = rng.random(20000) < 0.3
    plain.refs[taken] = 1
    plain.lens[:] = 0
    dev = lambda x: torch.from_numpy(np.array(x, dtype=np.int32)).cuda()  # noqa: E731
    refs, table, lens, status = dev(plain.refs), dev(plain.table), dev(plain.lens), dev([9])
    for grow in (rng.integers(0, 6, 4096), rng.integers(0, 7, 4096), rng.integers(4, 8, 4096)):
        api.pages_reserve(refs, table, lens, dev(grow), 2, refs, table, status)
        assert status.item() == plain.reserve(grow.tolist())
        assert np.array_equal(refs.cpu().numpy(), plain.refs) and np.array_equal(table.cpu().numpy(), plain.table)


@pytest.mark.gpu
def test_fork_refuses_bad_sequences(built_lib):
    import torch
    from g4dense_b200 import api
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.zeros(2, 6, 8, 16, dtype=torch.bfloat16, device="cuda")
    refs, table, lens, status = dev([1, 1, 1, 0, 0, 0]), dev([[0, 1], [2, -1], [-1, -1], [-1, -1]]), dev([12, 3, 0, 0]), dev([9])

    def fork(src, dst, **kw):
        a = dict(refs=refs, table=table, lens=lens) | kw
        out = [torch.full_like(a[n], 5) for n in ("refs", "table", "lens")]
        api.pages_fork(pool, a["refs"], a["table"], a["lens"], dev(src), dev(dst), *out, status)
        if status.item():
            assert all(torch.equal(o, a[n]) for o, n in zip(out, ("refs", "table", "lens")))
        return status.item()
    assert fork([0], [2]) == 0
    assert fork([0, 1], [2, 3]) == 0
    assert fork([0, 1], [2, 2]) == 3
    assert fork([0], [1]) == 3
    assert fork([0], [0]) == 3
    assert fork([4], [2]) == 3
    assert fork([-1], [2]) == 3
    assert fork([0, 2], [2, 3]) == 3
    assert fork([0], [2], table=dev([[0, 99], [2, -1], [-1, -1], [-1, -1]])) == 4
    assert fork([0], [2], lens=dev([40, 3, 0, 0])) == 2
    assert fork([0, 0, 1], [2, 3, 2]) == 3
    assert fork([0], [2], refs=dev([1, 1, 1, 1, 1, 1])) == 1
    with pytest.raises(ValueError, match="refs_out"):
        api.pages_fork(pool, refs, table, lens, dev([0]), dev([2]), refs.long(), table, lens, status)
    with pytest.raises(RuntimeError, match="16 bytes"):
        odd = torch.zeros(2, 6, 8, 9, dtype=torch.bfloat16, device="cuda")
        api.pages_fork(odd, refs, table, lens, dev([0]), dev([2]), refs, table, lens, status)
    with pytest.raises(RuntimeError, match="differ"):
        api.pages_fork(pool[:, :5], refs, table, lens, dev([0]), dev([2]), refs, table, lens, status)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,page,planes", [(8, 1, 1), (4096, 16, 7), (1000, 24, 3), (20000, 8, 2)])
def test_copy_pages(built_lib, rows, page, planes):
    """Copies between pools of different page counts and strides; ids out of range are skipped."""
    import torch
    from g4dense_b200 import api
    a = torch.randint(0, 2 ** 15, (planes, 9, page, rows), dtype=torch.int16, device="cuda")
    wide = torch.zeros(planes, 14, page, rows, dtype=torch.int16, device="cuda")
    b = wide[:, 1:13]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    src, dst = [3, 8, 0, 3, 9, -1, 5], [11, 0, 7, 4, 1, 2, 12]
    want = b.clone()
    for s, d in zip(src, dst):
        if 0 <= s < 9 and 0 <= d < 12:
            want[:, d] = a[:, s]
    api.pages_copy(a, b, dev(src), dev(dst))
    assert torch.equal(b, want) and (wide[:, 0] == 0).all() and (wide[:, 13] == 0).all()
    c = a.clone()
    api.pages_copy(c, c, dev([0, 1]), dev([7, 8]))
    assert torch.equal(c[:, 7], a[:, 0]) and torch.equal(c[:, 8], a[:, 1]) and torch.equal(c[:, :7], a[:, :7])
    api.pages_copy(a, b, dev([]), dev([]))


def test_tree_mask():
    from g4dense_b200 import api
    mask, depth = api.tree_mask([-1, 0, 0, 1, 3, 2])
    assert depth.tolist() == [0, 1, 1, 2, 3, 2]
    assert mask[:, 0].tolist() == [1, 0b11, 0b101, 0b1011, 0b11011, 0b100101]
    mask, depth = api.tree_mask([-1] + list(range(69)), 3)
    assert mask.view(np.uint32)[69].tolist() == [0xFFFFFFFF, 0xFFFFFFFF, 0x3F] and depth[69] == 69
    with pytest.raises(ValueError):
        api.tree_mask([-1, 2, 0])


def test_packed_arguments_match_the_header(tmp_path):
    """The bindings pack argument structs by hand: their sizes and last fields have to be the header's."""
    import ctypes
    import subprocess
    from pathlib import Path

    from g4dense_b200 import api
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "g4dense_b200_ops.h"\n'
                   'int main(void) { printf("%zu %zu %zu %zu %zu %zu", sizeof(g4b_tree_attention_args), '
                   'offsetof(g4b_tree_attention_args, scale), sizeof(g4b_page_pool), offsetof(g4b_page_pool, row_bytes), '
                   'sizeof(g4b_page_tables), offsetof(g4b_page_tables, page_size)); return 0; }\n')
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-I", str(include), str(src), "-o", str(tmp_path / "s")], check=True)
    size = list(map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()))
    import struct
    at = lambda s, f: struct.calcsize(s.format.split("f")[0] if f else s.format) - (0 if f else ctypes.sizeof(ctypes.c_int))  # noqa: E731
    assert size == [api._TREE_ATTENTION.size, at(api._TREE_ATTENTION, True), api._PAGE_POOL.size, at(api._PAGE_POOL, False),
                    api._PAGE_TABLES.size, at(api._PAGE_TABLES, False)]
