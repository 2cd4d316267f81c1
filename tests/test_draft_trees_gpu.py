"""A step that verifies drafted trees on the GPU: each operator against the plain float64 one, and a run of them together."""
import math
import random

import pytest
import torch

import plain_draft_trees as plain
from tffinfer_amd.kernels import ops
from tffinfer_amd.kernels.lib import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def ints(x, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device=DEV)
    return t if shape is None else t.view(shape)


class Cache:
    """A paged cache with the requests' places in pages of any order; all other places hold ``rest``."""

    def __init__(self, lengths, nkv, d, page, dtype, rest=math.nan, seed=0, spare=3):
        rng = random.Random(seed)
        need = [-(-n // page) for n in lengths]
        pool = list(range(sum(need) + spare))
        rng.shuffle(pool)
        self.k = torch.full((len(pool), nkv, page, d), rest, dtype=dtype)
        self.v = torch.full((len(pool), nkv, d, page), rest, dtype=dtype)
        self.table = torch.zeros(len(need), max(1, max(need)), dtype=torch.int32)
        self.keys, self.values, self.page = [], [], page
        for r, n in enumerate(lengths):
            mine = [pool.pop() for _ in range(need[r])]
            self.table[r, :need[r]] = torch.tensor(mine, dtype=torch.int32)
            k, v = torch.randn(n, nkv, d).to(dtype), torch.randn(n, nkv, d).to(dtype)
            self.keys.append(k)
            self.values.append(v)
            for i in range(n):
                self.put(r, i, k[i], v[i])

    def put(self, r, i, k, v):
        p = self.table[r, i // self.page]
        self.k[p, :, i % self.page], self.v[p, :, :, i % self.page] = k, v

    def gpu(self):
        return self.k.to(DEV), self.v.to(DEV), self.table.to(DEV)


def attention_tol(dtype, d, places, out, out_abs, most):
    """|error| of one output element: a score is a sum of d products (each rounded, and the sums of them: (d + 8) half steps of their
    absolute values), which moves its weight by that share, and the denominator's too; the exponential and the sums over the places
    round (places + 16) times; bf16 rounds each weight before the product, and the result (half a step, 2^-8, each)."""
    u = 2.0 ** -24
    t = out_abs * (2 * (d + 8) * u * most + (places + 16) * 2 * u)
    if dtype == BF16:
        t = t + 2.0 ** -8 * out_abs * 1.01 + 2.0 ** -8 * out.abs() * 1.01
    return t + u * out.abs() + 1e-30


def check_attention(nq, nkv, d, page, dtype, starts, trees, window=0, softcap=0.0, sinks=False, sees=None, words=None, rest=math.nan, seed=0, qscale=2.0,
                    poison=None, scale=None, extra=0, before=0):
    """trees: parents by request; sees: the nodes' bits where they are no paths.  ``extra`` rows behind the last node, ``before`` ones before the first."""
    sees = sees or [plain.paths(t) for t in trees]
    cache = Cache([s + len(t) for s, t in zip(starts, sees)], nkv, d, page, dtype, rest, seed)
    if poison is not None:
        poison(cache)
    cu = [before]
    for t in sees:
        cu.append(cu[-1] + len(t))
    words = words or max(1, -(-max(len(t) for t in sees) // 32))
    q = (qscale * torch.randn(cu[-1] + extra, nq * d)).to(dtype)
    bits = plain.packed([[0]] * before + [row for t in sees for row in t] + [[0]] * extra, words)
    sink = torch.randn(nq) if sinks else None
    kc, vc, table = cache.gpu()
    out = torch.full((cu[-1] + extra, nq * d), 7.0, dtype=dtype, device=DEV)
    args = (q.to(DEV), nq, nkv, d, kc, vc, table, ints(cu), ints(starts), bits.to(DEV))
    kw = dict(window=window, softcap=softcap, scale=scale, sinks=None if sink is None else sink.to(DEV))
    got = ops.tree_attention(*args, **kw, out=out)
    assert got.data_ptr() == out.data_ptr()
    got = got.cpu()
    assert bool((got[cu[-1]:] == 7.0).all()) and bool((got[:before] == 7.0).all())
    worst = 0.0
    for r, s in enumerate(starts):
        n = len(sees[r])
        if not n:
            continue
        o, o_abs, most = plain.attention(q[cu[r]:cu[r + 1]].view(n, nq, d), cache.keys[r], cache.values[r], s,
                                         [[j for j in row if j < n] for row in sees[r]], nq, nkv, window, scale, sink, softcap)
        mine = got[cu[r]:cu[r + 1]].double().view(n, nq, d)
        assert torch.equal(torch.isfinite(mine), torch.isfinite(o)), f"request {r}"
        fine = torch.isfinite(o)
        tol = attention_tol(dtype, d, s + n, o, o_abs, most)
        if softcap:
            tol = tol + o_abs * 2 * 64 * 2.0 ** -24 * softcap
        err = ((mine - o).abs() / tol)[fine]
        if err.numel():
            worst = max(worst, float(err.max()))
    assert worst <= 1.0, worst
    if not extra and not before:
        assert torch.equal(ops.tree_attention(*args, **kw).cpu().view(torch.int16 if dtype == BF16 else torch.int32),
                           got.view(torch.int16 if dtype == BF16 else torch.int32))


def some_trees(rng, sizes, depth=6):
    return [plain.random_tree(rng, n, depth) if n else [] for n in sizes]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d, page", [(64, 16), (128, 16), (128, 8), (256, 32), (80, 16), (40, 24), (8, 8), (192, 64), (512, 16)])
def test_attention_head_and_page_sizes(dtype, d, page):
    rng = random.Random(d + page)
    check_attention(4, 2, d, page, dtype, [0, 1, 37, 130], some_trees(rng, [5, 1, 9, 17]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq, nkv", [(1, 1), (8, 8), (8, 1), (5, 1), (40, 8), (14, 2), (17, 1), (64, 2)])
def test_attention_heads(dtype, nq, nkv):
    check_attention(nq, nkv, 64, 16, dtype, [33, 0, 70], some_trees(random.Random(nq), [7, 3, 12]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("start", [0, 1, 7, 8, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 255, 257, 1000, 2049])
def test_attention_one_request_of_any_length(dtype, start):
    check_attention(4, 2, 128, 16, dtype, [start], some_trees(random.Random(start), [11]))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 255, 256])
def test_attention_trees_of_any_size(n):
    check_attention(8, 2, 64, 16, BF16, [45, 3], some_trees(random.Random(n), [n, max(1, n // 3)], 12))
    check_attention(2, 1, 64, 16, F32, [45], some_trees(random.Random(n), [n], 12))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 2, 3, 5, 16, 31, 32, 40, 64, 200])
def test_attention_window(dtype, window):
    rng = random.Random(window)
    check_attention(4, 2, 64, 16, dtype, [0, 3, 64, 150], some_trees(rng, [9, 40, 33, 12], 9), window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("softcap, sinks", [(20.0, False), (0.0, True), (5.0, True)])
def test_attention_cap_and_sinks(dtype, softcap, sinks):
    check_attention(8, 2, 128, 16, dtype, [90, 0, 17], some_trees(random.Random(3), [20, 4, 33]), softcap=softcap, sinks=sinks)
    check_attention(8, 2, 128, 16, dtype, [300], some_trees(random.Random(4), [40]), softcap=softcap, sinks=sinks, window=50)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sinks", [False, True])
def test_attention_rows_that_see_nothing(dtype, sinks):
    """Any bits: none at all, others than a path's, none of the cached places, nodes that the request has not."""
    sees = [[[], [0], [], [1, 2], [0, 40, 63]], [[], [], [0, 1]], [[3], [2, 3], [], [0]]]
    check_attention(4, 2, 64, 16, dtype, [0, 20, 0], None, sees=sees, words=2, sinks=sinks)
    check_attention(4, 2, 64, 16, dtype, [0, 20, 0], None, sees=sees, words=8, sinks=sinks, window=2)


def test_attention_requests_without_nodes_and_rows_behind_the_last():
    for dtype in (BF16, F32):
        check_attention(4, 2, 64, 16, dtype, [5, 90, 0, 31], some_trees(random.Random(1), [0, 6, 0, 3]), extra=4)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_keeps_what_is_not_finite_to_those_who_see_it(dtype, bad):
    """A node's key and value that are not finite reach the nodes that see it, and no others; a cached one before the window likewise."""
    chain_and_leaf = [-1, 0, 0, 1, 1, 2, 2, 5]

    def poison(c):
        for r in range(2):
            c.values[r][-7, 0, 3] = bad       # node 1 of eight
            c.values[r][-2, 1, 5] = bad       # node 6
            if math.isnan(bad):
                c.keys[r][-6, 0, 2] = bad     # node 2
            for i in (-7, -2, -6):
                n = len(c.keys[r]) + i
                c.put(r, n, c.keys[r][n], c.values[r][n])
        c.values[1][4, 0, 9] = bad            # far before the window
        c.put(1, 4, c.keys[1][4], c.values[1][4])
    check_attention(4, 2, 64, 16, dtype, [20, 70], [chain_and_leaf] * 2, window=30, poison=poison)


def test_attention_of_many_requests_of_uneven_lengths():
    rng = random.Random(5)
    starts = [rng.choice((0, 3, 60, 200, 700, 1500)) for _ in range(70)]
    check_attention(2, 1, 64, 16, BF16, starts, some_trees(rng, [rng.randint(1, 9) for _ in starts]))
    check_attention(2, 1, 64, 16, F32, starts[:20], some_trees(rng, [rng.randint(1, 9) for _ in starts[:20]]))


@pytest.mark.parametrize("nq, dtype, n", [(8, BF16, 2), (8, BF16, 40), (4, F32, 3)])
def test_attention_of_a_long_cache(nq, dtype, n):
    """More partial results of a group of columns than a wave has lanes, and pages of many tokens."""
    check_attention(nq, 1, 128, 256, dtype, [20000], some_trees(random.Random(n), [n]))
    check_attention(nq, 1, 64, 16, dtype, [9001], some_trees(random.Random(n), [n]), window=8600, sinks=True)


@pytest.mark.parametrize("d, page", [(64, 64), (128, 128), (256, 8)])
def test_attention_of_many_wide_requests(d, page):
    """More requests than a wave has lanes, of many columns: blocks that begin and end in the middle of a request, and requests without nodes."""
    rng = random.Random(d)
    starts = [rng.choice((0, 3, 60, 200, 700)) for _ in range(70)]
    check_attention(16, 1, d, page, BF16, starts, some_trees(rng, [rng.choice((0, 1, 5, 9)) for _ in starts], 4), window=0 if d == 64 else 90)


def test_attention_of_more_pages_than_a_block_holds_numbers_of():
    """As many kv heads as the GPU has CUs, small pages: a block goes through a whole request of more pages than LDS has room for."""
    nkv, d, page, start, n = 256, 64, 8, 9000, 20
    k, v = torch.randn(40, nkv, page, d).to(BF16), torch.randn(40, nkv, d, page).to(BF16)
    table = torch.randint(0, 40, (1, -(-(start + n) // page)), dtype=torch.int32)
    q = torch.randn(n, 2 * nkv * d).to(BF16)
    see = plain.paths(plain.random_tree(random.Random(1), n, 6))
    got = ops.tree_attention(q.to(DEV), 2 * nkv, nkv, d, k.to(DEV), v.to(DEV), table.to(DEV), ints([0, n]), ints([start]), plain.packed(see, 1).to(DEV))
    got = got.cpu().double().view(n, 2 * nkv, d)
    for g in (0, 101, 255):
        keys, values = k[table[0].long(), g].reshape(-1, 1, d), v[table[0].long(), g].transpose(1, 2).reshape(-1, 1, d)
        heads = slice(2 * g, 2 * g + 2)
        o, o_abs, most = plain.attention(q.view(n, 2 * nkv, d)[:, heads], keys, values, start, see, 2, 1)
        assert bool(((got[:, heads] - o).abs() <= attention_tol(BF16, d, start + n, o, o_abs, most)).all()), g


@pytest.mark.parametrize("nq, d", [(4, 80), (4, 64), (40, 128)])
def test_attention_leaves_rows_that_no_request_has(nq, d):
    """Rows before the first node and behind the last, and nodes for which the ancestors have no bits."""
    check_attention(nq, 2, d, 16, BF16, [5, 90], some_trees(random.Random(1), [6, 3]), extra=4, before=3)
    q, k, v = (torch.randn(s, device=DEV).to(BF16) for s in ((40, nq * d), (4, 2, 16, d), (4, 2, d, 16)))
    out = torch.full((40, nq * d), 7.0, dtype=BF16, device=DEV)
    ops.tree_attention(q, nq, 2, d, k, v, ints([[3, 1, 0, 2]]), ints([0, 40]), ints([9]), torch.ones(40, 1, dtype=torch.int32, device=DEV), out=out)
    assert bool((out[32:] == 7.0).all()) and not bool((out[:32] == 7.0).all(1).any())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nodes, G", [(8, 8), (14, 8), (20, 8), (33, 8), (33, 5), (3, 16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_of_many_columns_keeps_what_is_not_finite_to_those_who_see_it(d, nodes, G, bad):
    """Groups of one to four tiles of columns a wave, whose waves share keys and values: what is not finite lies in the slice of keys that the nodes
    begin in, in the last one, and in a cached place that the window passes for some nodes."""
    rng = random.Random(nodes)
    trees = [plain.random_tree(rng, nodes, 5) for _ in range(2)]
    starts = [20, 100]

    def poison(c):
        for r, s in enumerate(starts):
            for i, g, e in ((s + 1, 0, 3), (s + nodes - 1, 1, 5), (s - 18, 1, d - 1)):
                c.values[r][i, g, e] = bad
            if math.isnan(bad):
                c.keys[r][s + 2, 0, 2] = bad
            for i in (s + 1, s + nodes - 1, s - 18, s + 2):
                c.put(r, i, c.keys[r][i], c.values[r][i])
    check_attention(2 * G, 2, d, 16, BF16, starts, trees, poison=poison)
    check_attention(2 * G, 2, d, 16, BF16, starts, trees, window=20, poison=poison, sinks=True)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nodes", [5, 20, 33])
def test_attention_of_many_columns_under_a_cap_and_with_sinks(d, nodes):
    rng = random.Random(nodes)
    for softcap, sinks, window in ((20.0, False, 0), (0.0, True, 0), (5.0, True, 0), (10.0, True, 40)):
        check_attention(16, 2, d, 16, BF16, [90, 0, 300], some_trees(rng, [nodes, nodes, 3]), window=window, softcap=softcap, sinks=sinks)


@pytest.mark.parametrize("nq, nkv, dtype, sizes", [(40, 8, BF16, (40, 7, 48, 1)), (18, 2, BF16, (60, 64, 57, 64)), (18, 2, F32, (60, 64, 57, 64)),
                                                   (66, 1, BF16, (30, 9, 1, 25))])
def test_attention_whose_merge_takes_four_heads_a_wave(nq, nkv, dtype, sizes):
    """More than 16,384 (node, q head) pairs: a wave merges four heads, which lie in groups of columns of different numbers of partial results, beside heads
    that are not there where nq is no multiple of four."""
    rng = random.Random(nq)
    sizes = [n for _ in range(4 if sum(sizes) > 200 else 5) for n in sizes]
    starts = [rng.choice((0, 40, 130, 300, 700)) for _ in sizes]
    assert sum(sizes) * nq > 16384
    check_attention(nq, nkv, 64, 16, dtype, starts, some_trees(rng, sizes), sinks=nq == 18)


def test_attention_window_of_any_size():
    q, k, v = (torch.randn(s, device=DEV).to(BF16) for s in ((3, 256), (4, 2, 16, 64), (4, 2, 64, 16)))
    args = (q, 4, 2, 64, k, v, ints([[3, 1, 0, 2]]), ints([0, 3]), ints([40]), ints([[1], [3], [5]]))
    every = ops.tree_attention(*args)
    for window in (42, 1 << 31, (1 << 32) + 5):
        assert torch.equal(ops.tree_attention(*args, window=window), every)
    with pytest.raises(KernelError):
        ops.tree_attention(*args, window=-(1 << 32))


def test_attention_of_large_scores():
    """Scores of some hundred: one weight takes all, and the running maximum moves from key to key."""
    for dtype in (BF16, F32):
        check_attention(4, 2, 128, 16, dtype, [500], some_trees(random.Random(8), [13]), qscale=60.0)
        check_attention(4, 2, 128, 16, dtype, [500], some_trees(random.Random(9), [13]), scale=-0.3)


def test_attention_behind_32_bits_of_a_cache():
    """Pages whose elements lie beyond 2^31 and 2^32 bytes, keys and values at the far end of the pool."""
    nkv, page, d = 8, 64, 128
    pages = (5 << 30) // (nkv * page * d * 2)
    k = torch.zeros(pages, nkv, page, d, dtype=BF16, device=DEV)
    v = torch.zeros(pages, nkv, d, page, dtype=BF16, device=DEV)
    small = Cache([70], nkv, d, page, BF16, rest=0.0)
    far = [pages - 1, pages - 2 - (1 << 14)]
    for i, p in enumerate(far):
        k[p], v[p] = small.k[small.table[0, i]].to(DEV), small.v[small.table[0, i]].to(DEV)
    tree = plain.random_tree(random.Random(2), 6, 4)
    q = torch.randn(6, 16 * d).to(BF16)
    got = ops.tree_attention(q.to(DEV), 16, nkv, d, k, v, ints(far, (1, 2)), ints([0, 6]), ints([64]), plain.packed(plain.paths(tree), 1).to(DEV))
    o, o_abs, most = plain.attention(q.view(6, 16, d), small.keys[0], small.values[0], 64, plain.paths(tree), 16, nkv)
    assert bool(((got.cpu().double().view(6, 16, d) - o).abs() <= attention_tol(BF16, d, 70, o, o_abs, most)).all())
    kept = ints([[0, 5, 3]])
    want_k, want_v = small.keys[0][[64, 69, 67]], small.values[0][[64, 69, 67]]
    ops.cache_keep([(k, v)], ints(far, (1, 2)), ints([64]), kept, ints([3]))
    assert torch.equal(k[far[1], :, :3].cpu().transpose(0, 1), want_k) and torch.equal(v[far[1], :, :, :3].cpu().permute(2, 0, 1), want_v)


# ---- options on logits ----

def check_adjust(R, V, lens, prompts, pens, biases=None, masks=None, mask_rows=None, trees=None, in_place=False, logits=None):
    rng = random.Random(V + R)
    rows = R if trees is None else sum(len(t[0]) for t in trees)
    logits = 3 * torch.randn(rows, V) if logits is None else logits
    hist = [[rng.randrange(V) if rng.random() < 0.5 else rng.randrange(min(V, 7)) for _ in range(n)] for n in lens]
    rep, pres, freq = zip(*pens)
    cu = [sum(lens[:i]) for i in range(R + 1)]
    kw = {}
    if biases is not None:
        cub = [sum(len(b) for b in biases[:i]) for i in range(R + 1)]
        flat = [x for b in biases for x in b]
        kw["bias"] = (ints([v for v, _ in flat]), torch.tensor([b for _, b in flat], dtype=F32, device=DEV), ints(cub))
    if mask_rows is not None:
        kw["masks"] = (plain.packed(masks, -(-V // 32)).to(DEV).view(len(masks), -(-V // 32)), ints(mask_rows))
    if trees is not None:
        n = max([1] + [len(t[0]) for t in trees])
        cun = [sum(len(t[0]) for t in trees[:i]) for i in range(R + 1)]
        kw["drafts"] = (ints([x for t in trees for x in t[0]]), ints(cun), plain.packed([s for t in trees for s in t[1]], -(-n // 32)).to(DEV))
    dev = logits.to(DEV)
    before = dev.clone()
    f = lambda x: torch.tensor([float(torch.tensor(y, dtype=F32)) for y in x], dtype=F32, device=DEV)  # noqa: E731
    got = ops.adjust_logits(dev, ints([x for h in hist for x in h]), ints(cu), ints(prompts), f(rep), f(pres), f(freq), out=dev if in_place else None, **kw)
    assert (got.data_ptr() == dev.data_ptr()) == in_place or not dev.numel()
    if not in_place:
        assert torch.equal(dev.nan_to_num(5.0), before.nan_to_num(5.0))
    as32 = lambda x: [float(torch.tensor(y, dtype=F32)) for y in x]  # noqa: E731
    b32 = None if biases is None else [[(v, float(torch.tensor(b, dtype=F32))) for v, b in bs] for bs in biases]
    want, size = plain.adjust(logits, hist, prompts, as32(rep), as32(pres), as32(freq), b32, masks, mask_rows, trees)
    got = got.cpu().double()
    gone = want == -math.inf
    assert torch.equal(got[gone], want[gone])
    same = (size == 0) & ~gone
    assert torch.equal(got[same].nan_to_num(5.0), want[same].nan_to_num(5.0))
    # a product, a quotient or a sum rounds by half a step of what it gives; there are at most six of them, none of whose results is larger
    # than the sum of the absolute values of the terms
    rest = ~same & ~gone & torch.isfinite(want)
    assert bool(((got - want).abs()[rest] <= 6 * 2.0 ** -24 * size[rest] + 1e-37).all())


PENS = [(1.0, 0.0, 0.0), (1.2, 0.0, 0.0), (0.8, 0.5, 0.0), (1.0, 0.0, 0.3), (1.3, -0.7, -0.2), (1.0, 1.5, 0.1)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 97, 1000, 8191, 8192, 8193, 20001])
def test_adjust_penalties(V, in_place):
    lens = [0, 1, 5, 300, 40, 2]
    check_adjust(6, V, lens, [0, 0, 5, 120, 0, 2], PENS, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("V", [1, 33, 1000, 8193, 20001])
def test_adjust_biases_and_masks(V, in_place):
    rng = random.Random(V)
    biases = [[(rng.randrange(V), rng.uniform(-5, 5)) for _ in range(n)] for n in (0, 1, 30, 3, 700, 2)]
    biases[3] = [(0, 1.0), (0, 2.5), (V - 1, -100.0)]                # equal tokens: the last counts
    masks = [[], list(range(V)), [V - 1], sorted(rng.sample(range(V), max(1, V // 3)))]
    check_adjust(6, V, [3, 0, 50, 7, 1, 90], [1, 0, 25, 0, 1, 90], PENS, biases, masks, [0, -1, 3, 1, 2, 99], in_place=in_place)
    check_adjust(6, V, [3, 0, 50, 7, 1, 90], [1, 0, 25, 0, 1, 90], PENS, None, masks, [3, 3, -1, 2, 0, 1], in_place=in_place)
    check_adjust(6, V, [3, 0, 50, 7, 1, 90], [1, 0, 25, 0, 1, 90], [(1.0, 0.0, 0.0)] * 6, biases, in_place=in_place)


@pytest.mark.parametrize("V, n", [(50, 1), (1000, 9), (8193, 40), (300, 100)])
def test_adjust_rows_of_trees(V, n):
    rng = random.Random(n)
    parents = [plain.random_tree(rng, k, 6) for k in (n, max(1, n // 2), n)]
    trees = [([rng.randrange(V) for _ in p], plain.paths(p)) for p in parents]
    trees.insert(1, ([], []))
    rows = sum(len(t[0]) for t in trees)
    masks = [sorted(rng.sample(range(V), V // 2)), []]
    for in_place in (False, True):
        check_adjust(4, V, [20, 0, 3, 0], [10, 0, 0, 0], PENS[2:], None, masks, [rng.randrange(-1, 2) for _ in range(rows)], trees, in_place)
        check_adjust(4, V, [20, 0, 3, 0], [10, 0, 0, 0], PENS[2:], [[(3, 1.0)], [], [(V - 1, -2.0)], []], trees=trees, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R, V", [(40, 60001), (14, 151936)])
def test_adjust_of_many_rows_of_a_real_vocabulary(R, V, in_place):
    """Rows enough for runs of 4,096 logits, that begin anywhere, and a history that a block's threads go through in several turns, from an odd place on."""
    rng = random.Random(V)
    lens = [3, 10001, 0, 1, 4099] + [rng.randint(0, 60) for _ in range(R - 5)]
    prompts = [rng.randint(0, n) for n in lens]
    biases = [[(rng.randrange(V), rng.uniform(-5, 5)) for _ in range(rng.choice((0, 3, 300)))] for _ in lens]
    masks = [list(range(V)), sorted(rng.sample(range(V), V // 50)), sorted(rng.sample(range(V), V - 5)), []]
    pens = [PENS[r % 6] if r != 1 else (1.3, 0.5, 0.25) for r in range(R)]
    check_adjust(R, V, lens, prompts, pens, biases, masks, [rng.randrange(-1, 4) for _ in lens], in_place=in_place)
    check_adjust(R, V, lens, prompts, pens, in_place=in_place)


def test_adjust_of_many_rows_of_trees():
    rng = random.Random(12)
    V, parents = 8193, [plain.random_tree(rng, n, 6) for n in (100, 50, 100)]
    trees = [([rng.randrange(V) if rng.random() < 0.5 else rng.randrange(9) for _ in p], plain.paths(p)) for p in parents]
    masks = [sorted(rng.sample(range(V), V // 2)), []]
    for in_place in (False, True):
        check_adjust(3, V, [20, 5000, 3], [10, 100, 0], PENS[2:5], None, masks, [rng.randrange(-1, 2) for _ in range(250)], trees, in_place)


def test_adjust_leaves_rows_that_no_request_has():
    x, f = torch.randn(7, 3000, device=DEV), torch.full((2,), 2.0, device=DEV)
    tokens, cu, bits = ints([5] * 7), ints([2, 3, 5]), ints([[1]] * 7)
    masks = (torch.zeros(1, 94, dtype=torch.int32, device=DEV), ints([0] * 7))
    got = ops.adjust_logits(x, ints([7, 9]), ints([0, 1, 2]), ints([1, 0]), f, f, f, masks=masks, drafts=(tokens, cu, bits))
    assert torch.equal(got[:2], x[:2]) and torch.equal(got[5:], x[5:]) and bool((got[2:5] == -math.inf).all())


def test_adjust_values_that_are_not_finite():
    V = 700
    x = torch.randn(3, V)
    x[:, ::5], x[:, 1::5], x[:, 2::5] = math.inf, -math.inf, math.nan
    masks = [list(range(0, V, 2)), []]
    for in_place in (False, True):
        check_adjust(3, V, [0, 0, 0], [0, 0, 0], PENS[1:4], None, masks, [0, 1, -1], in_place=in_place, logits=x.clone())


def test_adjust_repetition_gives_the_bits_of_the_penalty_alone():
    R, V = 5, 4099
    rng = random.Random(1)
    hist = [[rng.randrange(V) for _ in range(n)] for n in (0, 1, 64, 500, 9)]
    x = torch.randn(R, V, device=DEV)
    pen = torch.tensor([1.1, 1.3, 0.7, 1.05, 1.0], device=DEV)
    zero = torch.zeros(R, device=DEV)
    sets = [sorted(set(h)) for h in hist]
    old = x.clone()
    ops.repetition_penalty(old, ints([v for s in sets for v in s]), ints([sum(map(len, sets[:i])) for i in range(R + 1)]), pen)
    new = ops.adjust_logits(x, ints([v for h in hist for v in h]), ints([sum(map(len, hist[:i])) for i in range(R + 1)]), ints([len(h) // 2 for h in hist]),
                            pen, zero, zero)
    assert torch.equal(old, new)


def test_adjust_tokens_and_tables_outside():
    """Token ids outside the vocabulary and bounds outside the history are passed over, not followed."""
    x = torch.randn(2, 50, device=DEV)
    one, half = torch.ones(2, device=DEV), torch.full((2,), 0.5, device=DEV)
    got = ops.adjust_logits(x, ints([3, -1, 50, 1 << 30, -(1 << 31), 3]), ints([-5, 4, 1000]), ints([-3, 1 << 30]), one * 2, half, half,
                            bias=(ints([50, -1, 7]), torch.ones(3, device=DEV), ints([0, 3, 99])))
    want = x.clone()
    want[0, 3] = (x[0, 3] / 2 if x[0, 3] > 0 else x[0, 3] * 2) - 0.5 - 0.5
    want[0, 7] += 1
    want[1, 3] = x[1, 3] / 2 if x[1, 3] > 0 else x[1, 3] * 2
    assert torch.equal(got, want)


# ---- the walk and the move ----

@pytest.mark.parametrize("sizes, max_path", [([1], 1), ([8], 4), ([5, 0, 64, 1, 33], 8), ([256, 255, 100], 256), ([20] * 70, 6), ([40], 1), ([0], 3)])
def test_accept(sizes, max_path):
    rng = random.Random(sum(sizes) + max_path)
    trees = [plain.random_tree(rng, n, 40) if n else [] for n in sizes]
    tokens = [[rng.randrange(4) for _ in t] for t in trees]          # (children of one token are frequent: the first counts)
    choices = [[rng.randrange(4) for _ in t] for t in trees]
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    flat = lambda x: ints([v for s in x for v in s])  # noqa: E731
    bits = plain.packed([p for t in trees for p in plain.paths(t)], max(1, -(-max(sizes) // 32))).to(DEV)
    path, counts, following = ops.tree_accept(flat(choices), flat(tokens), ints(cu), bits, max_path)
    want = plain.accept(choices, tokens, trees, max_path)
    assert path.tolist() == [w[0] for w in want]
    assert counts.tolist() == [w[1] for w in want] and following.tolist() == [w[2] for w in want]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d, page, nkv, layers", [(128, 16, 8, 2), (64, 8, 1, 3), (40, 24, 3, 1), (512, 16, 2, 1), (7, 5, 2, 66)])
def test_keep(dtype, d, page, nkv, layers):
    """Any path: rising, falling, with places that are both sources and targets, the same source twice, none at all; nothing else moves."""
    starts = [0, 13, 50, 7, 3]
    paths = [[0, 2, 5, 6], [0, 1, 2, 3], [3, 0, 1, 2], [0, 7, 7, -1], [5, 4, 3, 2]]
    counts = [4, 4, 4, 3, 0]
    caches = [Cache([s + 9 for s in starts], nkv, d, page, dtype, rest=3.0, seed=5) for _ in range(layers)]
    on_gpu = [c.gpu() for c in caches]
    assert all(torch.equal(c.table, caches[0].table) for c in caches)
    ops.cache_keep([(k, v) for k, v, _ in on_gpu], on_gpu[0][2], ints(starts), ints(paths), ints(counts))
    for c, (k, v, _) in zip(caches, on_gpu):
        for r, s in enumerate(starts):
            for i in range(counts[r]):
                if paths[r][i] >= 0:
                    c.put(r, s + i, c.keys[r][s + paths[r][i]], c.values[r][s + paths[r][i]])
        assert torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v)


def test_keep_long_paths():
    rng = random.Random(4)
    for dtype, n, d in ((BF16, 256, 128), (F32, 256, 64), (BF16, 100, 256)):
        path = rng.sample(range(n + 20), n)
        c = Cache([31 + n + 20], 2, d, 16, dtype, rest=0.0)
        k, v, table = c.gpu()
        ops.cache_keep([(k, v)], table, ints([31]), ints([path]), ints([n]))
        for i, p in enumerate(path):
            c.put(0, 31 + i, c.keys[0][31 + p], c.values[0][31 + p])
        assert torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v)


def test_keep_places_outside_the_table_are_passed_over():
    c = Cache([40], 2, 64, 16, BF16, rest=1.0)
    k, v, table = c.gpu()
    table[0, 2] = 1 << 20                                            # no page of the pool
    ops.cache_keep([(k, v)], table, ints([20]), ints([[3, 1 << 30, 17, -7, 1]]), ints([1000]))
    c.put(0, 20, c.keys[0][23], c.values[0][23])
    c.put(0, 24, c.keys[0][21], c.values[0][21])
    assert torch.equal(k.cpu(), c.k) and torch.equal(v.cpu(), c.v)


# ---- refusals ----

def test_refusals():
    q, i1 = torch.zeros(3, 128, dtype=BF16, device=DEV), ints([0, 3])
    k, v = torch.zeros(4, 2, 16, 32, dtype=BF16, device=DEV), torch.zeros(4, 2, 32, 16, dtype=BF16, device=DEV)
    table, start, bits = ints([[0, 1]]), ints([5]), ints([[1], [3], [5]])
    good = (q, 4, 2, 32, k, v, table, i1, start, bits)
    ops.tree_attention(*good)

    def attention(**kw):
        names = ("q", "nq", "nkv", "d", "k", "v", "table", "cu", "start", "bits")
        ops.tree_attention(*[kw.pop(n, x) for n, x in zip(names, good)], **kw)
    for bad in (dict(q=q[:, :100]), dict(q=q.float()), dict(q=q.t()), dict(k=v), dict(v=v.float()), dict(table=table.long()), dict(table=ints([[0, 1]] * 2)),
                dict(cu=ints([0, 3, 3])), dict(bits=ints([1, 3, 5])), dict(bits=bits[:2]), dict(bits=torch.zeros(3, 9, dtype=torch.int32, device=DEV)),
                dict(bits=bits.long()), dict(start=start.cpu()), dict(sinks=torch.zeros(3, device=DEV)), dict(window=-1), dict(softcap=-2.0),
                dict(out=torch.zeros(3, 64, dtype=BF16, device=DEV)), dict(out=q), dict(q=torch.zeros(3, 96, dtype=BF16, device=DEV), nq=3)):
        with pytest.raises(KernelError):
            attention(**bad)
    x, f = torch.zeros(2, 40, device=DEV), torch.ones(2, device=DEV)
    h, cu, p = ints([1, 2, 3]), ints([0, 1, 3]), ints([0, 0])
    good_a = (x, h, cu, p, f, f, f)
    ops.adjust_logits(*good_a)
    room = torch.zeros(5, 40, device=DEV)
    for args, kw in (((x.bfloat16(),) + good_a[1:], {}), ((x[:, ::2],) + good_a[1:], {}), ((x[:1],) + good_a[1:], {}), ((x, h.long()) + good_a[2:], {}),
                     ((x, h, cu[:2]) + good_a[3:], {}), (good_a, dict(masks=(ints([[1]]), ints([0, 0])))), (good_a, dict(masks=(ints([[1, 1]]), ints([0])))),
                     (good_a, dict(bias=(ints([1]), torch.zeros(2, device=DEV), ints([0, 0, 1])))), (good_a, dict(bias=(ints([1]), f[:1], ints([0, 1])))),
                     (good_a, dict(drafts=(ints([1, 2]), ints([0, 2]), ints([[1], [1]])))), (good_a, dict(drafts=(ints([1, 2]), ints([0, 1, 2]), ints([[1]])))),
                     (good_a, dict(out=torch.zeros(2, 41, device=DEV))), ((room[:2],) + good_a[1:], dict(out=room[1:3]))):
        with pytest.raises(KernelError):
            ops.adjust_logits(*args, **kw)
    t = ints([1, 2, 3])
    for args in ((t, t[:2], i1, bits, 4), (t, t, i1, bits, 0), (t, t, i1, bits, 257), (t, t, i1[:0], bits, 3), (t.long(), t, i1, bits, 3), (t, t, i1, bits[:2], 3)):
        with pytest.raises(KernelError):
            ops.tree_accept(*args)
    path, n = ints([[0, 2]]), ints([2])
    both = torch.zeros(6, 2, 16, 32, dtype=BF16, device=DEV)
    for args in (([(both[:4], v), (both[2:], v.clone())], table, start, path, n), ([(k, k)], table, start, path, n), ([(k, v), (k, v)], table, start, path, n), ([(k, v), (k.float(), v.float())], table, start, path, n),
                 ([(k, v)], table, start, path[0], n), ([(k, v)], table, start, path, ints([1, 2])), ([(k, v)], ints([[0], [1]]), start, path, n),
                 ([(k, v)], table, start, torch.zeros(1, 257, dtype=torch.int32, device=DEV), n), ([(k.cpu(), v.cpu())], table, start, path, n)):
        with pytest.raises(KernelError):
            ops.cache_keep(*args)
    ops.cache_keep([], table, start, path, n)


def test_empty_calls():
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    k, v = torch.zeros(4, 2, 16, 32, dtype=BF16, device=DEV), torch.zeros(4, 2, 32, 16, dtype=BF16, device=DEV)
    assert ops.tree_attention(torch.zeros(0, 128, dtype=BF16, device=DEV), 4, 2, 32, k, v, e.view(0, 1), ints([0]), e, e.view(0, 1)).shape == (0, 128)
    f = torch.zeros(0, device=DEV)
    assert ops.adjust_logits(torch.zeros(0, 9, device=DEV), e, ints([0]), e, f, f, f).shape == (0, 9)
    path, counts, following = ops.tree_accept(e, e, ints([0, 0, 0]), e.view(0, 1), 3)
    assert path.tolist() == [[-1] * 3] * 2 and counts.tolist() == [0, 0] and following.tolist() == [-1, -1]
    ops.cache_keep([(k, v)], e.view(0, 2), e, e.view(0, 3), e)


# ---- together ----

class Step:
    """A toy decoder of one attention layer that verifies trees: embeddings as queries, keys and values (rotated by position), its output
    against the embeddings as logits."""

    def __init__(self, dtype=BF16, nq=4, nkv=2, d=64, V=300, page=16, seed=3):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.nq, self.nkv, self.d, self.V, self.page = dtype, nq, nkv, d, V, page
        self.qkv = torch.randn(V, (nq + 2 * nkv) * d, generator=g).to(dtype).to(DEV)
        self.head = torch.randn(V, nq * d, generator=g).to(DEV)
        angle = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))
        self.cos_sin = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous().to(DEV)

    def store(self, tokens, positions, slots, k, v):
        """Their keys and values to the pages; the rows with finished queries."""
        rows = self.qkv[tokens.long()].contiguous()
        ops.qk_norm_rope_kv(rows, self.nq, self.nkv, self.d, None, None, 1e-6, self.cos_sin, 0, positions, slots, k, v)
        return rows


def test_a_step_of_trees_agrees_with_decoding_token_by_token():
    """Three requests decode greedily under penalties, a bias and a grammar, token by token; then the same by steps that verify trees: the
    tokens agree, and so do the cache's kept places.  In float32: a weighted mean of numbers up to 4 is off by some 1e-5 whatever the order
    of its terms (70 places, 2^-23 each, at most), a logit, 256 of them times 0.05 and numbers of mean size 0.8, by 1e-4 at most; the
    best two candidates are ten times further apart (checked)."""
    s = Step(dtype=F32)
    rng = random.Random(2)
    page, R, steps = s.page, 3, 12
    prompts = [[rng.randrange(s.V) for _ in range(n)] for n in (5, 30, 17)]
    pens = dict(repetition=torch.tensor([1.1, 1.0, 1.2], device=DEV), presence=torch.tensor([0.0, 3.0, 0.5], device=DEV),
                frequency=torch.tensor([0.5, 0.0, 0.7], device=DEV))
    bias = (ints([7, 9, 7]), torch.tensor([4.0, -3.0, 2.0], device=DEV), ints([0, 2, 2, 3]))
    masks = plain.packed([list(range(0, s.V, 2)), list(range(s.V))], -(-s.V // 32)).to(DEV)
    width = 8
    table = ints(rng.sample(range(R * width), R * width), (R, width))

    def new_cache():
        return (torch.zeros(R * width, s.nkv, page, s.d, dtype=s.dtype, device=DEV), torch.zeros(R * width, s.nkv, s.d, page, dtype=s.dtype, device=DEV))

    def slots(places):
        return ints([int(table[r, p // page]) * page + p % page for r, p in places])

    def logits_of(k, v, seqs, cached, trees, tokens):
        """One step of trees (parents) behind the cached tokens, adjusted."""
        sees = [plain.paths(t) for t in trees]
        cu = [0]
        for t in trees:
            cu.append(cu[-1] + len(t))
        bits = plain.packed([x for t in sees for x in t], 1).to(DEV)
        at = [(r, cached[r] + i) for r, t in enumerate(trees) for i in range(len(t))]
        pos = ints([cached[r] + len(p) - 1 for r, t in enumerate(sees) for p in t])
        flat = ints([x for t in tokens for x in t])
        rows = s.store(flat, pos, slots(at), k, v)
        o = ops.tree_attention(rows[:, :s.nq * s.d].contiguous(), s.nq, s.nkv, s.d, k, v, table, ints(cu), ints(cached), bits)
        x = o.float() @ s.head.T * 0.05
        hist = [q[:c] for q, c in zip(seqs, cached)]
        cuh = [sum(map(len, hist[:i])) for i in range(R + 1)]
        rows_mask = ints([(0 if r == 2 else -1) for r, _ in at])
        ops.adjust_logits(x, ints([a for h in hist for a in h]), ints(cuh), ints([min(len(p), c) for p, c in zip(prompts, cached)]), **pens, bias=bias,
                          masks=(masks, rows_mask), drafts=(flat, ints(cu), bits), out=x)
        return x, flat, ints(cu), bits

    def fill(k, v):
        for r, p in enumerate(prompts):
            n = len(p) - 1
            s.store(ints(p[:n]), ints(list(range(n))), slots([(r, i) for i in range(n)]), k, v)
        return [len(p) - 1 for p in prompts]

    # token by token: trees of one node
    k, v = new_cache()
    cached = fill(k, v)
    one = [list(p) for p in prompts]
    for _ in range(steps):
        x = logits_of(k, v, one, cached, [[-1]] * R, [[q[-1]] for q in one])[0]
        top = x.topk(2, dim=1).values
        assert bool((top[:, 0] - top[:, 1] > 1e-3).all())
        for r, t in enumerate(ops.argmax(x).tolist()):
            one[r].append(t)
            cached[r] += 1
    # by trees: guesses from the answer, some wrong
    k2, v2 = new_cache()
    cached2 = fill(k2, v2)
    many, taken = [list(p) for p in prompts], []
    while min(len(q) - len(p) for q, p in zip(many, prompts)) < steps:
        trees, tokens = [], []
        for r in range(R):
            n, m = rng.randint(1, 14), len(many[r])
            t = plain.random_tree(rng, n, 5)
            depth = [len(p) - 1 for p in plain.paths(t)]
            right = one[r][m - 1:] + [0] * 8
            trees.append(t)
            tokens.append([right[depth[i]] if i == 0 or rng.random() < 0.6 else rng.randrange(s.V) for i in range(n)])
        x, flat, cu, bits = logits_of(k2, v2, many, cached2, trees, tokens)
        choices = ops.argmax(x)
        path, counts, following = ops.tree_accept(choices, flat, cu, bits, 6)
        ops.cache_keep([(k2, v2)], table, ints(cached2), path, counts)
        for r in range(R):
            kept = path[r, :int(counts[r])].tolist()
            many[r] += [tokens[r][i] for i in kept[1:]] + [int(following[r])]
            cached2[r] += len(kept)
            taken.append(len(kept))
    assert max(taken) > 2 and min(taken) == 1
    for r in range(R):
        m = min(len(many[r]), len(one[r]))
        assert many[r][:m] == one[r][:m]
        for p in range(min(cached[r], cached2[r])):
            a, b = int(table[r, p // page]), p % page
            assert torch.equal(k[a, :, b], k2[a, :, b]) and torch.equal(v[a, :, :, b], v2[a, :, :, b])


def test_captured_and_on_another_stream():
    """The four together in a captured graph: every replay on new inputs gives the eager bits, with eager work between; and on a side stream."""
    rng = random.Random(6)
    R, V, nq, nkv, d, page = 3, 5000, 8, 2, 128, 16
    starts = [40, 700, 9]
    trees = some_trees(rng, [12, 20, 1])
    c = Cache([s + len(t) for s, t in zip(starts, trees)], nkv, d, page, BF16, rest=0.0)
    k, v, table = c.gpu()
    cu = ints([0, 12, 32, 33])
    bits = plain.packed([p for t in trees for p in plain.paths(t)], 1).to(DEV)
    q = torch.randn(33, nq * d, device=DEV).to(BF16)
    logits = torch.randn(33, V, device=DEV)
    tokens = ints([rng.randrange(6) for _ in range(33)])
    hist, cuh, prompt = ints([rng.randrange(20) for _ in range(60)]), ints([0, 10, 50, 60]), ints([5, 10, 0])
    pen = torch.tensor([1.2, 1.0, 1.5], device=DEV)
    masks = (plain.packed([[0, 1, 2, 3, 4, 5]], -(-V // 32)).to(DEV), ints([0] * 33))

    def together(k, v):
        o = ops.tree_attention(q, nq, nkv, d, k, v, table, cu, ints_start, bits)
        x = ops.adjust_logits(logits, hist, cuh, prompt, pen, pen, pen, masks=masks, drafts=(tokens, cu, bits))
        choices = ops.argmax(x)
        path, counts, following = ops.tree_accept(choices, tokens, cu, bits, 5)
        ops.cache_keep([(k, v)], table, ints_start, path, counts)
        return o, x, path, counts, following

    ints_start = ints(starts)
    gk, gv = k.clone(), v.clone()
    together(gk, gv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = k.clone(), v.clone()
        first = [x.clone() for x in together(a, b)]
    torch.cuda.current_stream().wait_stream(side)
    ek, ev = k.clone(), v.clone()
    for x, y in zip(first, together(ek, ev)):
        assert torch.equal(x, y)
    assert torch.equal(a, ek) and torch.equal(b, ev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = together(gk, gv)
    for i in range(4):
        q.copy_(torch.randn(33, nq * d, device=DEV).to(BF16))
        logits.copy_(torch.randn(33, V, device=DEV))
        tokens.copy_(ints([rng.randrange(6) for _ in range(33)]))
        ints_start.copy_(ints([40 - i, 700 - 90 * i, 9 - i]))
        gk.copy_(k)
        gv.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        ek, ev = k.clone(), v.clone()
        for x, y in zip(held, together(ek, ev)):
            assert torch.equal(x, y), i
        assert torch.equal(gk, ek) and torch.equal(gv, ev)


def test_two_streams_at_once():
    """Calls of one shape on two streams, in flight together, give what they give one after the other."""
    rng = random.Random(8)
    trees, starts, nq, nkv, d, page = some_trees(rng, [30, 9, 12]), [3000, 50, 900], 16, 2, 128, 16
    cu, bits = ints([0, 30, 39, 51]), plain.packed([p for t in trees for p in plain.paths(t)], 1).to(DEV)
    sides = []
    for seed in range(2):
        k, v, table = Cache([s + len(t) for s, t in zip(starts, trees)], nkv, d, page, BF16, 0.0, seed).gpu()
        q, x = torch.randn(51, nq * d, device=DEV).to(BF16), torch.randn(51, 20000, device=DEV)
        hist = ints([rng.randrange(20000) for _ in range(4000)])
        sides.append((q, k, v, table, x, hist))
    pen, three, cuh = torch.full((3,), 1.3, device=DEV), ints(starts), ints([0, 3000, 3050, 3950])

    def step(q, k, v, table, x, hist):
        o = ops.tree_attention(q, nq, nkv, d, k, v, table, cu, three, bits)
        y = ops.adjust_logits(x, hist, cuh, three, pen, pen, pen, drafts=(hist[:51].contiguous(), cu, bits))
        return o, y, *ops.tree_accept(ops.argmax(y), hist[:51].contiguous(), cu, bits, 5)
    alone = [step(*s) for s in sides]
    streams = [torch.cuda.Stream() for _ in sides]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sides[i]))
    torch.cuda.synchronize()
    for i, want in enumerate(alone):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want))


# ---- sinks that are not finite ----

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq, d", [(4, 64), (4, 80), (40, 128)])
def test_attention_sinks_of_any_size(dtype, nq, d):
    """A sink of -inf is none, one of +inf takes all the weight; where a node sees nothing the result is zeros whatever the sink, a NaN among them."""
    n, starts, nkv, page = 5, [0, 40], 2, 16
    k, v = (torch.randn(s, device=DEV).to(dtype) for s in ((8, nkv, page, d), (8, nkv, d, page)))
    q, table, cu = torch.randn(2 * n, nq * d, device=DEV).to(dtype), ints(list(range(8)), (2, 4)), ints([0, n, 2 * n])
    see = plain.packed([[], [0], [1, 2], [], [4]] * 2, 1).to(DEV)
    args = (q, nq, nkv, d, k, v, table, cu, ints(starts), see)
    none = ops.tree_attention(*args)
    sinks = torch.full((nq,), -math.inf, device=DEV)
    got = ops.tree_attention(*args, sinks=sinks)
    assert bool((got[[0, 3]] == 0).all()) and torch.equal(got, none)
    for x in (math.inf, math.nan, 1e30, -1e30):
        got = ops.tree_attention(*args, sinks=torch.full((nq,), x, device=DEV))
        assert bool((got[[0, 3]] == 0).all())
        rest = torch.tensor([1, 2, 4, 5, 6, 7, 8, 9], device=DEV)
        assert bool(torch.isnan(got[rest]).all()) if math.isnan(x) else bool((got[rest] == (0 if x > 0 else none[rest])).all())


# ---- alignment ----

@pytest.mark.parametrize("what", ["out", "q", "k", "v"])
@pytest.mark.parametrize("nodes", [5, 30])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_tensors_that_begin_anywhere(what, nodes, dtype):
    """An operand that begins at a multiple of its elements' size and no other is as good as any, and what lies before and behind the output stays."""
    rng = random.Random(nodes)
    nq, nkv, d, page, start = 8, 2, 64, 16, 70
    c = Cache([start + nodes], nkv, d, page, dtype, 0.0)
    t = dict(zip(("k", "v", "table"), c.gpu()))
    t["q"] = torch.randn(nodes, nq * d, device=DEV).to(dtype)
    t["out"] = torch.full((nodes, nq * d), 7.0, device=DEV, dtype=dtype)
    room = torch.full((t[what].numel() + 2,), 7.0, device=DEV, dtype=dtype)
    assert room.data_ptr() % 16 == 0
    room[1:-1] = t[what].flatten()
    t[what] = room[1:-1].view(t[what].shape)
    see = plain.paths(plain.random_tree(rng, nodes, 6))
    got = ops.tree_attention(t["q"], nq, nkv, d, t["k"], t["v"], t["table"], ints([0, nodes]), ints([start]), plain.packed(see, 1).to(DEV), out=t["out"])
    assert got.data_ptr() == t["out"].data_ptr() and bool((room[[0, -1]] == 7.0).all())
    o, o_abs, most = plain.attention(t["q"].cpu().view(nodes, nq, d), c.keys[0], c.values[0], start, see, nq, nkv)
    assert bool(((got.cpu().double().view(nodes, nq, d) - o).abs() <= attention_tol(dtype, d, start + nodes, o, o_abs, most)).all())


# ---- the weights' sum ----

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq, d, nodes", [(4, 64, 5), (4, 128, 7), (8, 256, 3), (8, 64, 7), (16, 64, 30), (8, 128, 20), (16, 256, 12), (4, 80, 5)])
def test_attention_of_equal_values_is_the_value(nq, d, nodes, dtype):
    """Where all values of a head are one, so is the result, whatever the weights: their sum is that of the weights as the product has them, some of them
    most of it.  In float32 product and sum go over up to 100 places, half a step of 2^-24 for each term and a few for the quotient; that is far from
    half a step of bfloat16, where the result has the value's own bits."""
    rng = random.Random(d)
    for start in (0, 1, 9, 70):
        c = Cache([start + nodes], 2, d, 16, dtype, 0.0, seed=start)
        k, v, table = c.gpu()
        v.copy_(torch.randn(2, d, device=DEV)[None, :, :, None].to(dtype).expand_as(v))
        q = (3 * torch.randn(nodes, nq * d, device=DEV)).to(dtype)
        see = plain.packed(plain.paths(plain.random_tree(rng, nodes, 6)), 1).to(DEV)
        got = ops.tree_attention(q, nq, 2, d, k, v, table, ints([0, nodes]), ints([start]), see).view(nodes, 2, nq // 2, d)
        want = v[0, :, :, 0][None, :, None].expand_as(got)
        if dtype == BF16:
            assert torch.equal(got, want), start
        else:
            assert bool(((got - want).abs() <= 2 * (start + nodes + 8) * 2.0 ** -24 * want.abs()).all()), start


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq, d, nodes", [(4, 64, 5), (4, 128, 7), (8, 256, 3), (16, 64, 30), (8, 128, 20), (4, 80, 5)])
def test_attention_of_a_place_that_takes_most_of_the_weight(nq, d, nodes, dtype):
    """A late place whose score is ahead of all before it, by less than a running maximum follows: its weight is some hundred, and rounds.  All values of a
    head are one, which the result is, too, bound as above (2 * 160 half steps)."""
    start, scores = 135, [-40.0] * 160
    for seed in range(6):
        rng = random.Random(seed)
        for place in (5, 40, 70, 100):
            scores[place] = 0.0
        scores[130] = rng.uniform(4.0, 4.5)
        k = torch.zeros(20, 2, 16, d, dtype=dtype)                   # (two tables' worth; the request has the first ten pages)
        k[:10, :, :, 0] = torch.tensor(scores).view(10, 1, 16).to(dtype)
        v = torch.randn(2, d).to(dtype)[None, :, :, None].expand(20, 2, d, 16).contiguous()
        q = torch.zeros(nodes, nq, d, dtype=dtype)
        q[:, :, 0] = (1.0 + 0.2 * torch.rand(nodes, nq)).to(dtype)
        see = plain.packed(plain.paths(plain.random_tree(rng, nodes, 6)), 1).to(DEV)
        got = ops.tree_attention(q.to(DEV).view(nodes, nq * d), nq, 2, d, k.to(DEV), v.to(DEV), ints(list(range(10)), (1, 10)), ints([0, nodes]),
                                 ints([start]), see, scale=1.0).cpu().view(nodes, 2, nq // 2, d)
        want = v[0, :, :, 0][None, :, None].expand_as(got)
        if dtype == BF16:
            assert torch.equal(got, want), seed
        else:
            assert bool(((got - want).abs() <= 2 * 160 * 2.0 ** -24 * want.abs()).all()), seed


# ---- a cap far above the scores ----

@pytest.mark.parametrize("d", [64, 128, 256, 80])
@pytest.mark.parametrize("softcap", [1.0, 50.0, 3e4])
def test_attention_in_float32_holds_a_capped_score_by_its_own_size(d, softcap):
    """c tanh(s / c) is off by some steps of the score, however large c is: a product, a quotient, tanh (two units in the last place, four half steps)
    and two products more, 8 half steps of the largest |score| together, beside those of the score itself."""
    n, nq, start = 9, 4, 60
    see = plain.paths(plain.random_tree(random.Random(d), n, 5))
    c = Cache([start + n], 2, d, 16, F32, 0.0, seed=d)
    k, v, table = c.gpu()
    q = torch.randn(n, nq * d)
    got = ops.tree_attention(q.to(DEV), nq, 2, d, k, v, table, ints([0, n]), ints([start]), plain.packed(see, 1).to(DEV), softcap=softcap)
    o, o_abs, most = plain.attention(q.view(n, nq, d), c.keys[0], c.values[0], start, see, nq, 2, softcap=softcap)
    tol = attention_tol(F32, d, start + n, o, o_abs, most) + o_abs * 2 * 8 * 2.0 ** -24 * most
    assert bool(((got.cpu().double().view(n, nq, d) - o).abs() <= tol).all())


# ---- node 0 and the history ----

@pytest.mark.parametrize("V", [30, 5000])
def test_adjust_rows_of_trees_are_rows_of_requests_that_have_their_path(V):
    """What a request gets that has a node's path at its end, prompt and output in full and without a word of trees, the node's row gets: the same counts, so
    the same bits.  Node 0 is the last token of a prompt of one token, of longer prompts, and of an output."""
    rng = random.Random(V)
    word = lambda: rng.randrange(min(V, 12))  # noqa: E731
    cases = [(1, 0), (7, 0), (7, 1), (300, 40), (5, 9)]              # tokens of the prompt, of the output
    have = [[word() for _ in range(p + o)] for p, o in cases]
    trees = some_trees(rng, [6, 11, 1, 20, 33])
    tokens = [h[-1:] + [word() for _ in t[1:]] for h, t in zip(have, trees)]
    sees = [plain.paths(t) for t in trees]
    rows = [(r, [tokens[r][j] for j in see]) for r, s in enumerate(sees) for see in s]
    x = 3 * torch.randn(len(rows), V, device=DEV)
    rep, pres, freq = ([rng.uniform(0.7, 1.6) for _ in cases], [rng.uniform(-1, 2) for _ in cases], [rng.uniform(-0.5, 1) for _ in cases])
    bias = [[(word(), rng.uniform(-3, 3)) for _ in range(3)] for _ in cases]
    f32 = lambda a: torch.tensor(a, dtype=F32, device=DEV)  # noqa: E731

    def cu(lists):
        return ints([sum(map(len, lists[:i])) for i in range(len(lists) + 1)])

    def flat(lists):
        return ints([y for s in lists for y in s])

    def biases(lists):
        return flat([[t for t, _ in s] for s in lists]), f32([b for s in lists for _, b in s]), cu(lists)
    hist = [h[:-1] for h in have]
    got = ops.adjust_logits(x, flat(hist), cu(hist), ints([p for p, _ in cases]), f32(rep), f32(pres), f32(freq), bias=biases(bias),
                            drafts=(flat(tokens), cu(tokens), plain.packed([see for s in sees for see in s], 2).to(DEV)))
    full = [hist[r] + path for r, path in rows]
    each = lambda a: [a[r] for r, _ in rows]  # noqa: E731
    want = ops.adjust_logits(x, flat(full), cu(full), ints([cases[r][0] for r, _ in rows]), f32(each(rep)), f32(each(pres)), f32(each(freq)),
                             bias=biases(each(bias)))
    assert torch.equal(got, want)
