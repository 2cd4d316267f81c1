"""The operators around a step that verifies drafted tokens, as they are measured: attention of a tree of drafted tokens over the paged
cache, what a request's options do to its logits, the walk that keeps the drafted tokens the model agrees with, and the move of their keys
and values to the places they have from then on.

A request brings a tree of ``n`` tokens to a step: node 0 is the last token it already has, the others are guesses, a node's parent always
before it.  ``ancestors`` int32 [nodes of all requests, words] holds a bit per node of the same request: bit j of node i's row says that i
sees j (its ancestors and itself).  Keys and values of node i lie in the request's pages at place ``start_pos + i``.

With ``own`` false, ``run`` computes an operator from its definition by elementary operations in 32 bits; with ``own`` true it makes the
framework's calls.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
VOCAB = 151936
HEADS = {"0.6b": (16, 8), "8b": (32, 8), "14b": (40, 8), "32b": (64, 8)}    # query and kv heads


# ---- the cases ------------------------------------------------------------------------------------------------------

def _attention(name, heads, batch, tokens, nodes, spread=1, d=128, page=16, window=0, softcap=0.0, sinks=False, dtype="bfloat16"):
    return dict(name=name, op="tree_attention", heads=heads, batch=batch, tokens=tokens, nodes=nodes, spread=spread, d=d, page=page,
                window=window, softcap=softcap, sinks=sinks, dtype=dtype)


def _adjust(name, batch, tokens, spread=1, vocab=VOCAB, nodes=0, kept=1.0, bias=0):
    return dict(name=name, op="adjust_logits", batch=batch, tokens=tokens, spread=spread, vocab=vocab, nodes=nodes, kept=kept, bias=bias)


def _accept(name, batch, nodes, depth):
    return dict(name=name, op="tree_accept", batch=batch, nodes=nodes, depth=depth)


def _keep(name, batch, nodes, depth, layers, page=16, d=128, heads="8b", dtype="bfloat16"):
    return dict(name=name, op="cache_keep", batch=batch, nodes=nodes, depth=depth, layers=layers, page=page, d=d, heads=heads, dtype=dtype)


def listed():
    return [
        # one short chat with a small model and a small tree: latency
        _attention("attend_one_chat", "0.6b", 1, 300, 8),
        # the benchmark's decode step, 8 requests of 2,048 tokens, each with a tree of 26 nodes
        _attention("attend_8x2048", "8b", 8, 2048, 26),
        # a busy server: requests of very different lengths, trees of up to 48 nodes
        _attention("attend_24_ragged", "14b", 24, 8192, 48, spread=32),
        # long documents under the largest trees: 256 columns a kv head
        _attention("attend_4x32k", "8b", 4, 32768, 64),
        # the float32 path, which replays and comparisons run on
        _attention("attend_float32", "0.6b", 2, 401, 21, spread=2, dtype="float32"),
        # one request with a penalty, nothing masked: latency
        _adjust("adjust_one", 1, 500),
        # a busy server under grammars: few tokens allowed, biases, long histories
        _adjust("adjust_48_grammar", 48, 8192, spread=32, kept=0.02, bias=100),
        # a tree's nodes: every node has the tokens on its path as well
        _adjust("adjust_8_trees", 8, 2048, nodes=26, kept=0.9, bias=10),
        # which guesses were right: one request, and a busy server
        _accept("accept_one", 1, 8, 4),
        _accept("accept_64", 64, 64, 8),
        # all layers of a small model for one request; a busy server's
        _keep("keep_one_28_layers", 1, 8, 4, 28, heads="0.6b"),
        _keep("keep_32_8_layers", 32, 48, 8, 8),
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "attention", "float32", "adjust", "adjust", "adjust", "accept", "keep"))
    nodes = _between(rng, 2, 64)
    if kind == "attention":
        batch, heads = _between(rng, 1, 48), rng.choice(("0.6b", "8b", "8b", "14b", "32b"))
        c = _attention("", heads, batch, _between(rng, 20, min(40000, 120000 // batch)), min(nodes, 2048 // HEADS[heads][0]),
                       spread=rng.choice((1, 2, 8, 32)), d=rng.choice((64, 128, 128, 128)), page=rng.choice((16, 16, 32, 64)),
                       window=rng.choice((0, 0, 0, 1024)), softcap=rng.choice((0.0, 0.0, 0.0, 30.0)), sinks=rng.random() < 0.25)
    elif kind == "float32":
        c = _attention("", rng.choice(("0.6b", "8b")), rng.randint(1, 4), _between(rng, 16, 1500), nodes, spread=rng.choice((1, 4)),
                       d=rng.choice((64, 128)), page=rng.choice((16, 32)), window=rng.choice((0, 0, 256)), dtype="float32")
    elif kind == "adjust":
        n = rng.choice((0, 0, _between(rng, 2, 40)))
        batch = _between(rng, 1, 64 if n == 0 else 8)
        c = _adjust("", batch, _between(rng, 8, 16000), spread=rng.choice((1, 8, 32)), vocab=rng.choice((VOCAB, _between(rng, 5001, 152001))),
                    nodes=n, kept=rng.choice((1.0, 1.0, 0.9, 0.1, 0.01)), bias=rng.choice((0, 0, 5, 300)))
    elif kind == "accept":
        c = _accept("", _between(rng, 1, 128), nodes, rng.randint(2, 10))
    else:
        batch = _between(rng, 1, 32)
        c = _keep("", batch, max(nodes, 4), rng.randint(2, 8), rng.randint(1, 8), page=rng.choice((16, 32)), d=rng.choice((64, 128)),
                  heads=rng.choice(("0.6b", "14b")), dtype=rng.choice(("bfloat16", "bfloat16", "float32")))
    del c["name"]
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _sizes(c):
    """The requests' lengths and how many nodes each tree has, by the case alone: one request has the most of each, the lengths of
    the others lie between a ``spread``-th of it and all of it, their trees between half and all."""
    rng = random.Random(c["batch"] * 7919 + c["nodes"])
    most, tokens = c["nodes"], c.get("tokens", 60)
    n = [tokens] + [_between(rng, max(1, tokens // c.get("spread", 8)), tokens) for _ in range(c["batch"] - 1)]
    rng.shuffle(n)
    return n, [most] + [rng.randint(-(-most // 2), most) for _ in range(c["batch"] - 1)]


def _tree(rng, n, depth):
    """Parents of a tree of n nodes, at most ``depth`` on a path: the likeliest path first, then branches off it."""
    depth = max(1, min(depth, n))
    parents, at = [-1], [0]
    for i in range(1, n):
        p = i - 1 if i < depth else rng.choice([j for j in range(i) if at[j] < depth - 1] or [0])
        parents.append(p)
        at.append(at[p] + 1)
    return parents


def _trees(c, rng):
    """The requests' trees: the parents by request, the depth of the deepest path, and the tables on the host."""
    depth, sizes = c.get("depth") or max(2, min(8, c["nodes"] // 2)), _sizes(c)[1]
    trees = [_tree(rng, n, depth) for n in sizes]
    words = -(-c["nodes"] // 32)
    bits = np.zeros((sum(sizes), words), dtype=np.uint32)
    cu = np.cumsum([0] + sizes).astype(np.int32)
    for r, parents in enumerate(trees):
        for i, p in enumerate(parents):
            row = bits[cu[r] + i]
            if p >= 0:
                row[:] = bits[cu[r] + p]
            row[i // 32] |= np.uint32(1 << (i % 32))
    return trees, depth, cu, bits.view(np.int32)


def _send(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(DEVICE)


def _children(parents):
    kids = [[] for _ in parents]
    for i, p in enumerate(parents):
        if p >= 0:
            kids[p].append(i)
    return kids


def prepare(case, seed):
    rng = random.Random(seed * 1000003 + 17)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"tree_attention": _prepare_attention, "adjust_logits": _prepare_adjust, "tree_accept": _prepare_accept,
            "cache_keep": _prepare_keep}[case["op"]](case, rng, gen) | {"case": case}


def _pages(rng, lengths, page):
    """A pool's pages dealt to requests of these lengths in any order: the tables, and how many pages the pool has."""
    need = [-(-n // page) for n in lengths]
    order = list(range(sum(need) + 3))
    rng.shuffle(order)
    table = np.zeros((len(need), max(need)), dtype=np.int32)
    for r, k in enumerate(need):
        table[r, :k] = order[:k]
        del order[:k]
    return table, sum(need) + 3


def _prepare_attention(c, rng, gen):
    nq, nkv = HEADS[c["heads"]]
    dt = getattr(torch, c["dtype"])
    start = _sizes(c)[0]
    _, _, cu, bits = _trees(c, rng)
    table, pool = _pages(rng, [s + int(n) for s, n in zip(start, np.diff(cu))], c["page"])
    s = dict(q=(2.0 * torch.randn(int(cu[-1]), nq * c["d"], device=DEVICE, generator=gen)).to(dt),
             k=torch.randn(pool, nkv, c["page"], c["d"], device=DEVICE, generator=gen, dtype=dt),
             v=torch.randn(pool, nkv, c["d"], c["page"], device=DEVICE, generator=gen, dtype=dt),
             sinks=torch.randn(nq, device=DEVICE, generator=gen) if c["sinks"] else None,
             table=_send(table), cu=_send(cu), start=_send(start), bits=_send(bits), nq=nq, nkv=nkv)
    return s


def _prepare_adjust(c, rng, gen):
    V, R = c["vocab"], c["batch"]
    lens = _sizes(c)[0]
    rows, drafts = R, None
    if c["nodes"]:
        _, _, cu, bits = _trees(c, rng)
        rows = int(cu[-1])
        drafts = (torch.randint(0, V, (rows,), device=DEVICE, generator=gen, dtype=torch.int32), _send(cu), _send(bits))
    # tokens repeat as they do in texts: few tokens often, many once
    u = torch.rand(sum(lens), device=DEVICE, generator=gen)
    history = (V * u.square() * u.square()).to(torch.int32).clamp_(max=V - 1)
    s = dict(logits=4.0 * torch.randn(rows, V, device=DEVICE, generator=gen), history=history, drafts=drafts,
             cu=_send(np.cumsum([0] + lens)), prompt=_send([rng.randint(0, n) for n in lens]),
             repetition=_send([rng.choice((1.0, 1.1, 1.3)) for _ in lens], np.float32),
             presence=_send([rng.choice((0.0, 0.5, 1.5)) for _ in lens], np.float32),
             frequency=_send([rng.choice((0.0, 0.2, 1.0, -0.3)) for _ in lens], np.float32),
             bias=None, masks=None)
    if c["bias"]:
        k = [rng.randint(0, c["bias"]) for _ in lens]
        k[0] = c["bias"]
        ids = np.concatenate([np.asarray(rng.sample(range(V), n), dtype=np.int32) for n in k])
        s["bias"] = (_send(ids), _send([rng.choice((-100.0, -2.5, 0.7, 5.0)) for _ in ids], np.float32), _send(np.cumsum([0] + k)))
    if c["kept"] < 1.0:
        words, M = -(-V // 32), max(1, min(rows, 40))
        hit = torch.rand(M, words * 32, device=DEVICE, generator=gen) < c["kept"]
        packed = (hit.view(M, words, 32).to(torch.int64) << torch.arange(32, device=DEVICE)).sum(-1)
        packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        s["masks"] = (packed, _send([rng.randrange(-1 if i % 8 == 7 else 0, M) for i in range(rows)]))
    return s


def _prepare_accept(c, rng, gen):
    trees, depth, cu, bits = _trees(c, rng)
    tokens = np.array([rng.randrange(VOCAB) for _ in range(int(cu[-1]))], dtype=np.int32)
    choices = np.array([rng.randrange(VOCAB) for _ in range(int(cu[-1]))], dtype=np.int32)
    for r, parents in enumerate(trees):
        for i, kids in enumerate(_children(parents)):
            if kids and rng.random() < 0.8:       # the model agrees with one of the guesses
                choices[cu[r] + i] = tokens[cu[r] + rng.choice(kids)]
    return dict(tokens=_send(tokens), choices=_send(choices), cu=_send(cu), bits=_send(bits), depth=depth)


def _prepare_keep(c, rng, gen):
    nkv, dt = HEADS[c["heads"]][1], getattr(torch, c["dtype"])
    trees, depth, cu, _ = _trees(c, rng)
    start = _sizes(c)[0]
    table, pool = _pages(rng, [s + len(t) for s, t in zip(start, trees)], c["page"])
    path, counts = np.full((len(trees), depth), -1, dtype=np.int32), []
    for r, parents in enumerate(trees):
        kids, at = _children(parents), [0]
        while kids[at[-1]] and len(at) < depth and rng.random() < 0.85:
            at.append(rng.choice(kids[at[-1]]))
        path[r, :len(at)] = at
        counts.append(len(at))
    caches = [(torch.randn(pool, nkv, c["page"], c["d"], device=DEVICE, generator=gen, dtype=dt),
               torch.randn(pool, nkv, c["d"], c["page"], device=DEVICE, generator=gen, dtype=dt)) for _ in range(c["layers"])]
    return dict(caches=caches, table=_send(table), start=_send(start), path=_send(path), counts=_send(counts))


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    return {"tree_attention": _run_attention, "adjust_logits": _run_adjust, "tree_accept": _run_accept,
            "cache_keep": _run_keep}[state["case"]["op"]](state)


def _unpacked(bits):
    """[rows, words] of 32 bits each -> truth values [rows, 32 words]."""
    at = torch.arange(32, device=bits.device, dtype=torch.int32)
    return ((bits[:, :, None] >> at) & 1).bool().view(bits.shape[0], -1)


def _owners(cu, rows):
    """The request of each row."""
    return torch.searchsorted(cu, torch.arange(rows, device=cu.device, dtype=cu.dtype), right=True) - 1


def _run_attention(s):
    c = s["case"]
    nq, nkv, d = s["nq"], s["nkv"], c["d"]
    scale = 1.0 / math.sqrt(d)
    if own:
        from tffinfer_amd.kernels import ops
        return ops.tree_attention(s["q"], nq, nkv, d, s["k"], s["v"], s["table"], s["cu"], s["start"], s["bits"], window=c["window"],
                                  scale=scale, sinks=s["sinks"], softcap=c["softcap"])
    T, R = s["q"].shape[0], s["start"].numel()
    G, N = nq // nkv, 32 * s["bits"].shape[1]
    k = s["k"][s["table"].long()].permute(0, 2, 1, 3, 4).reshape(R, nkv, -1, d).float()           # [R, nkv, places, d]
    v = s["v"][s["table"].long()].permute(0, 2, 1, 4, 3).reshape(R, nkv, -1, d).float()
    owner = _owners(s["cu"], T)
    node = torch.arange(T, device=DEVICE) - s["cu"][owner]
    q = torch.zeros(R, N, nkv, G, d, device=DEVICE)
    q[owner, node] = s["q"].float().view(T, nkv, G, d)
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(R, nkv, N * G, d), k.transpose(2, 3).contiguous()) * scale
    if c["softcap"] > 0:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    # what a node sees: the cached tokens, then the nodes that its bits name; under a window the last of these
    seen = _unpacked(s["bits"])
    place = torch.arange(k.shape[2], device=DEVICE)
    drafted = place[None] - s["start"][:, None]                                                   # [R, places]: which node lies there
    inside = (drafted[owner] >= 0) & (drafted[owner] < N) & seen.gather(1, drafted[owner].clamp(0, N - 1))
    cached = drafted[owner] < 0
    visible = cached | inside
    if c["window"]:
        below = seen.sum(1)[:, None] - inside.long().cumsum(1)                                    # visible nodes behind this place
        behind = torch.where(cached, s["start"][owner][:, None] - 1 - place[None] + seen.sum(1)[:, None], below)
        visible = visible & (behind < c["window"])
    full = torch.zeros(R, N, k.shape[2], dtype=torch.bool, device=DEVICE)
    full[owner, node] = visible
    score = torch.where(full[:, None, :, None, :], score.view(R, nkv, N, G, -1), -math.inf)
    most = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, nkv, 1, G, 1)
        most = torch.maximum(most, sink)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp(score - most)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - most)
    o = torch.matmul(p.view(R, nkv, N * G, -1), v).view(R, nkv, N, G, d) / total
    return o.permute(0, 2, 1, 3, 4)[owner, node].reshape(T, nq * d).to(s["q"].dtype)


def _run_adjust(s):
    if own:
        from tffinfer_amd.kernels import ops
        return ops.adjust_logits(s["logits"], s["history"], s["cu"], s["prompt"], s["repetition"], s["presence"], s["frequency"],
                                 bias=s["bias"], masks=s["masks"], drafts=s["drafts"])
    rows, V = s["logits"].shape
    R = s["cu"].numel() - 1
    owner = torch.arange(rows, device=DEVICE) if s["drafts"] is None else _owners(s["drafts"][1], rows)
    whose = _owners(s["cu"], s["history"].numel())
    tokens = s["history"].long()
    is_output = (torch.arange(tokens.numel(), device=DEVICE) - s["cu"][whose]) >= s["prompt"][whose]
    count = torch.zeros(R, V, device=DEVICE).index_put_((whose, tokens), is_output.float(), accumulate=True)[owner]
    seen = torch.zeros(R, V, device=DEVICE).index_put_((whose, tokens), torch.ones_like(tokens, dtype=torch.float32), accumulate=True)[owner]
    if s["drafts"] is not None:
        drafted, cu, bits = s["drafts"]
        on_path = _unpacked(bits)
        at = (cu[owner][:, None] + torch.arange(on_path.shape[1], device=DEVICE)).clamp(max=rows - 1)
        path = torch.zeros(rows, V, device=DEVICE).scatter_add_(1, drafted[at].long(), on_path.float())
        count, seen = count + path, seen + path
    x, pen = s["logits"], s["repetition"][owner][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / pen, x * pen), x)
    x = x - s["frequency"][owner][:, None] * count - s["presence"][owner][:, None] * (count > 0)
    if s["bias"] is not None:
        ids, values, cu_bias = s["bias"]
        x = x + torch.zeros(R, V, device=DEVICE).index_put_((_owners(cu_bias, ids.numel()), ids.long()), values)[owner]
    if s["masks"] is not None:
        packed, which = s["masks"]
        allowed = _unpacked(packed)[:, :V][which.clamp(min=0).long()] | (which < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    return x


def _run_accept(s):
    if own:
        from tffinfer_amd.kernels import ops
        return ops.tree_accept(s["choices"], s["tokens"], s["cu"], s["bits"], s["depth"])
    T, R, N = s["tokens"].numel(), s["cu"].numel() - 1, 32 * s["bits"].shape[1]
    owner = _owners(s["cu"], T)
    node = torch.arange(T, device=DEVICE) - s["cu"][owner]
    seen = _unpacked(s["bits"])
    at = torch.arange(N, device=DEVICE)
    parent = torch.where(seen & (at[None] < node[:, None]), at[None], -1).amax(1)
    parent_row = s["cu"][owner] + parent.clamp(min=0)
    right = (parent < 0) & (node == 0) | (parent >= 0) & (s["tokens"] == s["choices"][parent_row])
    # of a node's children that are right, the first
    same = torch.full((T,), N, device=DEVICE, dtype=torch.int64).scatter_reduce_(0, parent_row, torch.where(right & (parent >= 0), node, N), "amin")
    right = right & ((node == 0) | (same[parent_row] == node))
    # a node is kept if all on its path are, and the path is short enough
    row = s["cu"][owner][:, None] + at.clamp(max=N - 1)
    kept = (~seen | right[row.clamp(max=T - 1)]).all(1) & (seen.sum(1) <= s["depth"])
    depth = seen.sum(1) - 1
    path = torch.full((R, s["depth"]), -1, device=DEVICE, dtype=torch.int32)
    path[owner, torch.where(kept, depth, 0)] = torch.where(kept, node, 0).to(torch.int32)
    counts = torch.zeros(R, device=DEVICE, dtype=torch.int32).index_put_((owner,), kept.to(torch.int32), accumulate=True)
    last = path.gather(1, (counts.long() - 1)[:, None])[:, 0]
    return path, counts, s["choices"][s["cu"][:-1] + last]


def _moved(cache, slot_from, slot_to, keep, page, values):
    """One cache's kept places: [page, head, place, element], for values [page, head, element, place]."""
    a, b = (slot_from // page, slot_from % page), (slot_to // page, slot_to % page)
    if values:
        cache[b[0], :, :, b[1]] = torch.where(keep[:, None, None], cache[a[0], :, :, a[1]], cache[b[0], :, :, b[1]])
    else:
        cache[b[0], :, b[1]] = torch.where(keep[:, None, None], cache[a[0], :, a[1]], cache[b[0], :, b[1]])


def _run_keep(s):
    if own:
        from tffinfer_amd.kernels import ops
        ops.cache_keep(s["caches"], s["table"], s["start"], s["path"], s["counts"])
        return s["caches"]
    page, D = s["case"]["page"], s["path"].shape[1]
    i = torch.arange(D, device=DEVICE)
    keep = (i[None] < s["counts"][:, None]).reshape(-1)
    source = s["start"][:, None] + torch.where(i[None] < s["counts"][:, None], s["path"], 0)
    target = s["start"][:, None] + torch.where(i[None] < s["counts"][:, None], i[None], 0)
    slots = [(s["table"].gather(1, (x // page).long()).long() * page + x % page).reshape(-1) for x in (source, target)]
    # (a place that is not kept writes node 0's own bits to node 0's place)
    for k, v in s["caches"]:
        _moved(k, *slots, keep, page, False)
        _moved(v, *slots, keep, page, True)
    return s["caches"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    (lens, nodes), size = _sizes(c), 4 if c.get("dtype") == "float32" else 2
    rows = sum(nodes)
    if c["op"] == "tree_attention":
        nq, nkv = HEADS[c["heads"]]
        keys = pairs = 0
        for n, t in zip(lens, _trees(c, random.Random(1))[0]):
            depth = []
            for p in t:
                depth.append(1 if p < 0 else depth[p] + 1)
            most = c["window"] or math.inf
            keys += min(n, most) + len(t)
            pairs += sum(min(n + k, most) for k in depth)
        return {"bytes": 2 * keys * nkv * c["d"] * size + 2 * rows * nq * c["d"] * size + 4 * rows * -(-c["nodes"] // 32) + 4 * keys / c["page"],
                "flops": 4 * pairs * nq * c["d"]}
    if c["op"] == "adjust_logits":
        rows, V = rows or c["batch"], c["vocab"]
        masks = 4 * min(rows, 40) * -(-V // 32) if c["kept"] < 1 else 0
        # a masked logit is written and not read
        return {"bytes": 4 * rows * V * (1 + c["kept"]) + masks + 4 * sum(lens) + 8 * c["bias"] * c["batch"] / 2, "flops": 4 * rows * V * c["kept"]}
    if c["op"] == "tree_accept":
        return {"bytes": rows * 4 * (2 + -(-c["nodes"] // 32)) + 4 * c["batch"] * (c["depth"] + 3), "flops": rows}
    # (about half of a path's places are moved: the others have their nodes already)
    moved = c["batch"] * c["depth"] / 4
    return {"bytes": moved * 2 * 2 * HEADS[c["heads"]][1] * c["d"] * size * c["layers"] + 4 * c["batch"] * (c["depth"] + 2), "flops": 0}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree_attention": _exact_attention, "adjust_logits": _exact_adjust, "tree_accept": _exact_accept,
            "cache_keep": _exact_keep}[case["op"]](s, case)


def _bits_of(words, n):
    """The numbers below n whose bits are set."""
    return [j for j in range(n) if (int(words[j // 32]) >> (j % 32)) & 1]


def _exact_attention(s, c):
    nq, nkv, d, page = s["nq"], s["nkv"], c["d"], c["page"]
    G = nq // nkv
    cu, start, bits = s["cu"].tolist(), s["start"].tolist(), s["bits"].cpu().numpy()
    out = torch.zeros(cu[-1], nq, d, dtype=torch.float64, device=DEVICE)
    for r, first in enumerate(start):
        n = cu[r + 1] - cu[r]
        pages = s["table"][r, :-(-(first + n) // page)].long()
        k = s["k"][pages].double().transpose(0, 1).reshape(nkv, -1, d)
        v = s["v"][pages].double().permute(1, 0, 3, 2).reshape(nkv, -1, d)
        hidden = torch.ones(n, k.shape[1], dtype=torch.bool)
        for i in range(n):
            sees = list(range(first)) + [first + j for j in _bits_of(bits[cu[r] + i], n)]
            hidden[i, sees[-c["window"]:] if c["window"] else sees] = False
        hidden = hidden.to(DEVICE)
        q = s["q"][cu[r]:cu[r + 1]].double().view(n, nkv, G, d)
        for g in range(nkv):
            z = (q[:, g].reshape(n * G, d) @ k[g].T).view(n, G, -1) / math.sqrt(d)
            if c["softcap"]:
                z = torch.tanh(z / c["softcap"]) * c["softcap"]
            z = z.masked_fill(hidden[:, None], -math.inf)
            if s["sinks"] is not None:
                z = torch.cat([z, s["sinks"].double().view(1, nkv, G)[:, g, :, None].expand(n, G, 1)], dim=2)
            w = torch.softmax(z, dim=-1)[:, :, :k.shape[1]]
            out[cu[r]:cu[r + 1], g * G:(g + 1) * G] = (w.reshape(n * G, -1) @ v[g]).view(n, G, d)
    return out.view(cu[-1], nq * d)


def _exact_adjust(s, c):
    rows, V = s["logits"].shape
    x = s["logits"].double()
    cu, prompt = s["cu"].tolist(), s["prompt"].tolist()
    rep, pres, freq = (s[n].double().tolist() for n in ("repetition", "presence", "frequency"))
    owner, trees = list(range(rows)), None
    if s["drafts"] is not None:
        trees, bits, first = s["drafts"][0].tolist(), s["drafts"][2].cpu().numpy(), s["drafts"][1].tolist()
        owner = [r for r in range(len(prompt)) for _ in range(first[r], first[r + 1])]
    allowed = None
    if s["masks"] is not None:
        which = s["masks"][1].tolist()
        allowed = np.unpackbits(s["masks"][0].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V]
        allowed = torch.from_numpy(allowed).to(DEVICE).bool()
    history = s["history"].long()
    for t, r in enumerate(owner):
        past = history[cu[r]:cu[r + 1]]
        outputs = past[prompt[r]:]
        if trees is not None:
            mine = [trees[first[r] + j] for j in _bits_of(bits[t], first[r + 1] - first[r])]
            mine = torch.tensor(mine, device=DEVICE, dtype=torch.int64)
            past, outputs = torch.cat([past, mine]), torch.cat([outputs, mine])
        there = torch.bincount(past, minlength=V) > 0
        times = torch.bincount(outputs, minlength=V).double()
        row = x[t]
        row = torch.where(there & (row > 0), row / rep[r], torch.where(there, row * rep[r], row))
        row = row - freq[r] * times - pres[r] * torch.sign(times)
        if s["bias"] is not None:
            b0, b1 = s["bias"][2][r:r + 2].tolist()
            row[s["bias"][0][b0:b1].long()] += s["bias"][1][b0:b1].double()
        if allowed is not None and which[t] >= 0:
            row[~allowed[which[t]]] = -math.inf
        x[t] = row
    return x


def _exact_accept(s, c):
    cu, bits = s["cu"].tolist(), s["bits"].cpu().numpy()
    tokens, choices = s["tokens"].tolist(), s["choices"].tolist()
    path, counts, following = [], [], []
    for a, b in zip(cu, cu[1:]):
        kept = [0]
        while len(kept) < s["depth"]:
            children = [i for i in range(kept[-1] + 1, b - a) if _bits_of(bits[a + i], i)[-1:] == [kept[-1]] and tokens[a + i] == choices[a + kept[-1]]]
            if not children:
                break
            kept.append(children[0])
        path.append(kept + [-1] * (s["depth"] - len(kept)))
        counts.append(len(kept))
        following.append(choices[a + kept[-1]])
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in (path, counts, following))


def _exact_keep(s, c):
    page, table, path = c["page"], s["table"].tolist(), s["path"].tolist()
    out = [(k.clone(), v.clone()) for k, v in s["caches"]]
    for r, (first, n) in enumerate(zip(s["start"].tolist(), s["counts"].tolist())):
        for i in range(n):
            (pa, sa), (pb, sb) = (divmod(first + x, page) for x in (path[r][i], i))
            for (k, v), (k2, v2) in zip(s["caches"], out):
                k2[table[r][pb], :, sb] = k[table[r][pa], :, sa]
                v2[table[r][pb], :, :, sb] = v[table[r][pa], :, :, sa]
    return out
