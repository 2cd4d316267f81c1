"""Trees of drafted tokens, options on logits: the operators of a verifying step in plain float64 loops, by their definitions."""
import math

import numpy as np
import torch


def random_tree(rng, n, depth):
    """Parents (-1 first) of n nodes, each behind its parent, no path longer than ``depth``."""
    parents, at = [-1], [1]
    for i in range(1, n):
        p = rng.choice([j for j in range(i) if at[j] < max(2, depth)])
        parents.append(p)
        at.append(at[p] + 1)
    return parents


def paths(parents):
    """Every node's path from the root, itself included."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def packed(rows, words):
    """Lists of numbers -> int32 [rows, words] with their bits."""
    bits = np.zeros((len(rows), words), dtype=np.uint32)
    for i, r in enumerate(rows):
        for j in r:
            bits[i, j // 32] |= np.uint32(1 << (j % 32))
    return torch.from_numpy(bits.view(np.int32))


def attention(q, k, v, start, sees, nq, nkv, window=0, scale=None, sinks=None, softcap=0.0):
    """q [n, nq, d]; k, v [places, nkv, d] (the cached ones, then the nodes); sees[i]: the nodes that node i sees.  float64 [n, nq, d], and
    the same with |v| and the largest sum of |q k| scale: what bounds the error."""
    n, _, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out, out_abs, most = torch.zeros(n, nq, d, dtype=torch.float64), torch.zeros(n, nq, d, dtype=torch.float64), 0.0
    for i in range(n):
        places = list(range(start)) + [start + j for j in sees[i]]
        places = places[-window:] if window else places
        for h in range(nq):
            g = h // (nq // nkv)
            s = (k[places, g] @ q[i, h]) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            terms = torch.cat([s, sinks[h].double().view(1)]) if sinks is not None else s
            if not len(terms):
                continue
            p = torch.softmax(terms, 0)[:len(places)]
            out[i, h], out_abs[i, h] = p @ v[places, g], p @ v[places, g].abs()
            if places:
                most = max(most, float((k[places, g].abs() @ q[i, h].abs()).max()) * abs(scale))
    return out, out_abs, most


def adjust(logits, histories, prompt_lens, repetition, presence, frequency, biases=None, masks=None, mask_rows=None, trees=None):
    """Rows [rows, V]; histories and biases (lists of (token, value)) per request; trees: per request (tokens, sees).  float64, and a bound on
    what the terms' roundings to 24 bits add up to."""
    rows, V = logits.shape
    x = logits.double().clone()
    owner = [(r, None) for r in range(len(histories))]
    if trees is not None:
        owner = [(r, i) for r, (tokens, _) in enumerate(trees) for i in range(len(tokens))]
    size = torch.zeros_like(x)
    for t, (r, i) in enumerate(owner):
        past, outputs = list(histories[r]), list(histories[r][prompt_lens[r]:])
        if i is not None:
            mine = [trees[r][0][j] for j in trees[r][1][i]]
            past, outputs = past + mine, outputs + mine
        for v in sorted(set(past)):
            if 0 <= v < V:
                a = x[t, v].clone()
                x[t, v] = a / repetition[r] if a > 0 else a * repetition[r]
                n = outputs.count(v)
                size[t, v] = x[t, v].abs()
                if n:
                    x[t, v] -= frequency[r] * n + presence[r]
                    size[t, v] += abs(frequency[r] * n) + abs(presence[r])
        for v, b in dict(biases[r]).items() if biases is not None else ():
            if 0 <= v < V:
                size[t, v] += x[t, v].abs() + abs(b)
                x[t, v] += b
        if mask_rows is not None and 0 <= mask_rows[t] < len(masks):
            allowed = torch.zeros(V, dtype=torch.bool)
            allowed[[v for v in masks[mask_rows[t]] if v < V]] = True
            x[t, ~allowed] = -math.inf
    return x, size


def accept(choices, tokens, trees, max_path):
    """choices, tokens: lists per request; trees: the parents per request."""
    out = []
    for c, t, parents in zip(choices, tokens, trees):
        kept = [0] if parents else []
        while kept and len(kept) < max_path:
            right = [i for i, p in enumerate(parents) if p == kept[-1] and t[i] == c[kept[-1]]]
            if not right:
                break
            kept.append(right[0])
        out.append((kept + [-1] * (max_path - len(kept)), len(kept), c[kept[-1]] if kept else -1))
    return out
