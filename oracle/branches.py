"""Branching sequences over a paged cache, entry by entry on the CPU: forks, kept nodes, beams, trees.

The pages' functions work on lists and CPU tensors in place, one row, page and position after the
other, as the kernels' contract words them; attention and scores are computed in 64 bits.
"""
from __future__ import annotations

import math

import torch


def fork(k_pages, v_pages, table, lengths, parents, refs, room: int = 1) -> bool:
    """Fork ``table`` [S, P], ``lengths`` [S], ``refs`` [N] (int tensors) and the pages
    [layers, N, kv, page, hd] in place; False if a page was missing."""
    S, P = table.shape
    page = k_pages.shape[3]
    old, n_old = table.tolist(), lengths.tolist()
    ok = True
    for i, p in enumerate(parents.tolist()):
        new = list(old[p]) if p >= 0 else [-1] * P
        for was, now in zip(old[i], new):
            if was >= 0:
                refs[was] -= 1
            if now >= 0:
                refs[now] += 1
        table[i] = torch.tensor(new, dtype=table.dtype)
        lengths[i] = n_old[p] if p >= 0 else 0
    for i, p in enumerate(parents.tolist()):
        n = int(lengths[i])
        if p < 0 or n < 0 or room == 0:
            continue
        for c in range(n // page, min((n + room - 1) // page + 1, P)):
            g = int(table[i, c])
            if g >= 0 and int(refs[g]) == 1:
                continue
            free = (refs == 0).nonzero()[:, 0]
            dst = int(free[0]) if len(free) else -1
            if g >= 0:
                refs[g] -= 1
            table[i, c] = dst
            if dst < 0:
                ok = False
                continue
            refs[dst] = 1
            filled = n - c * page
            if g >= 0 and filled > 0:
                for pages in (k_pages, v_pages):
                    pages[:, dst, :, :filled] = pages[:, g, :, :filled]
    return ok


def keep_nodes(k_pages, v_pages, table, lengths, keep):
    """Move the kept nodes' rows in place; the new lengths (list)."""
    page = k_pages.shape[3]
    out = []
    for b, n in enumerate(lengths.tolist()):
        kept = 0
        for j, node in enumerate(keep[b].tolist() if n >= 0 else []):
            if node < 0:
                break
            src, dst = n + node, n + j
            for pages in (k_pages, v_pages):
                pages[:, table[b, dst // page], :, dst % page] = (
                    pages[:, table[b, src // page], :, src % page])
            kept += 1
        out.append(n + kept)
    return out


def beam_select(logits, scores, count: int):
    """(scores float64, parents, tokens) of one group: logits [K, V] and scores [K], by the definition;
    what is at -inf is no candidate and leaves (-inf, 0, 0)."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    found = []
    for k in range(x.shape[0]):
        top = x[k].max()
        d = torch.where(x[k] == top, 0.0, x[k] - top)
        v = float(scores[k]) + (d - d.exp().sum().log())
        v = torch.where(x[k].isneginf() | v.isnan(), -math.inf, v)
        order = torch.sort(x[k], descending=True, stable=True).indices[:count]
        found += [(float(v[t]), k, i, int(t)) for i, t in enumerate(order) if v[t] > -math.inf]
    found = sorted(found, key=lambda f: (-f[0], f[1], f[2]))[:count]
    found += [(-math.inf, 0, 0, 0)] * (count - len(found))
    return (torch.tensor([f[0] for f in found], dtype=torch.float64), [f[1] for f in found],
            [f[3] for f in found])


def tree_attention(q, k, v, seen, scale: float):
    """q [T, H, hd], k / v [n, KV, hd] of one sequence, ``seen`` bool [T, n] -> (out, weight, off)
    float64 as :func:`oracle.serving.attention` returns them; a node that sees nothing gives zeros.
    Values of keys that a node does not see have no effect, whatever they hold."""
    T, H, hd = q.shape
    n, KV = k.shape[:2]
    out = torch.zeros(T, H, hd, dtype=torch.float64)
    weight, off = torch.zeros_like(out), torch.zeros(T, H, 1, dtype=torch.float64)
    for t in range(T):
        at = seen[t].nonzero()[:, 0]
        if len(at) == 0:
            continue
        ks, vs = (x[at].double().repeat_interleave(H // KV, 1) for x in (k, v))
        s = torch.einsum("hd,nhd->hn", q[t].double(), ks) * scale
        p = torch.softmax(s, -1)
        out[t] = torch.einsum("hn,nhd->hd", p, vs)
        weight[t] = torch.einsum("hn,nhd->hd", p, vs.abs())
        big = torch.einsum("hd,nhd->hn", q[t].double().abs(), ks.abs()) * scale
        off[t] = big.amax(-1, keepdim=True) * hd * 2.0 ** -24
    return out, weight, off
