"""Cases of the operators that follow several continuations of a sequence over the paged cache.

``tree_attention`` (a tree of drafted tokens over a sequence's pages) and ``keep_nodes`` (the
accepted nodes' keys and values move to the front) are a step of speculative decoding;
``beam_select`` (the best continuations over beams and vocabulary) and ``fork_pages`` (each beam
becomes its parent's copy: pages shared, copied where written, freed) are a step of beam search.
With ``own`` false, :func:`run` computes a case in elementary torch operations in 32 bits, rounded
once; with ``own`` true it calls the framework.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One chat with a small draft, 32 query / 8 KV heads of 128: latency counts.
        {"name": "tree one short", "op": "tree_attention", "dtype": "fp16", "seqs": 1, "lo": 72,
         "hi": 72, "nodes": 16, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 1},
        # A serving batch of 64 sequences between 512 and 640 tokens, 8 drafted tokens each.
        {"name": "tree a batch", "op": "tree_attention", "dtype": "fp16", "seqs": 64, "lo": 512,
         "hi": 640, "nodes": 8, "heads": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 2},
        # Wide trees of 64 nodes over a few thousand tokens.
        {"name": "tree wide", "op": "tree_attention", "dtype": "bf16", "seqs": 16, "lo": 2049,
         "hi": 4095, "nodes": 64, "heads": 32, "kv": 8, "hd": 128, "page": 64, "lens_seed": 3},
        # Long documents: few sequences, the cache's length is the work; odd lengths and nodes.
        {"name": "tree long", "op": "tree_attention", "dtype": "bf16", "seqs": 2, "lo": 65537,
         "hi": 131071, "nodes": 27, "heads": 32, "kv": 8, "hd": 128, "page": 64, "lens_seed": 4},
        # One prompt, 4 beams, a vocabulary of 32000.
        {"name": "beams of one", "op": "beam_select", "dtype": "fp16", "seqs": 1, "beams": 4,
         "vocab": 32000, "count": 4},
        # A batch of prompts; twice the beams are asked for, so that ended ones can be set aside.
        {"name": "beams of a batch", "op": "beam_select", "dtype": "fp16", "seqs": 16, "beams": 4,
         "vocab": 32000, "count": 8},
        # Many beams over a wide vocabulary, fp32 logits.
        {"name": "beams wide", "op": "beam_select", "dtype": "fp32", "seqs": 32, "beams": 8,
         "vocab": 131072, "count": 16},
        # 4 beams of one prompt: a step's reordering, all 32 layers.
        {"name": "fork one", "op": "fork_pages", "dtype": "fp16", "seqs": 1, "beams": 4, "lo": 40,
         "hi": 40, "grown": 35, "layers": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 8},
        # 16 prompts of 4 beams each, pages of 64.
        {"name": "fork a batch", "op": "fork_pages", "dtype": "fp16", "seqs": 16, "beams": 4,
         "lo": 400, "hi": 512, "grown": 100, "layers": 32, "kv": 8, "hd": 128, "page": 64,
         "lens_seed": 9},
        # 32 prompts of 8 beams, the 8 layers of one stage of a pipeline.
        {"name": "fork many", "op": "fork_pages", "dtype": "bf16", "seqs": 32, "beams": 8,
         "lo": 129, "hi": 512, "grown": 77, "layers": 8, "kv": 8, "hd": 128, "page": 64,
         "lens_seed": 10},
        # One chat: the accepted path of a tree of 16, all 32 layers.
        {"name": "keep one", "op": "keep_nodes", "dtype": "fp16", "seqs": 1, "lo": 72, "hi": 72,
         "nodes": 16, "layers": 32, "kv": 8, "hd": 128, "page": 16, "lens_seed": 11},
        # A batch of 64 sequences, trees of 64 nodes.
        {"name": "keep a batch", "op": "keep_nodes", "dtype": "fp16", "seqs": 64, "lo": 100,
         "hi": 300, "nodes": 64, "layers": 32, "kv": 8, "hd": 128, "page": 64, "lens_seed": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "beam_select", "fork_pages", "keep_nodes"])
    if op == "beam_select":
        seqs, beams = _spread(rng, 1, 32), _spread(rng, 1, 8)
        return {"op": op, "dtype": rng.choice(["fp16", "bf16", "fp32"]), "seqs": seqs,
                "beams": beams, "vocab": _spread(rng, 4000, 131072),
                "count": rng.choice([beams, 2 * beams])}
    heads, kv = rng.choice([(32, 8), (32, 8), (32, 32), (16, 2), (28, 4), (8, 1), (4, 2)])
    case = {"op": op, "dtype": rng.choice(["fp16", "bf16"]), "kv": kv, "hd": rng.choice([64, 128]),
            "page": rng.choice([16, 32, 64, 128]), "lens_seed": rng.randrange(1 << 20)}
    if op == "fork_pages":
        seqs, beams = _spread(rng, 1, 32), _spread(rng, 1, 8)
        hi, grown = _spread(rng, 1, 512), _spread(rng, 1, 128)
        fit = (16 * 8 * 640 * 32) // (seqs * kv * (hi + beams * (grown + 2 * case["page"])))
        case.update(seqs=seqs, beams=beams, lo=max(1, hi // 4), hi=hi, grown=grown,
                    layers=_spread(rng, 1, max(1, min(32, fit))))
        return case
    seqs, nodes = _spread(rng, 1, 64), _spread(rng, 2, 64)
    if op == "keep_nodes":
        hi = _spread(rng, 1, 300)
        fit = (64 * 8 * 364 * 32) // (seqs * kv * (hi + nodes + case["page"]))
        case.update(seqs=seqs, nodes=nodes, lo=max(1, hi // 4), hi=hi,
                    layers=_spread(rng, 1, max(1, min(32, fit))))
        return case
    if rng.random() < 0.2:
        nodes = _spread(rng, 65, 200)
    most = min(131071, 2 * 65536 * 8 // (seqs * kv), 2 * 65536 * 27 * 32 // (seqs * nodes * heads))
    hi = _spread(rng, 1, max(1, most))
    case.update(seqs=seqs, nodes=nodes, heads=heads, lo=max(1, hi // 4), hi=hi)
    return case


# -- what a case fixes: lengths, trees, parents --------------------------------------------------

def _lengths(case):
    """The sequences' lengths: a property of the case, not of the seed."""
    rng = random.Random(case["lens_seed"])
    n = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    n[0] = case["hi"]
    return n


def _trees(case):
    """Each sequence's tree as every node's parent (-1: the node follows the cached tokens)."""
    rng = random.Random(case["lens_seed"] + 1)
    return [[rng.randint(max(-1, j - 8), j - 1) if j else -1 for j in range(case["nodes"])]
            for _ in range(case["seqs"])]


def _accepted(case):
    """A path from a root of each sequence's tree, as verification leaves it."""
    rng = random.Random(case["lens_seed"] + 2)
    kept = []
    for tree in _trees(case):
        path, at = [], -1
        while True:
            below = [j for j, p in enumerate(tree) if p == at]
            if not below or rng.random() < 0.1:
                break
            at = rng.choice(below)
            path.append(at)
        kept.append(path)
    return kept


def _parents(case):
    """Each beam's parent row: a few good beams have several children."""
    rng = random.Random(case["lens_seed"] + 3)
    K = case["beams"]
    return [b * K + min(rng.randrange(K), rng.randrange(K)) for b in range(case["seqs"])
            for _ in range(K)]


# -- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(lens, page, g):
    """A block table over shuffled pages (entries past a sequence's last page are -1) and the count."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3  # a pool is never exactly full
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    need_t = torch.tensor(need, device="cuda")
    col = torch.arange(max(need), device="cuda")[None, :]
    start = (torch.cumsum(need_t, 0) - need_t)[:, None]
    table = torch.where(col < need_t[:, None], order[(start + col).clamp(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total


def _masks(case):
    """int64 [seqs, nodes, words]: bit j of a node's words is set for its ancestors and itself."""
    T = case["nodes"]
    words = -(-T // 64)
    rows = []
    for tree in _trees(case):
        seen = []
        for j, p in enumerate(tree):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        for m in seen:
            w = [m >> (64 * i) & (1 << 64) - 1 for i in range(words)]
            rows.append([x - (1 << 64) if x >> 63 else x for x in w])
    return torch.tensor(rows, dtype=torch.int64, device="cuda").view(case["seqs"], T, words)


def prepare(case, seed):
    g = _gen(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "beam_select":
        return _prepare_beams(case, dt, g)
    KV, hd, page = case["kv"], case["hd"], case["page"]
    st = {"op": op, "KV": KV, "hd": hd, "dtype": dt, "page": page}
    if op == "fork_pages":
        return _prepare_fork(case, st, g)
    lens, T = _lengths(case), case["nodes"]
    st["table"], total = _pages([n + T for n in lens], page, g)
    st["lengths"] = _int32(lens)
    if op == "keep_nodes":
        shape = (case["layers"], total, KV, page, hd)
        kept = _accepted(case)
        most = max(max(map(len, kept)), 1)
        st["keep"] = _int32([p + [-1] * (most - len(p)) for p in kept])
    else:
        shape = (total, KV, page, hd)
        st["H"], st["T"] = case["heads"], T
        st["q"] = _randn((case["seqs"], T, case["heads"], hd), dt, g)
        st["visible"] = _masks(case)
    st["k_pages"], st["v_pages"] = _randn(shape, dt, g), _randn(shape, dt, g)
    return st


def _prepare_beams(case, dt, g):
    B, K, V = case["seqs"], case["beams"], case["vocab"]
    # A language model's logits: a broad bulk and a few hundred candidates that stand out.
    x = 2.0 * torch.randn((B * K, V), device="cuda", generator=g)
    stand_out = torch.rand((B * K, V), device="cuda", generator=g) < 200 / V
    x += stand_out * (3.0 + 2.5 * torch.randn((B * K, V), device="cuda", generator=g).abs())
    scores = -30.0 + 2.0 * torch.randn((B, K), device="cuda", generator=g)
    return {"op": "beam_select", "logits": x.to(dt), "count": case["count"],
            "scores": scores.sort(dim=-1, descending=True).values.contiguous()}


def _prepare_fork(case, st, g):
    """Beams that share their prompt's full pages and hold their own from there on."""
    page, K = case["page"], case["beams"]
    rows, lens, used = [], [], 0
    for n in _lengths(case):
        total = n + case["grown"]
        shared = list(range(used, used + n // page))
        used += len(shared)
        for _ in range(K):
            mine = -(-total // page) - len(shared)
            rows.append(shared + list(range(used, used + mine)))
            used += mine
            lens.append(total)
    pool = used + 2 * len(rows) + 3
    width = max(map(len, rows)) + 1
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    table = _int32([r + [-1] * (width - len(r)) for r in rows])
    st["table"] = torch.where(table >= 0, order[table.clamp(min=0).long()], -1).to(torch.int32)
    st["lengths"], st["parents"] = _int32(lens), _int32(_parents(case))
    st["refs"] = torch.zeros(pool, dtype=torch.int32, device="cuda")
    held = st["table"].flatten()
    st["refs"].index_add_(0, held.clamp(min=0), (held >= 0).to(torch.int32))
    shape = (case["layers"], pool, case["kv"], page, case["hd"])
    st["k_pages"], st["v_pages"] = _randn(shape, st["dtype"], g), _randn(shape, st["dtype"], g)
    return st


# -- one pass ------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _PLAIN[state["op"]])(state)


def _run_own(st):
    from moeinfra_b200 import kernels

    op = st["op"]
    if op == "tree_attention":
        return {"o": kernels.tree_attention(st["q"], st["k_pages"], st["v_pages"], st["table"],
                                            st["lengths"], st["visible"])}
    if op == "beam_select":
        scores, parents, tokens = kernels.beam_select(st["logits"], st["scores"], st["count"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    if op == "fork_pages":
        kernels.fork_pages(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["parents"],
                           st["refs"])
        return _forked(st)
    lengths = kernels.keep_nodes(st["k_pages"], st["v_pages"], st["table"], st["lengths"],
                                 st["keep"])
    return {"lengths": lengths, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _forked(st):
    return {name: st[name] for name in ("table", "lengths", "refs", "k_pages", "v_pages")}


# -- plain forms ---------------------------------------------------------------------------------

def _plain_tree_attention(st):
    H, KV, hd, T, page = st["H"], st["KV"], st["hd"], st["T"], st["page"]
    B, P = st["table"].shape
    n = P * page
    at = st["table"].clamp(min=0).long()
    keys = st["k_pages"][at].transpose(1, 2).reshape(B, KV, n, hd).float()
    q = st["q"].float().transpose(1, 2).reshape(B, KV, H // KV * T, hd)
    s = (q @ keys.transpose(2, 3)).view(B, KV, H // KV, T, n)
    del keys
    node = torch.arange(n, device="cuda")[None] - st["lengths"][:, None].long()  # [B, n]
    here = node.clamp(0, T - 1)
    word = st["visible"].gather(2, (here // 64)[:, None].expand(B, T, n))
    seen = (word >> (here % 64)[:, None]) & 1 == 1
    seen = torch.where((node >= 0)[:, None], seen & (node < T)[:, None], True)
    s = s.mul_(1.0 / math.sqrt(hd)).masked_fill_(~seen[:, None, None], float("-inf"))
    e = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    vals = st["v_pages"][at].transpose(1, 2).reshape(B, KV, n, hd).float()
    o = (e.view(B, KV, H // KV * T, n) @ vals).view(B, KV, H // KV, T, hd)
    o = (o / e.sum(-1, keepdim=True)).reshape(B, H, T, hd).transpose(1, 2)
    return {"o": o.contiguous().to(st["dtype"])}


def _plain_beam_select(st):
    """Order: larger score, then lower beam, in it larger logit, then lower token."""
    B, K = st["scores"].shape
    M = st["count"]
    x = st["logits"].float() + 0.0
    x = x.masked_fill(x.isnan(), float("-inf"))
    top = x.amax(-1, keepdim=True)
    d = torch.where(x == top, 0.0, x - top)
    lse = torch.log(torch.exp(d).double().sum(-1, keepdim=True)).float()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :M]
    v = st["scores"].view(-1, 1) + (d.gather(1, order) - lse)
    v = v.masked_fill(v.isnan() | (x.gather(1, order) == float("-inf")), float("-inf"))
    value, at = torch.sort(v.reshape(B, -1), dim=-1, descending=True, stable=True)
    value, at = value[:, :M], at[:, :M]
    tokens = order.reshape(B, -1).gather(1, at)
    none = value == float("-inf")
    parents = torch.div(at, order.shape[1], rounding_mode="floor").masked_fill(none, 0)
    return {"scores": value, "parents": parents.to(torch.int32), "tokens": tokens.masked_fill(none, 0)}


def _plain_fork_pages(st):
    """Every row takes its parent's pages; the next position's page becomes its own."""
    table, lengths, parents, refs = st["table"], st["lengths"], st["parents"], st["refs"]
    page = st["page"]
    S, P = table.shape
    live = parents >= 0
    new = torch.where(live[:, None], table[parents.clamp(min=0).long()], -1)
    n = torch.where(live, lengths[parents.clamp(min=0).long()], 0)
    for t, step in ((new, 1), (table, -1)):
        refs.index_add_(0, t.flatten().clamp(min=0), step * (t.flatten() >= 0).to(torch.int32))
    col = (n // page).long()
    use = live & (col < P)
    col = col.clamp(max=P - 1)
    held = new.gather(1, col[:, None])[:, 0]
    src = held.clamp(min=0).long()
    # Of rows that write to one page all copy it but the last, unless others hold it too.
    before = ((held[:, None] == held[None]) & use[None]).long().tril(-1).sum(-1)
    copy = use & (held >= 0) & (refs[src] - before > 1)
    need = use & (copy | (held < 0))
    refs.index_add_(0, src, -copy.to(torch.int32))
    free = torch.sort((refs != 0).to(torch.int32), stable=True).indices
    count = (refs == 0).sum()
    turn = need.long().cumsum(0) - 1
    got = need & (turn < count)
    dst = free[turn.clamp(0, free.numel() - 1)]
    refs.index_add_(0, dst, got.to(torch.int32))
    mine = torch.where(need, torch.where(got, dst, -1), held.long()).to(torch.int32)
    new.scatter_(1, col[:, None], torch.where(use, mine, new.gather(1, col[:, None])[:, 0])[:, None])
    table.copy_(new)
    lengths.copy_(n)
    rows = (copy & got).nonzero()[:, 0]
    keep = torch.arange(page, device="cuda")[None] < (n[rows] % page)[:, None]
    keep = keep[None, :, None, :, None]
    for pages in (st["k_pages"], st["v_pages"]):
        pages[:, dst[rows]] = torch.where(keep, pages[:, src[rows]], pages[:, dst[rows]])
    return _forked(st)


def _plain_keep_nodes(st):
    table, lengths, keep, page = st["table"], st["lengths"], st["keep"], st["page"]
    kept = (keep >= 0).long().cumprod(-1)
    b, j = kept.nonzero(as_tuple=True)
    start = lengths[b].long()
    src, dst = start + keep[b, j].long(), start + j
    page_of = lambda p: table[b, p // page].long()  # noqa: E731
    for pages in (st["k_pages"], st["v_pages"]):
        pages[:, page_of(dst), :, dst % page] = pages[:, page_of(src), :, src % page]
    return {"lengths": (lengths + kept.sum(-1)).to(torch.int32), "k_pages": st["k_pages"],
            "v_pages": st["v_pages"]}


_PLAIN = {"tree_attention": _plain_tree_attention, "beam_select": _plain_beam_select,
          "fork_pages": _plain_fork_pages, "keep_nodes": _plain_keep_nodes}


# -- the definition in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    """What is computed: attention's rows and the beams' scores.  Pages are copied, not computed."""
    if case["op"] == "tree_attention":
        return _exact_tree_attention(case, prepare(case, seed))
    if case["op"] == "beam_select":
        return _exact_beam_select(prepare(case, seed))
    return None


def _exact_tree_attention(case, st):
    H, KV, hd, T, page = st["H"], st["KV"], st["hd"], st["T"], st["page"]
    out = torch.empty((case["seqs"], T, H, hd), dtype=torch.float64, device="cuda")
    for b, (n, tree) in enumerate(zip(_lengths(case), _trees(case))):
        hidden = torch.ones((T, T), dtype=torch.bool)
        for j, p in enumerate(tree):
            if p >= 0:
                hidden[j] = hidden[p]
            hidden[j, j] = False
        hidden = torch.cat((torch.zeros((T, n), dtype=torch.bool), hidden), 1).cuda()
        at = st["table"][b, :-(-(n + T) // page)].long()
        for h in range(KV):
            k, v = (st[name][at, h].double().flatten(0, 1)[:n + T] for name in ("k_pages", "v_pages"))
            q = st["q"][b, :, h * (H // KV):(h + 1) * (H // KV)].double()
            s = torch.einsum("tgd,nd->gtn", q, k).mul_(hd ** -0.5).masked_fill_(hidden, float("-inf"))
            out[b, :, h * (H // KV):(h + 1) * (H // KV)] = (torch.softmax(s, -1) @ v).transpose(0, 1)
    return {"o": out}


def _exact_beam_select(st):
    scores = []
    B, K = st["scores"].shape
    for b in range(B):
        p = torch.log_softmax(st["logits"][b * K:(b + 1) * K].double(), -1)
        scores.append(torch.topk((p + st["scores"][b].double()[:, None]).flatten(), st["count"]).values)
    return {"scores": torch.stack(scores), "parents": None, "tokens": None}


def work(case):
    """Each input read once and each output written once; multiply-adds as two."""
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "beam_select":
        rows = case["seqs"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * e + 4) + case["seqs"] * case["count"] * 16,
                "flops": 4 * rows * case["vocab"]}
    lens, KV, hd, page = _lengths(case), case["kv"], case["hd"], case["page"]
    if case["op"] == "tree_attention":
        B, T, H = case["seqs"], case["nodes"], case["heads"]
        seen = sum(d + 1 for tree in _trees(case) for d in _depths(tree))
        pairs = T * sum(lens) + seen
        tables = sum(-(-(n + T) // page) for n in lens)
        return {"bytes": (sum(lens) + B * T) * 2 * KV * hd * e + 2 * B * T * H * hd * e
                + 8 * B * T * -(-T // 64) + 4 * tables + 4 * B, "flops": 4 * pairs * H * hd}
    row = 2 * case["layers"] * KV * hd * e  # a position's keys and values in all layers
    if case["op"] == "keep_nodes":
        moved = sum(j != k for path in _accepted(case) for j, k in enumerate(path))
        kept = sum(map(len, _accepted(case)))
        return {"bytes": 2 * moved * row + 8 * kept + 8 * case["seqs"], "flops": moved}
    K, S = case["beams"], case["seqs"] * case["beams"]
    parents, copied, entries = _parents(case), 0, 0
    for b, n in enumerate(lens):
        total = n + case["grown"]
        kids = [parents[i] for i in range(b * K, (b + 1) * K)]
        entries += K * -(-total // page)
        copied += (K - len(set(kids))) * (total % page)
    return {"bytes": 2 * copied * row + 4 * (2 * entries + 4 * S), "flops": entries}


def _depths(tree):
    depth = []
    for p in tree:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth
